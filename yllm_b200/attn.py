"""Host-side mirror of the engine's attention entry points on torch tensors.

Each function forwards to the C ABI (include/yllm_attn_sm100.h) with the
tensors' device pointers and the current torch stream.  Names and argument
meaning follow the reference's CUDA launchers (inference/cuda/cuda_kernels.h):
cuda_k_attn_decode, cuda_k_attn_prefill, cuda_k_store_kv(_batch), plus the
batched / split-KV / gated / GDN entry points the engine lacks today.
Nothing here computes attention on the host: every path launches the CUDA
library, and a missing library fails at import.
"""
from __future__ import annotations

import ctypes as C
import os
import threading
from dataclasses import dataclass
from typing import Optional, Sequence

import numpy as np
import torch

from . import _lib
from ._lib import (YattnDecodeItem, YattnDecodeNewRow, YattnDecodeWork, YattnQkNorm, YattnRopeItem, call,
                   call_void, lib)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _stream(stream: Optional[torch.cuda.Stream] = None) -> int:
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def _need(t: torch.Tensor, dtype: torch.dtype, name: str) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _kv_tensor(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda or t.dtype not in (torch.uint16, torch.float16, torch.int16):
        raise ValueError(f"{name} must be a CUDA fp16-bits tensor (uint16/float16/int16)")


# ----------------------------------------------------------------- drop-ins

def cuda_k_attn_decode(att_out: torch.Tensor, q: torch.Tensor, kcache: torch.Tensor, vcache: torch.Tensor,
                       pos: int, n_heads: int, n_kv_heads: int, head_dim: int, kv_dim: int) -> None:
    """Same contract as the reference launcher (cuda_kernels.h:55-58), legacy default stream."""
    _need(att_out, torch.float32, "att_out")
    _need(q, torch.float32, "q")
    _kv_tensor(kcache, "kcache")
    _kv_tensor(vcache, "vcache")
    call_void("cuda_k_attn_decode", att_out.data_ptr(), q.data_ptr(), kcache.data_ptr(), vcache.data_ptr(),
              pos, n_heads, n_kv_heads, head_dim, kv_dim)


def cuda_k_attn_prefill(att_out: torch.Tensor, q: torch.Tensor, kcache: torch.Tensor, vcache: torch.Tensor,
                        pos_start: int, B: int, n_heads: int, n_kv_heads: int, head_dim: int, kv_dim: int,
                        q_stride: int) -> None:
    """Same contract as the reference launcher (cuda_kernels.h:60-63), legacy default stream."""
    _need(att_out, torch.float32, "att_out")
    _need(q, torch.float32, "q")
    _kv_tensor(kcache, "kcache")
    _kv_tensor(vcache, "vcache")
    call_void("cuda_k_attn_prefill", att_out.data_ptr(), q.data_ptr(), kcache.data_ptr(), vcache.data_ptr(),
              pos_start, B, n_heads, n_kv_heads, head_dim, kv_dim, q_stride)


PREFILL_Q_F16 = 1   # YATTN_PREFILL_Q_F16: every q value is an fp16 value


def attn_prefill(att_out: torch.Tensor, q: torch.Tensor, kcache: torch.Tensor, vcache: torch.Tensor,
                 pos_start: int, B: int, n_heads: int, n_kv_heads: int, head_dim: int, kv_dim: int, q_stride: int,
                 gate: Optional[torch.Tensor] = None, q_f16: bool = False, stream=None) -> None:
    """Causal prefill of B tokens at pos_start (keys 0..pos_start+b), optional qwen35 gate.  q_f16=True
    promises that every q value is exactly an fp16 value (the kernel then skips q's lo plane; it checks the
    promise and reports a broken one as device status 202)."""
    _need(att_out, torch.float32, "att_out")
    _need(q, torch.float32, "q")
    if gate is not None:
        _need(gate, torch.float32, "gate")
    call("yattn_attn_prefill", att_out.data_ptr(), q.data_ptr(), kcache.data_ptr(), vcache.data_ptr(), _ptr(gate),
         pos_start, B, n_heads, n_kv_heads, head_dim, kv_dim, q_stride, PREFILL_Q_F16 if q_f16 else 0,
         _stream(stream))


def cuda_k_store_kv(kcache: torch.Tensor, vcache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pos: int,
                    kv_dim: int) -> None:
    call_void("cuda_k_store_kv", kcache.data_ptr(), vcache.data_ptr(), k.data_ptr(), v.data_ptr(), pos, kv_dim)


def cuda_k_store_kv_batch(kcache: torch.Tensor, vcache: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                          pos_start: int, B: int, kv_dim: int) -> None:
    call_void("cuda_k_store_kv_batch", kcache.data_ptr(), vcache.data_ptr(), k.data_ptr(), v.data_ptr(),
              pos_start, B, kv_dim)


# ------------------------------------------------------- error-returning API

def attn_decode(att_out: torch.Tensor, q: torch.Tensor, kcache: torch.Tensor, vcache: torch.Tensor, pos: int,
                n_heads: int, n_kv_heads: int, head_dim: int, kv_dim: int, gate: Optional[torch.Tensor] = None,
                stream=None) -> None:
    """One decode query (keys 0..pos) of one layer; optional qwen35 sigmoid gate."""
    _need(att_out, torch.float32, "att_out")
    _need(q, torch.float32, "q")
    if gate is not None:
        _need(gate, torch.float32, "gate")
    call("yattn_attn_decode", att_out.data_ptr(), q.data_ptr(), kcache.data_ptr(), vcache.data_ptr(), _ptr(gate),
         pos, n_heads, n_kv_heads, head_dim, kv_dim, _stream(stream))


def store_kv(kcache: torch.Tensor, vcache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pos_start: int,
             kv_dim: int, stream=None) -> None:
    """fp32 rows -> fp16 cache rows pos_start.. with the engine's f32_to_f16 rounding."""
    _need(k, torch.float32, "k")
    _need(v, torch.float32, "v")
    B = k.numel() // kv_dim
    call("yattn_store_kv", kcache.data_ptr(), vcache.data_ptr(), k.data_ptr(), v.data_ptr(), pos_start, B, kv_dim,
         _stream(stream))


@dataclass
class DecodePlan:
    """A split schedule for a batch of decode queries (one per item).

    The schedule depends only on the query positions, so one plan serves every
    layer of a decode step: run() takes a device array of items per call.
    """

    n_items: int
    n_heads: int
    n_kv_heads: int
    head_dim: int
    kv_dim: int
    work: torch.Tensor        # device bytes of YattnDecodeWork[n_work]
    n_work: int
    n_parts: int
    n_groups: int
    workspace: Optional[torch.Tensor]
    pool: Optional[tuple] = None      # (base pointer, bytes): run through the pooled tensor-copy kernels

    @staticmethod
    def build(positions: Sequence[int], n_heads: int, n_kv_heads: int, head_dim: int, kv_dim: int,
              split_tokens: int = 0, target_ctas: int = 0, device=None,
              pool: Optional[tuple] = None) -> "DecodePlan":
        """pool = (base, bytes) of one allocation holding every item's K and V rows
        (row stride kv_dim): the plan and runs use the pooled variants."""
        pos = np.ascontiguousarray(np.asarray(positions, dtype=np.uint32))
        n = int(pos.size)
        cap = max(1, n * n_kv_heads * 64)
        while True:
            work = (YattnDecodeWork * cap)()
            n_work, n_parts, n_groups = C.c_uint32(), C.c_uint32(), C.c_uint32()
            err = C.create_string_buffer(512)
            plan_fn = lib.yattn_decode_plan_pooled if pool is not None else lib.yattn_decode_plan
            rc = plan_fn(pos.ctypes.data_as(C.POINTER(C.c_uint32)), n, n_kv_heads, head_dim,
                         split_tokens, target_ctas, work, cap, C.byref(n_work), C.byref(n_parts),
                         C.byref(n_groups), err, 512)
            if rc == 0:
                break
            if n_work.value > cap:
                cap = n_work.value
                continue
            raise _lib.YattnError("yattn_decode_plan: " + err.value.decode())
        nbytes = n_work.value * C.sizeof(YattnDecodeWork)
        host = torch.frombuffer(bytearray(C.string_at(work, nbytes)), dtype=torch.uint8)
        dev = host.to(device or "cuda")
        ws_bytes = lib.yattn_decode_workspace_bytes(n_parts.value, n_groups.value, n_heads, n_kv_heads, head_dim)
        ws = None
        if ws_bytes:
            ws = torch.zeros(ws_bytes, dtype=torch.uint8, device=device or "cuda")
        return DecodePlan(n, n_heads, n_kv_heads, head_dim, kv_dim, dev, n_work.value, n_parts.value,
                          n_groups.value, ws, tuple(pool) if pool is not None else None)

    def run_rope(self, items_dev: torch.Tensor, rows_dev: torch.Tensor, rope_kind: int, theta: float,
                 n_rope_dims: int = 0, stream=None) -> None:
        """run() with the step's RoPE + KV store fused in (yattn_decode_run_pooled_rope): items' q unrotated,
        rows_dev (make_new_rows) the new tokens' k and v; pooled plans only."""
        if self.pool is None:
            raise ValueError("the fused RoPE store runs on a pooled plan")
        ws_ptr = self.workspace.data_ptr() if self.workspace is not None else None
        ws_len = self.workspace.numel() if self.workspace is not None else 0
        call("yattn_decode_run_pooled_rope", items_dev.data_ptr(), rows_dev.data_ptr(), self.work.data_ptr(),
             self.n_work, self.n_parts, self.n_groups, self.n_heads, self.n_kv_heads, self.head_dim, self.kv_dim,
             self.pool[0], self.pool[1], rope_kind, n_rope_dims, theta, ws_ptr, ws_len, _stream(stream))

    def run(self, items_dev: torch.Tensor, stream=None) -> None:
        ws_ptr = self.workspace.data_ptr() if self.workspace is not None else None
        ws_len = self.workspace.numel() if self.workspace is not None else 0
        if self.pool is not None:
            call("yattn_decode_run_pooled", items_dev.data_ptr(), self.work.data_ptr(), self.n_work, self.n_parts,
                 self.n_groups, self.n_heads, self.n_kv_heads, self.head_dim, self.kv_dim, self.pool[0],
                 self.pool[1], ws_ptr, ws_len, _stream(stream))
        else:
            call("yattn_decode_run", items_dev.data_ptr(), self.work.data_ptr(), self.n_work, self.n_parts,
                 self.n_groups, self.n_heads, self.n_kv_heads, self.head_dim, self.kv_dim, ws_ptr, ws_len,
                 _stream(stream))


def make_items(entries: Sequence[tuple], device=None) -> torch.Tensor:
    """Device array of YattnDecodeItem from (q, out, k, v, gate_or_None, pos) tuples of tensors."""
    arr = (YattnDecodeItem * len(entries))()
    for i, (q, out, k, v, gate, pos) in enumerate(entries):
        arr[i].q = q.data_ptr()
        arr[i].out = out.data_ptr()
        arr[i].k = k.data_ptr() if isinstance(k, torch.Tensor) else int(k)
        arr[i].v = v.data_ptr() if isinstance(v, torch.Tensor) else int(v)
        arr[i].gate = gate.data_ptr() if gate is not None else 0
        arr[i].pos = int(pos)
    raw = bytearray(C.string_at(arr, C.sizeof(arr)))
    return torch.frombuffer(raw, dtype=torch.uint8).to(device or "cuda")


ROPE_LLAMA, ROPE_QWEN, ROPE_MROPE = 0, 1, 2


def make_new_rows(entries: Sequence[tuple], device=None) -> torch.Tensor:
    """Device array of YattnDecodeNewRow from (k, v) tensors: each item's new token (fp32, n_kv_heads*head_dim)."""
    arr = (YattnDecodeNewRow * len(entries))()
    for i, (k, v) in enumerate(entries):
        _need(k, torch.float32, "k")
        _need(v, torch.float32, "v")
        arr[i].k = k.data_ptr()
        arr[i].v = v.data_ptr()
    raw = bytearray(C.string_at(arr, C.sizeof(arr)))
    return torch.frombuffer(raw, dtype=torch.uint8).to(device or "cuda")


def make_rope_items(entries: Sequence[tuple], device=None) -> torch.Tensor:
    """Device array of YattnRopeItem from (q, k, v, kcache, vcache, pos) tuples; kcache / vcache are
    tensors or raw device addresses of the layer's cache bases."""
    arr = (YattnRopeItem * len(entries))()
    for i, (q, k, v, kc, vc, pos) in enumerate(entries):
        arr[i].q = q.data_ptr()
        arr[i].k = k.data_ptr()
        arr[i].v = v.data_ptr()
        arr[i].kcache = kc.data_ptr() if isinstance(kc, torch.Tensor) else int(kc)
        arr[i].vcache = vc.data_ptr() if isinstance(vc, torch.Tensor) else int(vc)
        arr[i].pos = int(pos)
    raw = bytearray(C.string_at(arr, C.sizeof(arr)))
    return torch.frombuffer(raw, dtype=torch.uint8).to(device or "cuda")


def qk_norm(q_w: torch.Tensor, k_w: torch.Tensor, eps: float):
    """The QK-norm argument of rope_store_kv(_batch): the layer's q and k rmsnorm weights (head_dim values, fp32,
    or fp16 as int16/uint16/float16 tensors) and eps (engine.c:915-919, 1036-1045)."""
    f16 = q_w.dtype in (torch.int16, torch.uint16, torch.float16)
    if f16 != (k_w.dtype in (torch.int16, torch.uint16, torch.float16)):
        raise ValueError("q and k norm weights must have the same dtype")
    for name, w in (("q_w", q_w), ("k_w", k_w)):
        _need(w, w.dtype if f16 else torch.float32, name)
    norm = YattnQkNorm(q_w.data_ptr(), k_w.data_ptr(), 1 if f16 else 0, float(eps))
    norm.weights = (q_w, k_w)   # lives as long as the pointers to it
    return norm


def _norm_arg(norm, head_dim: int, dev: Optional[int] = None):
    """The call's pointer to norm; weights that qk_norm holds must be head_dim values (on device dev, where given)."""
    if norm is None:
        return None
    for w in getattr(norm, "weights", ()):
        if w.numel() != head_dim:
            raise ValueError(f"QK-norm weights have {w.numel()} values for head_dim {head_dim}")
        if dev is not None and w.get_device() != dev:
            raise ValueError(f"QK-norm weights must be on cuda:{dev}")
    return C.byref(norm)


def rope_store_kv(items: torch.Tensor, n_items: int, n_heads: int, n_kv_heads: int, head_dim: int, kv_dim: int,
                  rope_kind: int, theta: float, n_rope_dims: int = 0, norm=None, stream=None) -> None:
    """One decode step's RoPE of q (in place) and k, and the fp16 store of k and v at each item's position
    (engine.c:1052-1072 / cuda_fwd.c:136-147 for every item, one launch).  norm (qk_norm(...)) applies the
    per-head QK-norm first."""
    call("yattn_rope_store_kv", items.data_ptr(), n_items, n_heads, n_kv_heads, head_dim, kv_dim, rope_kind,
         n_rope_dims, theta, _norm_arg(norm, head_dim), _stream(stream))


def rope_store_kv_batch(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kcache: torch.Tensor,
                        vcache: torch.Tensor, pos_start: int, B: int, n_heads: int, n_kv_heads: int, head_dim: int,
                        kv_dim: int, rope_kind: int, theta: float, n_rope_dims: int = 0, q_stride: int = 0,
                        norm=None, stream=None) -> None:
    """RoPE + KV store of B consecutive tokens (rows of q, k, v) at positions pos_start.. (the batched prefill's
    cuda_fwd.c:207-218 in one launch).  q is rotated in place; norm as in rope_store_kv."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        _need(t, torch.float32, name)
    call("yattn_rope_store_kv_batch", q.data_ptr(), k.data_ptr(), v.data_ptr(), kcache.data_ptr(), vcache.data_ptr(),
         pos_start, B, q_stride or n_heads * head_dim, n_heads, n_kv_heads, head_dim, kv_dim, rope_kind, n_rope_dims,
         theta, _norm_arg(norm, head_dim), _stream(stream))


def decode_partial(ml: torch.Tensor, o: torch.Tensor, q: torch.Tensor, kcache: torch.Tensor, vcache: torch.Tensor,
                   t_begin: int, t_end: int, n_heads: int, n_kv_heads: int, head_dim: int, kv_dim: int,
                   stream=None) -> None:
    """Unmerged (m, l, o) over keys [t_begin, t_end): m in log2 units (score*log2 e)."""
    call("yattn_decode_partial", ml.data_ptr(), o.data_ptr(), q.data_ptr(), kcache.data_ptr(), vcache.data_ptr(),
         t_begin, t_end, n_heads, n_kv_heads, head_dim, kv_dim, None, 0, _stream(stream))


def merge_partials(out: torch.Tensor, ml: torch.Tensor, o: torch.Tensor, n_parts: int, n_heads: int,
                   head_dim: int, gate: Optional[torch.Tensor] = None, stream=None) -> None:
    """Log-sum-exp merge of [n_parts][n_heads] partials into out[n_heads*head_dim]."""
    call("yattn_merge_partials", out.data_ptr(), ml.data_ptr(), o.data_ptr(), n_parts, n_heads, head_dim,
         _ptr(gate), _stream(stream))


def merge_partials_packed(out: torch.Tensor, parts: torch.Tensor, n_parts: int, n_heads: int, head_dim: int,
                          gate: Optional[torch.Tensor] = None, stream=None) -> None:
    """Log-sum-exp merge of packed parts [n_parts][n_heads*2 (m, l) + n_heads*head_dim (o)]."""
    call("yattn_merge_partials_packed", out.data_ptr(), parts.data_ptr(), n_parts, n_heads, head_dim, _ptr(gate),
         _stream(stream))


def cuda_k_gdn_state_update(S: torch.Tensor, out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                            gate: torch.Tensor, beta: torch.Tensor, num_k_heads: int, hk: int, n_vheads: int,
                            hv: int) -> None:
    """gdn_state_update (matvec.h:35-37) on device tensors, legacy default stream."""
    call_void("cuda_k_gdn_state_update", S.data_ptr(), out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
              gate.data_ptr(), beta.data_ptr(), num_k_heads, hk, n_vheads, hv)


def gdn_decode(S, out, q, k, v, gate, beta, n_seqs: int, num_k_heads: int, hk: int, n_vheads: int, hv: int,
               norm_w: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, eps: float = 1e-6,
               stream=None) -> None:
    """One GDN token for each of n_seqs sequences (state updated in place)."""
    for name, t in (("S", S), ("out", out), ("q", q), ("k", k), ("v", v), ("gate", gate), ("beta", beta)):
        _need(t, torch.float32, name)
    call("yattn_gdn_decode", S.data_ptr(), out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
         gate.data_ptr(), beta.data_ptr(), n_seqs, num_k_heads, hk, n_vheads, hv, _ptr(norm_w), _ptr(z), float(eps),
         _stream(stream))


def gdn_inputs(qkv, conv_state, conv_w, alpha, beta_in, ssm_dt, ssm_a, q, k, v, gate, beta, n_seqs: int, T: int,
               kwidth: int, num_k_heads: int, hk: int, n_vheads: int, hv: int, eps: float = 1e-6,
               stream=None) -> None:
    """The GDN layer's inputs for T tokens of n_seqs sequences (engine.c:785-821): gates, conv1d + silu, q/k/v
    split with l2-normalised q and k heads; conv_state updated in place."""
    for name, t in (("qkv", qkv), ("conv_state", conv_state), ("conv_w", conv_w), ("alpha", alpha),
                    ("beta_in", beta_in), ("ssm_dt", ssm_dt), ("ssm_a", ssm_a), ("q", q), ("k", k), ("v", v),
                    ("gate", gate), ("beta", beta)):
        _need(t, torch.float32, name)
    conv_chan = 2 * num_k_heads * hk + n_vheads * hv
    call("yattn_gdn_inputs", qkv.data_ptr(), conv_state.data_ptr(), conv_w.data_ptr(), alpha.data_ptr(),
         beta_in.data_ptr(), ssm_dt.data_ptr(), ssm_a.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
         gate.data_ptr(), beta.data_ptr(), n_seqs, T, conv_chan, kwidth, num_k_heads, hk, n_vheads, hv, float(eps),
         _stream(stream))


def gdn_prefill(S, out, q, k, v, gate, beta, n_seqs: int, T: int, num_k_heads: int, hk: int, n_vheads: int,
                hv: int, norm_w: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                eps: float = 1e-6, stream=None) -> None:
    """T GDN tokens per sequence in order (state updated in place)."""
    for name, t in (("S", S), ("out", out), ("q", q), ("k", k), ("v", v), ("gate", gate), ("beta", beta)):
        _need(t, torch.float32, name)
    call("yattn_gdn_prefill", S.data_ptr(), out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
         gate.data_ptr(), beta.data_ptr(), n_seqs, T, num_k_heads, hk, n_vheads, hv, _ptr(norm_w), _ptr(z),
         float(eps), _stream(stream))


def gdn_prefill_recurrent(S, out, q, k, v, gate, beta, n_seqs: int, T: int, num_k_heads: int, hk: int,
                          n_vheads: int, hv: int, norm_w: Optional[torch.Tensor] = None,
                          z: Optional[torch.Tensor] = None, eps: float = 1e-6, stream=None) -> None:
    """gdn_prefill token by token in the reference's operation order (GPU cross-check)."""
    for name, t in (("S", S), ("out", out), ("q", q), ("k", k), ("v", v), ("gate", gate), ("beta", beta)):
        _need(t, torch.float32, name)
    call("yattn_gdn_prefill_recurrent", S.data_ptr(), out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
         gate.data_ptr(), beta.data_ptr(), n_seqs, T, num_k_heads, hk, n_vheads, hv, _ptr(norm_w), _ptr(z),
         float(eps), _stream(stream))


def gemv_q4k(y: torch.Tensor, w: torch.Tensor, x: torch.Tensor, out: int, in_: int, B: int = 1,
             stream=None) -> None:
    """y[B][out] = Q4_K W[out][in] . x[B][in] (cuda_kernels.cu:161-249 semantics, fp32 x)."""
    _need(y, torch.float32, "y")
    _need(x, torch.float32, "x")
    if w.dtype != torch.uint8 or not w.is_cuda or w.numel() < out * (in_ // 256) * 144:
        raise ValueError("w must be a CUDA uint8 tensor of out * in/256 Q4_K blocks")
    call("yattn_gemv_q4k", y.data_ptr(), w.data_ptr(), x.data_ptr(), out, in_, B, _stream(stream))


def gemv_q4k_multi(ys, ws, outs, x: torch.Tensor, in_: int, stream=None) -> None:
    """One token through up to four Q4_K matrices that read the same x, in one launch: ys[i][:outs[i]] =
    W_i . x, each bit-identical to gemv_q4k(ys[i], ws[i], x, outs[i], in_) (the engine's q/k/v or gate/up
    calls of cuda_fwd.c:94-168 fused)."""
    n = len(ws)
    if not (1 <= n <= 4) or len(ys) != n or len(outs) != n:
        raise ValueError("gemv_q4k_multi: 1 to 4 matrices, with as many outputs and row counts")
    _need(x, torch.float32, "x")
    for y, w, o in zip(ys, ws, outs):
        _need(y, torch.float32, "y")
        if w.dtype != torch.uint8 or not w.is_cuda or w.numel() < o * (in_ // 256) * 144:
            raise ValueError("w must be a CUDA uint8 tensor of out * in/256 Q4_K blocks")
    yp = (C.c_void_p * n)(*[y.data_ptr() for y in ys])
    wp = (C.c_void_p * n)(*[w.data_ptr() for w in ws])
    op = (C.c_uint32 * n)(*[int(o) for o in outs])
    call("yattn_gemv_q4k_multi", n, yp, wp, op, x.data_ptr(), in_, _stream(stream))


def gemv_f16(y: torch.Tensor, w: torch.Tensor, x: torch.Tensor, out: int, in_: int, B: int = 1,
             stream=None) -> None:
    """y[B][out] = fp16 W[out][in] . x[B][in] in fp32 (matvec.c:111-122 per token)."""
    _need(y, torch.float32, "y")
    _need(x, torch.float32, "x")
    if w.element_size() != 2 or not w.is_cuda or w.numel() < out * in_:
        raise ValueError("w must be a CUDA 16-bit tensor of out * in fp16 weights")
    call("yattn_gemv_f16", y.data_ptr(), w.data_ptr(), x.data_ptr(), out, in_, B, _stream(stream))


# ------------------------------------------------------------- paged KV cache

_ACT = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}   # YATTN_ACT_*
_F16_BITS = (torch.float16, torch.uint16, torch.int16)
_U32 = 0xFFFFFFFF   # a larger number would reach the library without its upper bits


_tls = threading.local()   # err: this thread's message buffer
_raw_stream = torch._C._cuda_getCurrentRawStream
_cur_dev = torch._C._cuda_getDevice                       # (torch.cuda's wrappers of these cost as much as a launch)
_capturing = torch._C._cuda_isCurrentStreamCapturing


def _call_on(name: str, dev: int, stream, *args) -> None:
    """call() on device dev, on the given stream of it or its current one.  One message buffer per thread: the
    library writes it on failure only."""
    if stream is None:
        raw = _raw_stream(dev)
    elif stream.device_index == dev:
        raw = stream.cuda_stream
    else:
        raise ValueError(f"{name}: the stream is on cuda:{stream.device_index}, the tensors on cuda:{dev}")
    try:
        err = _tls.err
    except AttributeError:
        err = _tls.err = C.create_string_buffer(512)
    if dev == _cur_dev():
        rc = getattr(lib, name)(*args, raw, err, 512)
    else:
        with torch.cuda.device(dev):
            rc = getattr(lib, name)(*args, raw, err, 512)
    if rc != 0:
        raise _lib.YattnError(f"{name}: {err.value.decode(errors='replace')}")


def _i32_on(dev: int, names: str, *tensors: torch.Tensor) -> None:
    i32 = torch.int32
    for i, t in enumerate(tensors):
        if t.dtype is not i32 or t.get_device() != dev or not t.is_contiguous():
            raise ValueError(f"{names.split()[i]} must be a contiguous int32 tensor on cuda:{dev}")


def _table_shape(tables: torch.Tensor, dev: int, n: int) -> tuple:
    """(pages per row, row stride) of a block table of n requests."""
    if tables.dtype is torch.int32 and tables.get_device() == dev and tables.dim() == 2:
        rows, width = tables.shape
        stride, one = tables.stride()
        if rows == 1 and width > 0:
            stride = width
        if rows == n and width > 0 and (one == 1 or width == 1) and width <= stride <= _U32:
            return width, stride
    raise ValueError(f"tables must be an int32 [{n} requests, pages] tensor on cuda:{dev} with contiguous rows")


def _pool_shape(kpool: torch.Tensor, vpool: torch.Tensor, dev: int, row: int) -> tuple:
    """(pages, page size, kv_dim) of a layer's pools."""
    shape = kpool.shape
    if (len(shape) != 3 or vpool.shape != shape or kpool.dtype not in _F16_BITS or vpool.dtype not in _F16_BITS
            or kpool.get_device() != dev or vpool.get_device() != dev or not kpool.is_contiguous()
            or not vpool.is_contiguous()):
        raise ValueError(f"kpool and vpool must be contiguous fp16 [pages, page_size, kv_dim] tensors of one shape on cuda:{dev}")
    if shape[2] < row:
        raise ValueError("the pools' rows are shorter than n_kv_heads * head_dim")
    return shape


def _token_stride(t: torch.Tensor, name: str, rows: int, cols: int, dtype: torch.dtype, dev: int) -> int:
    """Elements between the tokens of a [rows, cols] activation tensor whose heads are contiguous."""
    if t.dtype is dtype and t.get_device() == dev and t.dim() == 2:
        n, m = t.shape
        stride, one = t.stride()
        if rows == 1:
            stride = cols
        if n == rows and m == cols and one == 1 and (cols <= stride <= _U32 or n == 0):
            return stride
    raise ValueError(f"{name} must be [{rows}, {cols}] {dtype} on cuda:{dev}, heads contiguous, tokens less than 2^32 elements apart")


def _act_of(q: torch.Tensor) -> tuple:
    """(YATTN_ACT_*, dtype, device index, rows) of the queries."""
    act = _ACT.get(q.dtype)
    dev = q.get_device()
    if act is None or dev < 0 or q.dim() != 2:
        raise ValueError("q must be a CUDA [tokens, heads*head_dim] tensor of float32, float16 or bfloat16")
    return act, q.dtype, dev, q.shape[0]


def page_step(kv_len_out: torch.Tensor, cu_new: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor,
              state_out: torch.Tensor, tables: torch.Tensor, ring: torch.Tensor, state: torch.Tensor,
              kv_len: torch.Tensor, new_len: torch.Tensor, page_size: int, stream=None) -> None:
    """One serving step's block tables (tables and the free-page queue ring updated in place), slots and positions
    of the new tokens (slots.numel() is the token capacity), prefix sums and lengths, from kv_len and new_len (-1:
    the request ended).  state_out = {head, count, verdict, tokens}; see yattn_page_step for the verdicts."""
    dev = kv_len.get_device()
    if dev < 0:
        raise ValueError("kv_len must be a CUDA tensor")
    _i32_on(dev, "kv_len new_len kv_len_out cu_new slots positions state_out ring state", kv_len, new_len, kv_len_out,
            cu_new, slots, positions, state_out, ring, state)
    n, cap = kv_len.numel(), slots.numel()
    width, stride = _table_shape(tables, dev, n)
    if new_len.numel() != n or kv_len_out.numel() != n or cu_new.numel() != n + 1:
        raise ValueError("new_len, kv_len_out and cu_new (one more) must have one entry per request of kv_len")
    if positions.numel() != cap or state.numel() < 2 or state_out.numel() < 4:
        raise ValueError("positions must match slots; state holds 2 values or more, state_out 4")
    _call_on("yattn_page_step", dev, stream, kv_len_out.data_ptr(), cu_new.data_ptr(), slots.data_ptr(),
             positions.data_ptr(), cap, state_out.data_ptr(), tables.data_ptr(), width, stride, ring.data_ptr(),
             ring.numel(), state.data_ptr(), kv_len.data_ptr(), new_len.data_ptr(), n, page_size)


def rope_store_kv_paged(q_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kpool: torch.Tensor,
                        vpool: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor, n_heads: int,
                        n_kv_heads: int, head_dim: int, rope_kind: int, theta: float, n_rope_dims: int = 0, norm=None,
                        stream=None) -> None:
    """QK-norm (norm = qk_norm(...)), RoPE and the store of k and v into pages: q, k, v [tokens, heads*head_dim]
    (fp32, fp16 or bf16, any row stride), slots and positions from page_step; tokens with slot -1 are skipped.
    q_out may be q."""
    act, dtype, dev, rows = _act_of(q)
    cols, kv_cols = n_heads * head_dim, n_kv_heads * head_dim
    pages, page_size, kv_dim = _pool_shape(kpool, vpool, dev, kv_cols)
    _i32_on(dev, "slots positions", slots, positions)
    if slots.numel() != rows or positions.numel() != rows:
        raise ValueError("slots and positions must have one entry per row of q")
    _call_on("yattn_rope_store_kv_paged", dev, stream, q_out.data_ptr(),
             _token_stride(q_out, "q_out", rows, cols, dtype, dev), q.data_ptr(),
             _token_stride(q, "q", rows, cols, dtype, dev), k.data_ptr(),
             _token_stride(k, "k", rows, kv_cols, dtype, dev), v.data_ptr(),
             _token_stride(v, "v", rows, kv_cols, dtype, dev), act, kpool.data_ptr(), vpool.data_ptr(),
             pages * page_size, slots.data_ptr(), positions.data_ptr(), rows, n_heads, n_kv_heads, head_dim, kv_dim,
             rope_kind, n_rope_dims, theta, _norm_arg(norm, head_dim, dev))


_paged_ws: dict = {}   # (device, stream, head_dim) -> workspace of attn_paged's eager calls on that stream


def _new_workspace(head_dim: int, dev: int) -> torch.Tensor:
    """A workspace whose counters are zeroed in the order of the current stream of dev."""
    with torch.cuda.device(dev):
        ws = torch.empty(lib.yattn_attn_paged_workspace_bytes(head_dim), dtype=torch.uint8, device=torch.device("cuda", dev))
        ws[:4096].zero_()
    return ws


def paged_workspace(head_dim: int, device=None) -> torch.Tensor:
    """A workspace for attn_paged (its counters zeroed), for callers that keep their own (one per stream or graph in
    flight).  Made outside a capture, it is ready for any stream when the call returns."""
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise ValueError(f"paged_workspace: {device} is not a CUDA device")
    dev = torch.cuda.current_device() if device.index is None else device.index
    ws = _new_workspace(head_dim, dev)
    if not torch.cuda.is_current_stream_capturing():
        torch.cuda.current_stream(dev).synchronize()
    return ws


def _paged_workspace(head_dim: int, dev: int, stream) -> torch.Tensor:
    """The stream's own workspace: calls on one stream run in order, so they can share it.  A call being captured
    gets a fresh one (its zeroing is captured too): the graph may be replayed beside other work."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return _paged_workspace(head_dim, dev, None)
    if _cur_dev() != dev:
        with torch.cuda.device(dev):
            return _paged_workspace(head_dim, dev, None)
    if _capturing():
        return _new_workspace(head_dim, dev)
    key = (dev, _raw_stream(dev), head_dim)
    ws = _paged_ws.get(key)
    if ws is None:
        ws = _paged_ws[key] = _new_workspace(head_dim, dev)
    return ws


def attn_paged(out: torch.Tensor, q: torch.Tensor, kpool: torch.Tensor, vpool: torch.Tensor, tables: torch.Tensor,
               cu_new: torch.Tensor, kv_len: torch.Tensor, max_new: int, n_heads: int, n_kv_heads: int, head_dim: int,
               gate: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None, stream=None) -> None:
    """Causal attention of ragged new tokens (rows cu_new[r]..cu_new[r+1] of q, fp32 / fp16 / bf16) over the first
    kv_len[r] rows of each request's pages, the new tokens' rows included; max_new bounds a request's new tokens.
    Rows of out behind the last request stay as they are."""
    act, dtype, dev, rows = _act_of(q)
    cols = n_heads * head_dim
    pages, page_size, kv_dim = _pool_shape(kpool, vpool, dev, n_kv_heads * head_dim)
    _i32_on(dev, "cu_new kv_len", cu_new, kv_len)
    n = kv_len.numel()
    width, stride = _table_shape(tables, dev, n)
    if cu_new.numel() != n + 1:
        raise ValueError("cu_new must have one entry more than kv_len")
    if max_new < 0:
        raise ValueError(f"max_new {max_new} is negative")
    if workspace is None:
        workspace = _paged_workspace(head_dim, dev, stream)
    elif workspace.get_device() != dev or not workspace.is_contiguous():
        raise ValueError(f"workspace must be a contiguous tensor on cuda:{dev} (paged_workspace)")
    _call_on("yattn_attn_paged", dev, stream, out.data_ptr(), _token_stride(out, "out", rows, cols, dtype, dev),
             q.data_ptr(), _token_stride(q, "q", rows, cols, dtype, dev), None if gate is None else gate.data_ptr(),
             0 if gate is None else _token_stride(gate, "gate", rows, cols, dtype, dev), act, kpool.data_ptr(),
             vpool.data_ptr(), pages, page_size, tables.data_ptr(), width, stride, cu_new.data_ptr(),
             kv_len.data_ptr(), n, rows, min(max_new, _U32), n_heads, n_kv_heads, head_dim, kv_dim, workspace.data_ptr(),
             workspace.nbytes)


def sess_kv_save(kv: torch.Tensor, n_blocks: int, kv_dim: int, max_seq: int, pos: int, path: str,
                 stream=None) -> None:
    """Writes the first pos rows of every block's K and V regions of the device blob kv
    ([2*n_blocks+1][max_seq][kv_dim] fp16) as the engine's session KV file (cache.c:174-195)."""
    if kv.numel() * kv.element_size() < (2 * n_blocks + 1) * max_seq * kv_dim * 2:
        raise ValueError("kv is smaller than the (2*n_blocks+1)-region blob")
    call("yattn_sess_kv_save", kv.data_ptr(), n_blocks, kv_dim, max_seq, pos, os.fsencode(path), _stream(stream))


def sess_kv_load(kv: torch.Tensor, n_blocks: int, kv_dim: int, max_seq: int, path: str, stream=None) -> int:
    """Reads an engine session KV file into the device blob kv; returns the file's pos (cache.c:219-247)."""
    if kv.numel() * kv.element_size() < (2 * n_blocks + 1) * max_seq * kv_dim * 2:
        raise ValueError("kv is smaller than the (2*n_blocks+1)-region blob")
    p = C.c_uint32(0)
    call("yattn_sess_kv_load", kv.data_ptr(), n_blocks, kv_dim, max_seq, os.fsencode(path), C.byref(p),
         _stream(stream))
    return p.value


def device_status(clear: bool = True) -> int:
    st = C.c_int(0)
    call("yattn_device_status", C.byref(st), 1 if clear else 0)
    if st.value != 0:
        # a paged attention that gave up (601) leaves its workspace's counters other than zero.  The word holds the first
        # code only, so any code may stand before a 601
        _paged_ws.clear()
    return st.value


def reserve(nbytes: int) -> None:
    call("yattn_reserve", nbytes)


def version() -> int:
    return lib.yattn_version()
