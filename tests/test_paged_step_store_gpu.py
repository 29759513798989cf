"""The page step and the paged QK-norm + RoPE + KV store against plain 64-bit forms.

Tolerances.  u = eps/2 of fp32 = 2^-24.
q and k in fp32: the angle in half turns is rounded once (|t| <= 1: at most u/2 half turns = 2^-24 rad about) and
sincospif is within 2 ulp of values up to 1, so sine and cosine are within 2^-22 of the truth; the rotation adds 3
roundings of terms up to the pair's norm; a norm factor adds about (hd/32 + 8) roundings.  Per element the error is
below (4 + 3 + hd/32 + 8) u * |pair| < 2^-19 |pair|, and the 16-bit roundings add half a step of the value."""
import numpy as np
import pytest
import torch

import paged_ref

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    torch.cuda.set_device(0)
    return torch.device("cuda:0")


def _i32(x, dev):
    return torch.tensor(np.asarray(x, np.int32), device=dev)


class Step:
    """Device buffers of a page step and its call."""

    def __init__(self, dev, tables, ring, head, count, kv_len, new_len, page, cap):
        self.np_in = (tables, ring, head, count, np.asarray(kv_len), np.asarray(new_len), page, cap)
        n = len(kv_len)
        self.page = page
        self.tables, self.ring = _i32(tables, dev), _i32(ring, dev)
        self.state = _i32([head, count], dev)
        self.kv_len, self.new_len = _i32(kv_len, dev), _i32(new_len, dev)
        e = lambda k: torch.full((k,), -77, dtype=torch.int32, device=dev)
        self.kv_out, self.cu, self.slots, self.pos, self.state_out = e(n), e(n + 1), e(cap), e(cap), e(4)

    def run(self, stream=None):
        from yllm_b200 import attn
        attn.page_step(self.kv_out, self.cu, self.slots, self.pos, self.state_out, self.tables, self.ring, self.state,
                       self.kv_len, self.new_len, self.page, stream=stream)

    def check(self):
        torch.cuda.synchronize()
        w = paged_ref.page_step(*self.np_in)
        for name, got in (("tables", self.tables), ("ring", self.ring), ("cu", self.cu), ("slots", self.slots),
                          ("positions", self.pos), ("kv_len", self.kv_out), ("state", self.state_out)):
            np.testing.assert_array_equal(got.cpu().numpy(), np.asarray(w[name]), err_msg=name)
        return w


def _requests(rng, n, page, max_len, max_new, ended, spare_pages=3):
    kv = rng.integers(0, max_len + 1, n)
    new = rng.integers(0, max_new + 1, n)
    new[rng.permutation(n)[:ended]] = -1
    held = -(-kv // page)
    grow = -(-(kv + np.maximum(new, 0)) // page) - held
    n_pages = int(held.sum() + grow.sum() + spare_pages)
    width = int(max(1, (held + grow).max())) + 2
    order = rng.permutation(n_pages).astype(np.int32)
    tables = np.full((n, width), -5, np.int32)
    at = 0
    for r in range(n):
        tables[r, :held[r]] = order[at:at + held[r]]
        at += held[r]
    count = n_pages - at
    head = int(rng.integers(0, n_pages))
    ring = np.full(n_pages, -9, np.int32)
    ring[(head + np.arange(count)) % n_pages] = order[at:]
    return tables, ring, head, count, kv, new


@pytest.mark.parametrize("n,page,max_len,max_new,ended,spare", [
    (1, 16, 0, 1, 0, 0), (1, 16, 40, 700, 0, 5), (2, 32, 64, 1, 1, 0), (7, 256, 2000, 600, 2, 3),
    (64, 16, 8192, 1, 3, 0), (513, 16, 300, 3, 20, 11), (1500, 64, 500, 40, 100, 1), (33, 128, 128, 0, 33, 4),
    (16384, 16, 33, 1, 500, 7),
])
def test_page_step(dev, n, page, max_len, max_new, ended, spare):
    rng = np.random.default_rng(n * 31 + page)
    tables, ring, head, count, kv, new = _requests(rng, n, page, max_len, max_new, ended)
    cap = int(np.maximum(new, 0).sum()) + spare
    s = Step(dev, tables, ring, head, count, kv, new, page, cap)
    s.run()
    w = s.check()
    assert w["state"][2] == 0
    s.run()      # the inputs are untouched: the same call again gives the same answer
    s.check()


def test_page_step_boundaries(dev):
    """Lengths around a page's end, with no new tokens, one, and a whole page."""
    page = 16
    kv = [0, 0, 15, 15, 16, 16, 17, 31, 32, 1]
    new = [0, 16, 1, 2, 0, 1, 16, 17, -1, 31]
    rng = np.random.default_rng(3)
    order = rng.permutation(40).astype(np.int32)
    tables, at = np.full((10, 6), -1, np.int32), 0
    for r, c in enumerate(kv):
        h = -(-c // page)
        tables[r, :h] = order[at:at + h]
        at += h
    ring = np.full(40, -1, np.int32)
    ring[(37 + np.arange(40 - at)) % 40] = order[at:]
    s = Step(dev, tables, ring, 37, 40 - at, kv, new, page, 90)
    s.run()
    s.check()


@pytest.mark.parametrize("what,verdict", [("missing", 1), ("tokens", -1), ("table", -2), ("negative", -3), ("new", -3),
                                          ("head", -3), ("count", -3), ("held", -3)])
def test_page_step_denied(dev, what, verdict):
    rng = np.random.default_rng(5)
    tables, ring, head, count, kv, new = _requests(rng, 20, 16, 100, 20, 2, spare_pages=0)
    cap = int(np.maximum(new, 0).sum())
    new = new.copy()
    if what == "missing":
        count -= 1
    elif what == "tokens":
        cap -= 1
    elif what == "table":
        new[7] = 5000
        cap += 5000
    elif what == "negative":
        kv = kv.copy()
        kv[3] = -1
    elif what == "new":
        new[3] = -2
    elif what == "head":
        head = ring.size
    elif what == "count":
        count = ring.size + 1
    elif what == "held":
        kv = kv.copy()
        kv[0] = tables.shape[1] * 16 + 1
    s = Step(dev, tables, ring, head, count, kv, new, 16, cap)
    s.run()
    w = s.check()
    assert w["state"][2] == verdict


def test_page_step_capture(dev):
    """Two captured steps in turn (kv_len -> kv_len_out -> kv_len), replayed with new lengths in place."""
    from yllm_b200 import attn
    n, page, n_pages, steps = 9, 16, 64, 6
    tables = torch.full((n, 16), -1, dtype=torch.int32, device=dev)
    ring = torch.arange(n_pages, dtype=torch.int32, device=dev)
    e = lambda k: torch.zeros(k, dtype=torch.int32, device=dev)
    kv, st = [e(n), e(n)], [e(4), e(4)]
    st[0][1] = n_pages
    new, cu, slots, pos = e(n), e(n + 1), e(40), e(40)
    graphs = []
    for a in (0, 1):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            attn.page_step(kv[1 - a], cu, slots, pos, st[1 - a], tables, ring, st[a], kv[a], new, page)
        graphs.append(g)
    rng = np.random.default_rng(11)
    T, R, head, count, lens = np.full((n, 16), -1, np.int32), np.arange(n_pages, dtype=np.int32), 0, n_pages, [0] * n
    for i in range(steps):
        want_new = rng.integers(-1, 5, n)
        new.copy_(_i32(want_new, dev))
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        w = paged_ref.page_step(T, R, head, count, lens, want_new, page, 40)
        T, R, (head, count), lens = w["tables"], w["ring"], w["state"][:2], list(w["kv_len"])
        np.testing.assert_array_equal(slots.cpu().numpy(), w["slots"])
        np.testing.assert_array_equal(st[1 - i % 2].cpu().numpy(), w["state"])
        np.testing.assert_array_equal(tables.cpu().numpy(), T)
        np.testing.assert_array_equal(ring.cpu().numpy(), R)


# ------------------------------------------------------------------ the store

def _pair_norm(x, heads, hd, kind, n):
    """Per element the norm of its rotation pair (dims that do not rotate: |x|)."""
    x = np.abs(x).reshape(-1, heads, hd).copy()
    j = np.arange(n // 2)
    e0, e1 = (2 * j, 2 * j + 1) if kind == 0 else (j, j + n // 2)
    r = np.hypot(x[..., e0], x[..., e1])
    x[..., e0], x[..., e1] = r, r
    return x.reshape(-1, heads * hd)


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,hd,kind,n_dims,theta,norm,T,pad,fused", [
    (32, 8, 128, 0, 0, 5e5, None, 9, 0, False),
    (14, 2, 64, 1, 0, 1e6, None, 1, 0, False),
    (16, 8, 128, 1, 0, 1e6, "f32", 37, 3, True),
    (16, 2, 256, 2, 64, 1e7, "f16", 21, 2, True),
    (5, 5, 64, 2, 16, 1e4, "f32", 130, 1, False),
    (3, 1, 256, 0, 0, 1e4, None, 2, 0, True),
    (64, 4, 256, 2, 256, 1e6, "f32", 3, 0, False),   # more items than one block of threads
])
def test_store(dev, act, H, KV, hd, kind, n_dims, theta, norm, T, pad, fused):
    from yllm_b200 import attn
    rng = np.random.default_rng(H * 7 + hd + T)
    kd, page, n_pages = KV * hd + (16 if not fused else 0), 16, -(-(T + pad) // 16) + 2
    rows = T + pad
    dt = DT[act]
    g = torch.Generator(device=dev).manual_seed(T + hd)
    qkv = torch.randn(rows, (H + 2 * KV) * hd, generator=g, device=dev).to(dt)
    q, k, v = qkv[:, :H * hd], qkv[:, H * hd:(H + KV) * hd], qkv[:, (H + KV) * hd:]
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    positions = rng.integers(0, 131072, rows)
    positions[0] = 131071
    slots = rng.permutation(n_pages * page)[:rows]
    slots[T:] = -1
    slots = slots[rng.permutation(rows)] if pad else slots    # padded rows need not be the last ones
    live = slots >= 0
    fill = lambda: torch.full((n_pages, page, kd), 0x7BCD, dtype=torch.int16, device=dev)
    kp, vp = fill(), fill()
    q_out = torch.full((rows, H * hd + 32), 7.0, dtype=dt, device=dev)
    wq = wk = n = None
    eps = 1e-6
    if norm:
        wq, wk = 1 + 0.3 * torch.randn(hd, generator=g, device=dev), 1 + 0.3 * torch.randn(hd, generator=g, device=dev)
        if norm == "f16":
            wq, wk = wq.half(), wk.half()
        n = attn.qk_norm(wq, wk, eps)
    attn.rope_store_kv_paged(q_out[:, :H * hd], q, k, v, kp, vp, _i32(slots, dev), _i32(positions, dev), H, KV, hd,
                             kind, theta, n_rope_dims=n_dims, norm=n)
    torch.cuda.synchronize()
    assert attn.device_status() == 0
    nd = n_dims if kind == 2 else hd
    f = lambda t: t.double().cpu().numpy()
    half_step = torch.finfo(dt).eps / 2

    def bars(want, heads, step):
        return 2.0 ** -19 * _pair_norm(want, heads, hd, kind, nd) + step * np.abs(want) + 2.0 ** -25

    want_q = paged_ref.rope_rows(f(q), positions, H, hd, kind, nd, theta, None if wq is None else f(wq), eps)[live]
    got_q = f(q_out)
    assert (np.abs(got_q[live][:, :H * hd] - want_q) <= bars(want_q, H, half_step)).all()
    assert (got_q[~live] == 7.0).all() and (got_q[:, H * hd:] == 7.0).all()
    want_k = paged_ref.rope_rows(f(k), positions, KV, hd, kind, nd, theta, None if wk is None else f(wk), eps)[live]
    rows_k, rows_v = kp.view(-1, kd).cpu().numpy(), vp.view(-1, kd).cpu().numpy()
    got_k = rows_k[slots[live]][:, :KV * hd].view(np.float16).astype(np.float64)
    assert (np.abs(got_k - want_k) <= bars(want_k, KV, 2.0 ** -11)).all()
    got_v = rows_v[slots[live]][:, :KV * hd].view(np.float16).astype(np.float64)
    want_v = f(v)[live]
    assert (np.abs(got_v - want_v) <= 2.0 ** -11 * np.abs(want_v) + 2.0 ** -25).all()
    other = np.ones(n_pages * page, bool)
    other[slots[live]] = False
    assert (rows_k[other] == 0x7BCD).all() and (rows_v[other] == 0x7BCD).all()
    assert (rows_k[:, KV * hd:] == 0x7BCD).all() and (rows_v[:, KV * hd:] == 0x7BCD).all()


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("T", [1500, 3001, 5003])
@pytest.mark.parametrize("H,KV,hd,kind,n_dims,norm", [(16, 8, 128, 1, 0, "f32"), (16, 2, 256, 2, 64, None), (16, 8, 128, 0, 0, None)])
def test_store_many_tokens(dev, act, T, H, KV, hd, kind, n_dims, norm):
    """Several tokens a block, one, two and four of them per barrier, the last ones of a group missing or skipped."""
    test_store(dev, act, H, KV, hd, kind, n_dims, 1e6, norm, T, 7, True)


def test_store_in_place_and_bad_slot(dev):
    """q_out = q; a slot outside the pool stores nothing and is reported."""
    from yllm_b200 import attn
    H, KV, hd, T = 4, 2, 64, 5
    q, k, v = (torch.randn(T, m * hd, device=dev) for m in (H, KV, KV))
    kp, vp = (torch.zeros(2, 16, KV * hd, dtype=torch.float16, device=dev) for _ in range(2))
    slots, pos = _i32([3, 32, 31, -1, 5], dev), _i32([0, 9, 100, 4, 77], dev)
    q2, out = q.clone(), torch.zeros_like(q)
    attn.rope_store_kv_paged(out, q, k, v, kp, vp, slots, pos, H, KV, hd, 1, 1e4)
    torch.cuda.synchronize()
    assert attn.device_status() == 602 and attn.device_status() == 0
    kp2, vp2 = kp.clone(), vp.clone()
    attn.rope_store_kv_paged(q2, q2, k, v, kp, vp, slots, pos, H, KV, hd, 1, 1e4)
    torch.cuda.synchronize()
    assert attn.device_status() == 602
    out[3] = q[3]    # a skipped token's row stays as it is
    assert torch.equal(q2, out) and torch.equal(kp, kp2) and torch.equal(vp, vp2)
    assert kp.view(32, -1)[[3, 31, 5]].abs().sum() > 0 and kp.view(32, -1)[[0, 1, 2, 4, 30]].abs().sum() == 0


def test_store_on_another_stream(dev):
    from yllm_b200 import attn
    H, KV, hd, T = 4, 4, 128, 64
    q, k, v = (torch.randn(T, m * hd, device=dev) for m in (H, KV, KV))
    kp, vp = (torch.zeros(8, 16, KV * hd, dtype=torch.float16, device=dev) for _ in range(2))
    slots, pos = _i32(np.arange(T), dev), _i32(np.arange(T), dev)
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    attn.rope_store_kv_paged(a, q, k, v, kp, vp, slots, pos, H, KV, hd, 0, 1e4)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    attn.rope_store_kv_paged(b, q, k, v, kp, vp, slots, pos, H, KV, hd, 0, 1e4, stream=s)
    s.synchronize()
    assert torch.equal(a, b)
