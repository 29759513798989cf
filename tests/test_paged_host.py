"""Argument checks of the paged-cache entry points, before any device work."""
import ctypes as C

import pytest

P = 0x10000    # stands for a device pointer: no refused call reads it


def _refused(name, args, word):
    from yllm_b200 import _lib
    err = C.create_string_buffer(512)
    assert getattr(_lib.lib, name)(*args, err, 512) == -1
    assert word in err.value.decode(), err.value.decode()


STEP = dict(kv_len_out=P, cu_new=P + 0x1000, slots=P + 0x2000, positions=P + 0x3000, max_tokens=8,
            state_out=P + 0x4000, tables=P + 0x5000, max_pages=4, table_stride=4, ring=P + 0x6000, n_pages=32,
            state=P + 0x7000, kv_len=P + 0x8000, new_len=P + 0x9000, n_seqs=4, page_size=16, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(kv_len_out=None), "null"), (dict(slots=None), "null"), (dict(page_size=8), "page_size"),
    (dict(page_size=48), "page_size"), (dict(page_size=512), "page_size"), (dict(n_seqs=0), "requests"),
    (dict(n_seqs=16385), "requests"), (dict(max_pages=0), "table"), (dict(table_stride=3), "table"),
    (dict(max_pages=1 << 27, table_stride=1 << 27), "table"), (dict(n_pages=0), "2^31"),
    (dict(n_pages=1 << 27), "2^31"), (dict(max_tokens=1 << 31), "2^31"), (dict(state_out=P + 0x4004), "aligned"),
    (dict(ring=P + 0x6001), "aligned"), (dict(kv_len_out=P + 0x8000), "overlaps"),
    (dict(cu_new=P + 0x9000 - 8), "overlaps"), (dict(state_out=P + 0x7000), "overlaps"),
])
def test_page_step_refuses(change, word):
    _refused("yattn_page_step", list(dict(STEP, **change).values()), word)


STORE = dict(q_out=P, qo_stride=512, q=P, q_stride=512, k=P, k_stride=128, v=P, v_stride=128, act=0, kpool=P, vpool=P,
             n_rows=64, slots=P, positions=P, n_tokens=3, n_heads=4, n_kv=1, head_dim=128, kv_dim=128, rope_kind=0,
             n_rope_dims=0, theta=1e4, norm=None, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(q=None), "null"), (dict(positions=None), "null"), (dict(act=3), "activation"), (dict(act=-1), "activation"),
    (dict(head_dim=80, q_stride=512), "head_dim"), (dict(n_heads=0), "geometry"), (dict(n_kv=5), "geometry"),
    (dict(kv_dim=120), "geometry"), (dict(kv_dim=132), "geometry"), (dict(rope_kind=3), "rope_kind"),
    (dict(rope_kind=2, n_rope_dims=0), "rotated"), (dict(rope_kind=2, n_rope_dims=24), "rotated"),
    (dict(rope_kind=2, n_rope_dims=144), "rotated"), (dict(theta=0.0), "theta"), (dict(theta=float("inf")), "theta"),
    (dict(theta=float("nan")), "theta"), (dict(q_stride=508), "strides"), (dict(k_stride=130), "strides"),
    (dict(act=1, v_stride=132), "strides"), (dict(v=P + 8), "aligned"), (dict(kpool=P + 2), "aligned"),
    (dict(slots=P + 2), "aligned"), (dict(n_rows=0), "pool rows"), (dict(n_rows=1 << 31), "pool rows"),
])
def test_store_refuses(change, word):
    _refused("yattn_rope_store_kv_paged", list(dict(STORE, **change).values()), word)


def test_store_refuses_bad_norm():
    from yllm_b200._lib import YattnQkNorm
    for norm, word in ((YattnQkNorm(P, None, 0, 1e-6), "QK-norm"), (YattnQkNorm(P + 2, P, 0, 1e-6), "aligned"),
                       (YattnQkNorm(P + 1, P, 1, 1e-6), "aligned")):
        _refused("yattn_rope_store_kv_paged", list(dict(STORE, norm=C.byref(norm)).values()), word)


def test_empty_calls_do_nothing():
    from yllm_b200 import _lib
    err = C.create_string_buffer(512)
    args = list(dict(STORE, n_tokens=0, q=None).values())
    assert _lib.lib.yattn_rope_store_kv_paged(*args, err, 512) == 0


ATTN = dict(out=P, out_stride=512, q=P, q_stride=512, gate=None, gate_stride=0, act=0, kpool=P, vpool=P, n_pages=8,
            page_size=16, tables=P, max_pages=4, table_stride=4, cu_new=P, kv_len=P, n_seqs=2, n_tokens=5, max_new=3,
            n_heads=4, n_kv=2, head_dim=128, kv_dim=256, ws=P, ws_bytes=1 << 30, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(out=None), "null"), (dict(tables=None), "null"), (dict(act=7), "activation"), (dict(page_size=24), "page_size"),
    (dict(head_dim=96), "head_dim"), (dict(n_kv=3), "multiple"), (dict(n_heads=0), "multiple"), (dict(n_kv=0), "multiple"),
    (dict(kv_dim=128), "kv_dim"), (dict(kv_dim=260), "kv_dim"), (dict(q_stride=500), "strides"),
    (dict(out_stride=514), "strides"), (dict(act=1, q_stride=516), "strides"),
    (dict(gate=P, gate_stride=256), "strides"), (dict(q=P + 4), "aligned"), (dict(gate=P + 4, gate_stride=512), "aligned"),
    (dict(ws=P + 8), "aligned"), (dict(cu_new=P + 1), "aligned"), (dict(max_pages=0), "table"),
    (dict(table_stride=3), "table"), (dict(max_pages=1 << 27, table_stride=1 << 27), "table"), (dict(n_pages=0), "2^31"),
    (dict(n_pages=1 << 27), "2^31"), (dict(n_seqs=65536), "requests"), (dict(n_tokens=1 << 30), "tokens"),
    (dict(n_tokens=1 << 28, max_pages=1 << 26, table_stride=1 << 26), "divide"), (dict(ws=None), "workspace"), (dict(ws_bytes=4096), "workspace"),
])
def test_attn_refuses(change, word):
    _refused("yattn_attn_paged", list(dict(ATTN, **change).values()), word)


@pytest.mark.parametrize("change", [dict(n_seqs=0), dict(n_tokens=0), dict(max_new=0)])
def test_attn_of_nothing(change):
    from yllm_b200 import _lib
    err = C.create_string_buffer(512)
    assert _lib.lib.yattn_attn_paged(*dict(ATTN, **change).values(), err, 512) == 0
