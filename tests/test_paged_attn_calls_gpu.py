"""Paged attention as callers mix it: wide pool rows, calls after skipped requests, host threads."""
import threading

import pytest
import torch

import test_paged_step_store_gpu as store
from test_paged_attn_gpu import Case, dev, many_rows  # noqa: F401  (dev is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,hd", [(14, 2, 64), (32, 8, 128), (16, 2, 256)])
@pytest.mark.parametrize("large", [False, True])
def test_chunks_in_wide_pool_rows(dev, act, H, KV, hd, large):  # noqa: F811
    """Pools whose rows are longer than the kv heads, whatever lies behind them."""
    c = Case(dev, H, KV, hd, 32, [40, 1, 129, 700, 0, 257], [40, 1, 129, 33, 0, 100], act=act, seed=H, kv_extra=24,
             pad=many_rows(H) if large else 2, gate=hd == 64)
    c.kp[:, KV * hd:] = float("nan")
    c.vp[:, KV * hd:] = float("inf")
    c.run()
    c.check()


@pytest.mark.parametrize("lens,new", [([9], [9]), ([1000], [1000]), ([40000], [33]), ([3, 0, 40], [60, 20, 40])])
@pytest.mark.parametrize("H,KV,hd", [(32, 8, 128), (14, 2, 64), (16, 2, 256)])
def test_fp16_chunk_lengths(dev, lens, new, H, KV, hd):  # noqa: F811
    c = Case(dev, H, KV, hd, 16, lens, new, act="f16", seed=sum(lens) + hd, pad=1)
    c.run()
    c.check()


@pytest.mark.parametrize("T", [1500, 3001, 5003])
@pytest.mark.parametrize("H,KV,hd,kind,n_dims,norm", [(16, 8, 128, 1, 0, "f32"), (16, 2, 256, 2, 64, None), (14, 2, 64, 0, 0, "f16")])
def test_fp16_store_of_many_tokens(dev, T, H, KV, hd, kind, n_dims, norm):  # noqa: F811
    store.test_store(dev, "f16", H, KV, hd, kind, n_dims, 1e6, norm, T, 7, True)


@pytest.mark.parametrize("act,new,large", [("f32", [2, 1, 2], 0), ("f32", [30, 1, 40], 0), ("bf16", [30, 1, 40], 0), ("bf16", [30, 1, 40], 1)])
@pytest.mark.parametrize("what", ["cu falls", "cu past the rows", "negative length", "length past the table", "max_new"])
def test_a_call_after_a_skipped_request(dev, what, act, new, large):  # noqa: F811
    """A call that skips a request leaves its workspace as it was: the next one, with the request mended, is right.  The
    contexts are long enough for cut units."""
    from yllm_b200 import attn
    c = Case(dev, 8, 2, 64, 16, [5000, 90, 6000], new, act=act, seed=7, pad=many_rows(8) if large else 0)
    ws = attn.paged_workspace(64)
    cu, kv = c.cu.clone(), c.kv.clone()
    kw = {}
    if what == "cu falls":
        c.cu[3] = int(c.cu[2]) - 1
    elif what == "cu past the rows":
        c.cu[3] = c.q.shape[0] + 1
    elif what == "negative length":
        c.kv[2] = -5
    elif what == "length past the table":
        c.kv[2] = c.tables.shape[1] * 16 + 1
    else:
        kw["max_new"] = new[2] - 1
    attn.device_status()
    c.run(workspace=ws, **kw)
    torch.cuda.synchronize()
    assert attn.device_status() == 603
    assert bool((ws[:4096] == 0).all())
    assert bool((c.out[sum(new[:2]):, :512] == 3.0).all())
    c.cu.copy_(cu)
    c.kv.copy_(kv)
    c.out.fill_(3.0)
    c.run(workspace=ws)
    c.check()
    assert bool((ws[:4096] == 0).all())


def test_host_threads(dev):  # noqa: F811
    """Calls of several forms from host threads of their own, each on its stream."""
    cases = [Case(dev, 32, 8, 128, 16, [20000], [1], seed=1), Case(dev, 8, 2, 64, 16, [9000, 40], [70, 1], seed=2),
             Case(dev, 8, 2, 256, 16, [5000], [33], act="bf16", seed=3), Case(dev, 8, 2, 128, 64, [4000], [50], act="f16", seed=4)]
    torch.cuda.synchronize()
    errors = []

    def work(c):
        try:
            torch.cuda.set_device(dev)
            s = torch.cuda.Stream()
            for _ in range(100):
                c.run(stream=s)
            s.synchronize()
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=(c,)) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for c in cases:
        c.check()
