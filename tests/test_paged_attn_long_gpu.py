"""Tiles-form attention over long contexts: a piece of many keys is not one truncating sum.

Tolerance.  16-bit activations sum 8192 keys in the tensor core's accumulator, 512 steps of 16 keys that each lose
less than a unit of 2^-23 of the sum so far, which is below 512 * 2^-23 = 2^-14 of it; L/8192 such sums are added in
fp32, 2^-24 each.  fp32 activations sum 256 keys (16 steps, 2^-19), then L/256 roundings.  Beside that the output's
half step, and 2^-20 for the row sum, its reciprocal and the merge of pieces."""
import numpy as np
import pytest
import torch

from test_paged_attn_gpu import DT, Case, dev, many_rows  # noqa: F401  (dev is a fixture)

pytestmark = pytest.mark.gpu


def drift(act, L):
    return 2.0 ** -19 + L / 256 * 2.0 ** -24 if act == "f32" else 2.0 ** -14 + L / 8192 * 2.0 ** -24


@pytest.mark.parametrize("act,hd,H,L", [
    ("f16", 64, 2, 131072), ("f16", 128, 2, 131072), ("f16", 128, 1, 1 << 20), ("bf16", 256, 1, 1 << 20),
    ("bf16", 128, 1, 1 << 20), ("f32", 128, 1, 131072), ("f32", 256, 1, 131072),
])
def test_long_pieces_of_equal_scores(dev, act, hd, H, L):  # noqa: F811
    """As many tiles as CTAs, each over the whole context: q = 0, so a token's output is the mean of the V rows it sees
    (scores, exponentials and P are exact here, and the sums alone can be off)."""
    from yllm_b200 import attn
    n = 2 * 128 * torch.cuda.get_device_properties(0).multi_processor_count // H
    page = 256
    g = torch.Generator(device=dev).manual_seed(L + hd)
    kp = torch.randn(L // page, page, hd, generator=g, device=dev).half()
    vp = (torch.rand(L // page, page, hd, generator=g, device=dev) + 0.5).half()
    q = torch.zeros(n, H * hd, dtype=DT[act], device=dev)
    out = torch.full_like(q, 3.0)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    attn.attn_paged(out, q, kp, vp, torch.arange(L // page, dtype=torch.int32, device=dev)[None], i32([0, n]), i32([L]), n,
                    H, 1, hd)
    torch.cuda.synchronize()
    assert attn.device_status() == 0
    want = vp.view(L, hd).double().cumsum(0)[L - n:] / torch.arange(L - n + 1, L + 1, device=dev)[:, None]
    err = ((out.view(n, H, hd).double() - want[:, None]) / want[:, None]).abs().max()
    assert float(err) <= torch.finfo(DT[act]).eps / 2 + drift(act, L) + 2.0 ** -20


@pytest.mark.parametrize("act,hd,H,KV,L,n", [
    ("f16", 64, 8, 8, 320000, 33), ("bf16", 128, 8, 8, 400000, 40), ("f16", 128, 4, 1, 130000, 600),
    ("bf16", 256, 4, 4, 400000, 9), ("f32", 256, 4, 1, 30000, 300),
])
@pytest.mark.parametrize("large", [False, True])
def test_long_pieces_of_random_scores(dev, act, hd, H, KV, L, n, large):  # noqa: F811
    """Pieces past 8192 keys whose running maximum moves before and after a fold, whole or cut, one CTA per SM and two;
    V is positive, so that the output is sum p |v| / l and the bar's share for long sums can be taken at its value."""
    c = Case(dev, H, KV, hd, 64, [L, 700], [n, 1], act=act, seed=L, pad=many_rows(H) if large else 1, q_scale=2.0)
    c.vp.abs_()
    # later keys score higher: the maximum keeps growing
    for h in range(KV):
        cols = slice(h * hd, (h + 1) * hd)
        ramp = torch.linspace(0.5, 2.0, L, device=dev).half()[:, None]
        c.kp[c.rows[0], cols] *= ramp
    c.run()
    torch.cuda.synchronize()
    want, bar = c.want(False)
    from yllm_b200 import attn
    assert attn.device_status() == 0
    per = torch.zeros(c.total, dtype=torch.float64, device=dev)
    at = 0
    for Lr, m in zip(c.lens, c.new):
        per[at:at + m] = (Lr / 16 + 16) * 2.0 ** -24 - drift(act, Lr)
        at += m
    bar = bar - want.clamp(min=0) * per.clamp(min=0)[:, None]
    err = (c.out[:c.total, :H * hd].double() - want).abs()
    assert bool((err <= bar).all()), float((err / bar).max())
    first = c.out.clone()
    for _ in range(2):
        c.out.fill_(3.0)
        c.run()
        assert torch.equal(c.out, first)
    assert bool((c.out[c.total:] == 3.0).all())


def test_own_workspace_on_another_stream(dev):  # noqa: F811
    """paged_workspace() zeroes its counters behind work of the current stream; a call on another stream does not wait
    for that stream, and may come at once."""
    from yllm_b200 import attn
    c = Case(dev, 32, 8, 128, 64, [30000], [1], seed=50)
    s = torch.cuda.Stream()
    c.run(stream=s)
    torch.cuda.synchronize()
    good = c.out.clone()
    c.out.fill_(3.0)
    junk = torch.full((attn.paged_workspace(128).numel(),), 255, dtype=torch.uint8, device=dev)
    torch.cuda.synchronize()
    at = junk.data_ptr()
    del junk
    torch.cuda._sleep(200_000_000)                     # about 0.1 s on the current stream
    ws = attn.paged_workspace(128)
    assert ws.data_ptr() == at                         # (the memory that is not zero)
    c.run(workspace=ws, stream=s)
    s.synchronize()
    torch.cuda.synchronize()
    assert attn.device_status() == 0 and torch.equal(c.out, good)
