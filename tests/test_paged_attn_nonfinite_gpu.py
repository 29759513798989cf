"""Paged attention where q, K or V hold infinities and NaN.  The definition says what comes out: a score of NaN or +inf
makes its row NaN, one of -inf has weight zero, and a row whose keys all score -inf is 0 / 0."""
import pytest
import torch

from test_paged_attn_gpu import Case, dev, many_rows  # noqa: F401  (dev is a fixture)

pytestmark = pytest.mark.gpu

FORMS = [(1, 0), (20, 0), (20, 1)]   # new tokens, large call: the decode form, the tiles, two CTAs per SM


def _case(dev, act, hd, L, new, large, **kw):  # noqa: F811
    return Case(dev, 8, 2, hd, 16, [max(L, new), 50], [new, 1], act=act, seed=L + hd, pad=many_rows(8) if large else 1, **kw)


def _status():
    from yllm_b200 import attn
    torch.cuda.synchronize()
    return attn.device_status()


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("L", [1, 17, 129, 9000])
@pytest.mark.parametrize("new,large", FORMS)
def test_all_scores_minus_infinity(dev, act, hd, L, new, large):  # noqa: F811
    """Whole and cut units: 0 / 0, not zeros, for every token that sees a key; the other request is untouched by it."""
    c = _case(dev, act, hd, L, new, large)
    c.run()
    assert _status() == 0
    other = c.out[new].clone()
    c.q[:new] = 1.0
    c.kp[c.rows[0]] = float("-inf")
    c.out.fill_(3.0)
    c.run()
    assert _status() == 0
    cols = slice(0, 8 * hd)
    assert bool(c.out[:new, cols].isnan().all())
    assert torch.equal(c.out[new], other) and bool((c.out[c.total:] == 3.0).all())


@pytest.mark.parametrize("act", ["f16", "bf16"])
@pytest.mark.parametrize("L", [40, 9000])
@pytest.mark.parametrize("large", [0, 1])
def test_some_scores_minus_infinity(dev, act, L, large):  # noqa: F811
    """One plane of q: keys that score -inf have weight zero, and rows keep the values of the other keys."""
    hd, new = 128, 20
    c = _case(dev, act, hd, L, new, large)
    c.q[:new].abs_().clamp_(min=0.1)
    bad = torch.arange(0, L, 3, device=dev)
    bad = bad[bad < L - new]                    # every token keeps a key
    c.kp[c.rows[0][bad]] = float("-inf")
    c.run()
    assert _status() == 0
    # the same softmax without them: they all lie before the new tokens, so what each token sees of the rest stays
    keep = torch.ones(L, dtype=torch.bool, device=dev)
    keep[bad] = False
    c.rows[0], c.lens[0] = c.rows[0][keep], int(keep.sum())
    c.check()


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("L", [17, 129, 9000])
@pytest.mark.parametrize("new,large", FORMS)
@pytest.mark.parametrize("what", ["q", "q element", "last key", "key 5", "+inf key", "v"])
def test_nan_reaches_the_tokens_that_see_it(dev, act, L, new, large, what):  # noqa: F811
    hd = 128
    c = _case(dev, act, hd, L, new, large)
    c.run()
    assert _status() == 0
    other = c.out[new].clone()
    L = c.lens[0]
    c.out.fill_(3.0)
    cols = slice(0, 8 * hd)
    if what == "q":
        c.q[new - 1] = float("nan")
    elif what == "q element":
        c.q[new - 1, 3 * hd + 7] = float("nan")
        cols = slice(3 * hd, 4 * hd)
    elif what == "last key":
        c.kp[c.rows[0][L - 1]] = float("nan")
    elif what == "key 5":
        c.kp[c.rows[0][5]] = float("nan")
    elif what == "+inf key":
        c.q[:new] = 1.0
        c.kp[c.rows[0][5]] = float("inf")
    else:
        c.vp[c.rows[0][5]] = float("nan")
    c.run()
    assert _status() == 0
    assert bool(c.out[new - 1, cols].isnan().all())
    assert torch.equal(c.out[new], other) and bool((c.out[c.total:] == 3.0).all())


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new,large", FORMS)
def test_gate_far_out(dev, act, hd, new, large):  # noqa: F811
    """Gates where the exponential passes fp32, up to the infinities: 0 and 1."""
    c = _case(dev, act, hd, 300, new, large, gate=True)
    vals = torch.tensor([-1e4, -200.0, -104.0, -89.0, -88.0, -20.0, 20.0, 89.0, 200.0, 1e4, float("inf"), float("-inf")], device=dev)
    c.gate.copy_(vals[torch.arange(c.gate.numel(), device=dev) % len(vals)].view(c.gate.shape))
    c.run()
    assert _status() == 0
    want, bar = c.want(new == 1)
    got = c.out[:c.total, :8 * hd].double()
    # (__expf is 2 + 1.2 |x| ulp off: at 20 that is 2^-19 of e^-20, at -104 2^-17 of a sigmoid below 2^-126)
    assert bool(((got - want).abs() <= bar + want.abs() * 2.0 ** -16 + 2.0 ** -126).all())
