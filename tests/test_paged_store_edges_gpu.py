"""The paged QK-norm + RoPE + KV store at the edges of its values."""
import numpy as np
import pytest
import torch

import paged_ref
from test_paged_step_store_gpu import DT, _i32, _pair_norm, dev  # noqa: F401  (dev is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("hd,kind,n_dims", [(64, 0, 0), (128, 1, 0), (256, 2, 64)])
def test_norm_of_very_large_and_zero_heads(dev, act, hd, kind, n_dims):  # noqa: F811
    """A head whose sum of squares passes fp32 comes out as zeros (1 / sqrt(inf) is 0), a zero head as zeros, and their
    neighbours hold the plain form's bar."""
    from yllm_b200 import attn
    H, KV, T, theta, eps = 5, 3, 7, 1e4, 1e-6
    g = torch.Generator(device=dev).manual_seed(hd)
    q, k, v = (torch.randn(T, m, hd, generator=g, device=dev) for m in (H, KV, KV))
    q[1, 2] *= 1e20
    q[3, 0] = 1e19                       # squares of 1e38, whose sum is past fp32
    q[4, 4] = 0
    q[5, 1, :] = 0
    q[5, 1, 7] = 3e38
    k[2, 1] *= -1e25
    k[6, 2] = 0
    q, k, v = (x.reshape(T, -1).to(DT[act]) for x in (q, k, v))
    w = 1 + 0.3 * torch.randn(2, hd, generator=g, device=dev)
    kp, vp = (torch.zeros(1, 16, KV * hd, dtype=torch.float16, device=dev) for _ in range(2))
    out = torch.full_like(q, 7.0)
    pos, slots = np.arange(T) * 100 + 3, np.arange(T) + 5
    attn.rope_store_kv_paged(out, q, k, v, kp, vp, _i32(slots, dev), _i32(pos, dev), H, KV, hd, kind, theta,
                             n_rope_dims=n_dims, norm=attn.qk_norm(w[0], w[1], eps))
    torch.cuda.synchronize()
    assert attn.device_status() == 0
    zeros_q, zeros_k = [(1, 2), (3, 0), (4, 4), (5, 1)], [(2, 1), (6, 2)]
    got_q = out.double().cpu().numpy().reshape(T, H, hd)
    got_k = kp.view(16, KV, hd)[5:5 + T].double().cpu().numpy()
    n = n_dims if kind == 2 else hd
    for got, x, heads, zeros, wt, step in ((got_q, q, H, zeros_q, w[0], torch.finfo(DT[act]).eps / 2),
                                           (got_k, k, KV, zeros_k, w[1], 2.0 ** -11)):
        want = paged_ref.rope_rows(x.double().cpu().numpy(), pos, heads, hd, kind, n, theta, wt.double().cpu().numpy(), eps)
        bar = 2.0 ** -19 * _pair_norm(want, heads, hd, kind, n) + step * np.abs(want) + 2.0 ** -25
        want, bar = want.reshape(T, heads, hd), bar.reshape(T, heads, hd)
        for z in zeros:
            assert (got[z] == 0).all(), z
            want[z] = bar[z] = 0
        assert (np.abs(got - want) <= bar).all()
