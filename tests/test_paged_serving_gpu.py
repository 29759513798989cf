"""A serving run through the paged cache -- page step, QK-norm + RoPE + store, attention, over layers and steps -- with
requests that come, grow in chunks and single tokens, and end, against plain 64-bit forms on contiguous histories."""
import numpy as np
import pytest
import torch

import paged_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    torch.cuda.set_device(0)
    return torch.device("cuda:0")


H, KV, HD, PAGE, LAYERS, SEATS, CAP = 8, 2, 64, 16, 2, 5, 96
# per step: new tokens of each seat (-1: the request ends; a seat at length 0 that gets tokens is a new request)
STEPS = [[40, 0, 17, 1, 0], [1, 30, 1, 1, 0], [1, 1, -1, 20, 16], [1, 1, 50, 1, 1], [-1, 1, 1, 1, 1], [33, 1, 1, -1, 1],
         [1, 1, 1, 0, 1]]


def _buffers(dev, n_pages):
    e = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)
    b = dict(tables=torch.full((SEATS, 12), -1, dtype=torch.int32, device=dev),
             ring=torch.arange(n_pages, dtype=torch.int32, device=dev).flip(0).contiguous(),
             kv=[e(SEATS), e(SEATS)], state=[e(4), e(4)], new=e(SEATS), cu=e(SEATS + 1), slots=e(CAP), pos=e(CAP),
             q=torch.zeros(LAYERS, CAP, H * HD, device=dev), k=torch.zeros(LAYERS, CAP, KV * HD, device=dev),
             v=torch.zeros(LAYERS, CAP, KV * HD, device=dev), qr=torch.zeros(LAYERS, CAP, H * HD, device=dev),
             out=torch.full((LAYERS, CAP, H * HD), 5.0, device=dev))
    b["state"][0][1] = n_pages
    b["pools"] = [tuple(torch.full((n_pages, PAGE, KV * HD), float("nan"), dtype=torch.float16, device=dev)
                        for _ in range(2)) for _ in range(LAYERS)]
    b["w"] = 1 + 0.1 * torch.randn(2, HD, device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    return b


def _step(b, a, max_new):
    """The calls of one serving step, from length buffers a to 1 - a."""
    from yllm_b200 import attn
    attn.page_step(b["kv"][1 - a], b["cu"], b["slots"], b["pos"], b["state"][1 - a], b["tables"], b["ring"],
                   b["state"][a], b["kv"][a], b["new"], PAGE)
    norm = attn.qk_norm(b["w"][0], b["w"][1], 1e-6)
    for i, (kp, vp) in enumerate(b["pools"]):
        attn.rope_store_kv_paged(b["qr"][i], b["q"][i], b["k"][i], b["v"][i], kp, vp, b["slots"], b["pos"], H, KV, HD,
                                 1, 1e6, norm=norm)
        attn.attn_paged(b["out"][i], b["qr"][i], kp, vp, b["tables"], b["cu"], b["kv"][1 - a], max_new, H, KV, HD)


@pytest.mark.parametrize("captured", [False, True])
def test_serving_run(dev, captured):
    from yllm_b200 import attn
    b = _buffers(dev, 40)
    if captured:
        _step(b, 0, CAP)             # first calls outside the capture, on lengths of zero
        torch.cuda.synchronize()
        b = _buffers(dev, 40)
        graphs = []
        for a in (0, 1):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                _step(b, a, CAP)
            graphs.append(g)
    rng = np.random.default_rng(12)
    hist = [[(np.zeros((0, KV * HD)), np.zeros((0, KV * HD))) for _ in range(SEATS)] for _ in range(LAYERS)]
    lens = [0] * SEATS
    w = b["w"].double().cpu().numpy()
    for n, new in enumerate(STEPS):
        total = sum(max(m, 0) for m in new)
        x = {name: rng.standard_normal((LAYERS, CAP, cols)).astype(np.float32)
             for name, cols in (("q", H * HD), ("k", KV * HD), ("v", KV * HD))}
        for name in x:
            b[name].copy_(torch.from_numpy(x[name]))
        b["new"].copy_(torch.tensor(new, dtype=torch.int32))
        b["out"].fill_(5.0)
        if captured:
            graphs[n % 2].replay()
        else:
            _step(b, n % 2, max(1, max(new)))
        torch.cuda.synchronize()
        assert attn.device_status() == 0
        state = b["state"][1 - n % 2].tolist()
        assert state[2:] == [0, total]
        at = 0
        for r, m in enumerate(new):
            if m < 0:
                lens[r] = 0
                for i in range(LAYERS):
                    hist[i][r] = (np.zeros((0, KV * HD)), np.zeros((0, KV * HD)))
                continue
            pos = np.arange(lens[r], lens[r] + m)
            lens[r] += m
            for i in range(LAYERS):
                rows = slice(at, at + m)
                # K as the cache holds it: the 64-bit value rounded to fp16 (the stored one is within a step of it)
                k = paged_ref.rope_rows(x["k"][i][rows], pos, KV, HD, 1, HD, 1e6, w[1], 1e-6)
                kc, vc = hist[i][r]
                kc, vc = np.concatenate([kc, k.astype(np.float16)]), np.concatenate([vc, x["v"][i][rows].astype(np.float16)])
                hist[i][r] = (kc, vc)
                if m == 0:
                    continue
                q = paged_ref.rope_rows(x["q"][i][rows], pos, H, HD, 1, HD, 1e6, w[0], 1e-6)
                t = np.arange(-(-lens[r] // PAGE))[None]
                pad = np.zeros((t.size * PAGE, KV * HD))
                kk, vv = pad.copy(), pad.copy()
                kk[:lens[r]], vv[:lens[r]] = kc, vc
                want = paged_ref.attn(q, kk, vv, t, [0, m], [lens[r]], PAGE, H, KV, HD)
                got = b["out"][i][rows].double().cpu().numpy()
                # a K or V element differs by at most a step of fp16 (2^-10 of it) where the two roundings fall on
                # either side of a tie: scores move by 2^-10 * sum |q k| / 8 at most, here under 2^-10 * 12, for few
                # elements; measured against |v| <= 5 that bounds the output's error by 2 * 0.012 * 5 and, as a mean over
                # the elements, far below it
                assert np.abs(got - want).max() < 0.12 and np.sqrt(np.mean((got - want) ** 2)) < 2e-4
            at += m
        assert bool((b["out"][:, total:] == 5.0).all())
        assert b["kv"][1 - n % 2].tolist() == lens
    held = sum(-(-x // PAGE) for x in lens)
    assert state[1] == 40 - held


def test_a_step_without_room_changes_nothing(dev):
    """The page step denies the whole step: the store and the attention that read its slots and offsets do nothing."""
    b = _buffers(dev, 4)
    b["new"].copy_(torch.tensor([40, 30, 0, 0, 0], dtype=torch.int32))      # five pages of four
    _step(b, 0, CAP)
    torch.cuda.synchronize()
    assert b["state"][1].tolist() == [0, 4, 1, 0] and b["kv"][1].tolist() == [0] * SEATS
    assert bool((b["out"] == 5.0).all()) and bool((b["qr"] == 0).all())
    assert all(bool(p.isnan().all()) for pools in b["pools"] for p in pools)


def test_paged_matches_contiguous_decode(dev):
    """The same cache rows, paged and contiguous: the paged decode form against the pooled batched decode."""
    from yllm_b200 import attn
    Hh, Kv, hd, page = 32, 8, 128, 16
    lens = [700, 130, 1500]
    g = torch.Generator(device=dev).manual_seed(3)
    caches = [(torch.randn(n, Kv * hd, generator=g, device=dev).half(), torch.randn(n, Kv * hd, generator=g, device=dev).half())
              for n in lens]
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need), generator=torch.Generator().manual_seed(4)).to(torch.int32)
    kp, vp = (torch.zeros(sum(need), page, Kv * hd, dtype=torch.float16, device=dev) for _ in range(2))
    tables = torch.zeros(3, max(need), dtype=torch.int32)
    at = 0
    for r, m in enumerate(need):
        tables[r, :m] = order[at:at + m]
        at += m
        t = torch.arange(lens[r])
        rows = (tables[r, t // page].long() * page + t % page).to(dev)
        kp.view(-1, Kv * hd)[rows], vp.view(-1, Kv * hd)[rows] = caches[r]
    q = torch.randn(3, Hh * hd, generator=g, device=dev)
    out, ref = torch.empty_like(q), torch.empty_like(q)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    attn.attn_paged(out, q, kp, vp, tables.to(dev), i32([0, 1, 2, 3]), i32(lens), 1, Hh, Kv, hd)
    for r, n in enumerate(lens):
        k, v = (x.view(torch.int16).view(torch.uint16).contiguous() for x in caches[r])
        attn.attn_decode(ref[r], q[r], k, v, n - 1, Hh, Kv, hd, Kv * hd)
    torch.cuda.synchronize()
    # both carry about 22 bits of q and p: each is within 2e-6 of the exact result on values of at most about 1
    assert float((out - ref).abs().max()) < 4e-6
