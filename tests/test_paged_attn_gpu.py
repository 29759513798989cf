"""Attention over the paged cache against a plain 64-bit form.

Tolerance, per output element o = sum_s p_s v_s / l with p_s = 2^(s_s - m) <= 1 and l >= 1 (64-bit values below):
  scores  q is a row's power of two times hi + lo fp16 planes: off by 2^-22 of the row's largest |q| (16-bit
          activations in 128-row tiles: one plane, exact down to 2^-25 of it).  With A = max_s sum_d max|q| |k_sd| /
          sqrt(hd), a product of hd terms accumulated in fp32 adds hd 2^-24 A, and scale, subtraction of m and the
          power of two's argument 4 * 2^-24 * 1.45 A: ds = A (2^-22 + 2^-25 + hd 2^-24 + 2^-21).
  p       relative 2^-22 from ex2.approx and 2^-22 from the hi + lo planes (one plane: 2^-11, the half step of fp16);
          p is scaled to 2^7 or more at the row's largest, so the planes' subnormals leave 2^-32 absolute.
  sums    L keys in steps of 16: (L/16 + 16) 2^-24 relative to sum p |v|, and pieces' merges 2^-20.
So |err| <= V (2 ds + e_p + (L/16) 2^-24 + 2^-20) + 2^-32 sum |v| / l, with V = sum p |v| / l, and a half
step of the output's type.  A gate's sigmoid (__expf, 2^-20 relative here) multiplies all of it."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ROWS = 8   # query rows per kv head that the decode form takes


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    torch.cuda.set_device(0)
    return torch.device("cuda:0")


class Case:
    """Random pages, tables and tokens; rows of the pages that no request owns are NaN."""

    def __init__(self, dev, H, KV, hd, page, lens, new, act="f32", gate=False, seed=0, pad=0, kv_extra=0, q_scale=1.0,
                 stride_extra=0, width_extra=2):
        self.geo = (H, KV, hd)
        self.page, self.lens, self.new = page, [int(x) for x in lens], [int(x) for x in new]
        g = torch.Generator(device=dev).manual_seed(seed)
        rng = np.random.default_rng(seed)
        need = [-(-x // page) for x in self.lens]
        n_pages = sum(need) + 3
        kd = KV * hd + kv_extra
        order = rng.permutation(n_pages)
        width = max(need + [1]) + width_extra
        tab = rng.integers(-5, 2 ** 31 - 1, (len(lens), width)).astype(np.int32)   # entries past a request: junk
        owned = np.zeros(n_pages * page, bool)
        at = 0
        self.rows = []
        for r, m in enumerate(need):
            tab[r, :m] = order[at:at + m]
            t = np.arange(self.lens[r])
            rows = tab[r, t // page].astype(np.int64) * page + t % page
            owned[rows] = True
            self.rows.append(torch.from_numpy(rows).to(dev))
            at += m
        self.tables = torch.from_numpy(tab).to(dev)
        owned = torch.from_numpy(owned).to(dev)
        self.kp, self.vp = (torch.randn(n_pages * page, kd, generator=g, device=dev).half() for _ in range(2))
        self.kp[~owned] = float("nan")
        self.vp[~owned] = float("nan")
        self.total = sum(self.new)
        T = self.total + pad
        wide = lambda: torch.randn(T, H * hd + stride_extra, generator=g, device=dev)[:, :H * hd]
        self.q = (wide() * q_scale).to(DT[act]) if not stride_extra else \
            torch.randn(T, H * hd + stride_extra, generator=g, device=dev).to(DT[act])[:, :H * hd]
        self.gate = wide().to(DT[act]) if gate else None
        self.out = torch.full((T, H * hd + 8), 3.0, dtype=DT[act], device=dev)
        self.cu = torch.tensor(np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32), device=dev)
        self.kv = torch.tensor(np.asarray(self.lens, np.int32), device=dev)

    def run(self, max_new=None, out=None, **kw):
        from yllm_b200 import attn
        H, KV, hd = self.geo
        out = self.out if out is None else out
        attn.attn_paged(out[:, :H * hd], self.q, self.kp.view(-1, self.page, self.kp.shape[1]),
                        self.vp.view(-1, self.page, self.vp.shape[1]), self.tables, self.cu, self.kv,
                        max(self.new) if max_new is None else max_new, H, KV, hd, gate=self.gate, **kw)

    def want(self, rows_form):
        """(values, bounds) in 64 bits for the rows of the requests."""
        H, KV, hd = self.geo
        g = H // KV
        one_plane = not rows_form and self.q.dtype != torch.float32
        e_p = 2.0 ** -11 + 2.0 ** -22 if one_plane else 2.0 ** -21
        o = torch.zeros(self.total, H * hd, dtype=torch.float64, device=self.q.device)
        bar = torch.zeros_like(o)
        a = 0
        for r, (L, n) in enumerate(zip(self.lens, self.new)):
            if n and L:
                k = self.kp[self.rows[r]][:, :KV * hd].double().view(L, KV, hd).permute(1, 0, 2)
                v = self.vp[self.rows[r]][:, :KV * hd].double().view(L, KV, hd).permute(1, 0, 2)
                q = self.q[a:a + n].double().reshape(n, KV, g, hd).permute(1, 2, 0, 3)            # KV g n hd
                s = torch.einsum("hgnd,hld->hgnl", q, k) / np.sqrt(hd)
                big = q.abs().amax(-1)                                                             # KV g n
                A = big * (k.abs().sum(-1).amax(-1) / np.sqrt(hd))[:, None, None]
                ds = A * (2.0 ** -22 + 2.0 ** -25 + hd * 2.0 ** -24 + 2.0 ** -21)
                pos = L - n + torch.arange(n, device=s.device)
                seen = torch.arange(L, device=s.device)[None, :] <= pos[:, None]
                s = s.masked_fill(~seen, -np.inf)
                p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
                l = p.sum(-1, keepdim=True).clamp(min=1e-300)
                val = torch.einsum("hgnl,hld->hgnd", p, v) / l
                V = torch.einsum("hgnl,hld->hgnd", p, v.abs()) / l
                tail = torch.einsum("nl,hld->hnd", seen.double(), v.abs())[:, None] / l * 2.0 ** -32
                b = V * (2 * ds[..., None] + e_p + (L / 16 + 16) * 2.0 ** -24 + 2.0 ** -20) + tail
                dead = (pos < 0)[None, None, :, None]
                val, b = val.masked_fill(dead, 0.0), b.masked_fill(dead, 0.0)
                o[a:a + n] = val.permute(2, 0, 1, 3).reshape(n, H * hd)
                bar[a:a + n] = b.permute(2, 0, 1, 3).reshape(n, H * hd)
            a += n
        if self.gate is not None:
            sg = torch.sigmoid(self.gate[:self.total].double())
            bar = bar * sg + (o * sg).abs() * 2.0 ** -20
            o = o * sg
        dt = self.q.dtype
        return o, bar + o.abs() * torch.finfo(dt).eps / 2 + (2.0 ** -25 if dt == torch.float16 else 2.0 ** -126)

    def check(self, out=None, max_new=None):
        torch.cuda.synchronize()
        from yllm_b200 import attn
        assert attn.device_status() == 0
        H, KV, hd = self.geo
        out = self.out if out is None else out
        rows_form = (max(self.new) if max_new is None else max_new) * (H // KV) <= ROWS
        want, bar = self.want(rows_form)
        got = out[:self.total, :H * hd].double()
        err = (got - want).abs()
        assert bool((err <= bar).all()), f"worst {float((err / bar).max()):.3g} of its bar, nan {int(got.isnan().sum())}"
        assert bool((out[self.total:] == 3.0).all()) and bool((out[:, H * hd:] == 3.0).all())


GEO = [(14, 2, 64), (32, 8, 128), (16, 2, 256), (4, 4, 128), (3, 3, 64), (5, 1, 128), (8, 1, 256)]


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,hd", GEO)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_single_tokens(dev, act, H, KV, hd, page):
    """One token per request: lengths of one, around pages and blocks, and long enough to be cut."""
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 1000]
    c = Case(dev, H, KV, hd, page, lens, [1] * len(lens), act=act, gate=(hd == 256), seed=H + hd + page, pad=2,
             kv_extra=16 if H == 32 else 0)
    c.run()
    c.check()


@pytest.mark.parametrize("lens,new", [
    ([5000], [1]), ([70000], [1]), ([0, 0, 9], [0, 0, 1]), ([33, 0, 1, 4097], [1, 0, 1, 1]), ([1], [1]),
])
@pytest.mark.parametrize("H,KV,hd", [(32, 8, 128), (14, 2, 64), (16, 2, 256)])
def test_single_tokens_lengths(dev, lens, new, H, KV, hd):
    c = Case(dev, H, KV, hd, 16, lens, new, seed=sum(lens), pad=1)
    c.run()
    c.check()
    first = c.out.clone()
    for _ in range(3):   # the pieces are merged in one order: the same bits every time
        c.out.fill_(3.0)
        c.run()
        assert torch.equal(c.out, first)


@pytest.mark.parametrize("n", [400, 1000])
def test_many_requests(dev, n):
    rng = np.random.default_rng(n)
    lens = rng.integers(0, 150, n)
    new = (rng.random(n) < 0.7).astype(int) * (lens > 0)
    c = Case(dev, 8, 2, 64, 16, lens, new, seed=n)
    c.run()
    c.check()


@pytest.mark.parametrize("H,KV,hd,new", [(8, 4, 128, [4, 1, 3, 2]), (4, 4, 64, [8, 5, 1, 0]), (2, 1, 256, [4, 4, 2, 1])])
def test_few_tokens_rows_form(dev, H, KV, hd, new):
    """Several tokens per request with at most 8 rows per kv head: each row has its own last key."""
    c = Case(dev, H, KV, hd, 32, [4, 700, 65, 2000], new, act="f32", seed=hd)
    c.run()
    c.check()


def test_token_with_no_key_gets_zeros(dev):
    """kv_len < new: the first tokens see nothing."""
    c = Case(dev, 4, 4, 64, 16, [2, 0, 5], [4, 3, 2], seed=9)
    c.run()
    c.check()
    assert bool((c.out[:2, :256] == 0).all()) and bool((c.out[4:7, :256] == 0).all())


@pytest.mark.parametrize("scale", [2.0 ** 20, 2.0 ** -30])
def test_rows_form_far_q(dev, scale):
    """q far outside fp16's range."""
    c = Case(dev, 8, 2, 128, 16, [50, 333], [1, 1], seed=4, q_scale=scale)
    c.run()
    c.check()


# ------------------------------------------------------------- 128-row tiles

@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,hd", GEO)
@pytest.mark.parametrize("page", [16, 128])
def test_chunks(dev, act, H, KV, hd, page):
    """Chunks of odd sizes beside single tokens and requests without any, from an empty cache and behind one."""
    lens = [40, 1, 129, 700, 0, 65, 257, 300]
    new = [40, 1, 130 - 1, 33, 0, 1, 2, 100]
    c = Case(dev, H, KV, hd, page, lens, new, act=act, gate=(hd == 256), seed=H + hd + page, pad=3,
             stride_extra=16 if page == 128 else 0)
    c.run()
    c.check()


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("lens,new", [
    ([9], [9]), ([128], [128]), ([1000], [1000]), ([5000], [16]), ([40000], [33]), ([17, 16, 15], [17, 16, 15]),
    ([3, 0, 40], [60, 20, 40]), ([2500, 31, 1], [70, 31, 1]),
])
@pytest.mark.parametrize("H,KV,hd", [(32, 8, 128), (14, 2, 64), (16, 2, 256)])
def test_chunks_lengths(dev, act, lens, new, H, KV, hd):
    """One request to a few: tiles cut over many CTAs, and tokens that see no key (kv_len < new)."""
    c = Case(dev, H, KV, hd, 16, lens, new, act=act, seed=sum(lens) + hd, pad=1)
    c.run()
    c.check()
    first = c.out.clone()
    for _ in range(3):
        c.out.fill_(3.0)
        c.run()
        assert torch.equal(c.out, first)


def test_chunks_many_requests(dev):
    rng = np.random.default_rng(8)
    n = 500
    new = np.where(rng.random(n) < 0.1, rng.integers(0, 60, n), 1)
    lens = new + rng.integers(0, 200, n)
    c = Case(dev, 8, 2, 128, 32, lens, new, seed=8)
    c.run()
    c.check()


def test_wide_group_single_tokens(dev):
    """16 heads per kv head: a single token does not fit the decode form."""
    c = Case(dev, 32, 2, 128, 16, [1, 16, 777, 3000], [1, 1, 1, 1], seed=2)
    c.run()
    c.check()


@pytest.mark.parametrize("act,scale", [("f32", 2.0 ** 20), ("f32", 2.0 ** -30), ("bf16", 2.0 ** 20)])
def test_tiles_far_q(dev, act, scale):
    c = Case(dev, 8, 2, 128, 16, [50, 333], [20, 100], act=act, seed=4, q_scale=scale)
    c.run()
    c.check()


def test_tiles_small_bf16_q_large_keys(dev):
    """bf16 q under fp16's normal range, halfway between two of its subnormals, against keys near fp16's largest: a
    plain conversion of q would be off by 2^-5 of it, scores of 0.67 by 0.02 and the outputs by 0.01."""
    c = Case(dev, 8, 2, 128, 16, [200, 130], [100, 130], "bf16", seed=19)
    c.q.fill_(2.0 ** -20 + 2.0 ** -25)
    c.q[::3] *= -1
    for rows in c.rows:
        sign = torch.where(torch.arange(len(rows), device=dev) % 2 == 0, 1.0, -1.0).half()[:, None]
        c.kp[rows] = (60000 * sign).expand(-1, c.kp.shape[1])
        c.vp[rows] = sign.expand(-1, c.vp.shape[1]).contiguous()
    c.run()
    c.check()


@pytest.mark.parametrize("H,KV,hd", [(8, 2, 128), (3, 3, 64), (14, 2, 64), (32, 2, 128)])
@pytest.mark.parametrize("gate", [False, True])
def test_few_rows_beside_many(dev, H, KV, hd, gate):
    """fp32 requests around half a tile of query rows, whole and cut over many CTAs, with rows that see no key and with
    q far outside fp16's range."""
    g = H // KV
    new = [64 // g, 64 // g + 1, 1, 64 // g - 1, 0, 65, 64 // g, 2, 9]
    lens = [64 // g, 700, 130, 3 * 128, 50, 300, 9000, 1, 20001]
    c = Case(dev, H, KV, hd, 16, lens, new, gate=gate, seed=H + hd, pad=2, q_scale=2.0 ** -20 if gate else 1.0)
    c.run(max_new=128)
    c.check(max_new=128)


@pytest.mark.parametrize("H,KV,hd,gate", [(14, 2, 64, False), (32, 8, 128, True), (16, 2, 256, False), (5, 5, 64, True)])
@pytest.mark.parametrize("page", [16, 128])
def test_mixed_batch_in_two_launches(dev, H, KV, hd, gate, page):
    """fp32, as many requests as make a kv head of one per SM: single tokens and small requests around 8 query rows
    per kv head beside chunks, requests without tokens, without keys, and with fewer keys than tokens."""
    rng = np.random.default_rng(H + page)
    n = -(-torch.cuda.get_device_properties(0).multi_processor_count // KV) + 3
    few = 8 // (H // KV)
    new = rng.choice([0, 1, 1, 1, 1, max(few, 1), few + 1], n)
    new[[1, n // 2]] = 150, 333
    lens = new + rng.integers(0, 700, n)
    lens[[0, 2, 5]] = 0, new[2], max(int(new[5]) - 1, 0)
    lens[1] = 100
    assert int(new.sum()) * 4 <= n * 333
    c = Case(dev, H, KV, hd, page, lens, new, gate=gate, seed=H + hd + page, pad=2)
    c.run()
    c.check()
    first = c.out.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run()
    for _ in range(3):
        c.out.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.out, first)


def test_mixed_batch_in_two_launches_skips_a_bad_request(dev):
    """A request longer than its table: reported, its rows not written, the others right."""
    from yllm_b200 import attn
    n = torch.cuda.get_device_properties(0).multi_processor_count
    new = [1] * n
    new[7], new[20] = 200, 60
    lens = [100 + i for i in range(n)]
    lens[7] = 300
    c = Case(dev, 8, 2, 128, 16, lens, new, seed=77)
    at = np.concatenate([[0], np.cumsum(new)])
    for bad in (3, 20):
        c.kv[bad] = c.tables.shape[1] * 16 + 1
    c.run()
    torch.cuda.synchronize()
    assert attn.device_status() == 603
    want, bar = c.want(False)
    err = (c.out[:c.total, :1024].double() - want).abs()
    for r in range(n):
        part = slice(at[r], at[r + 1])
        if r in (3, 20):
            assert bool((c.out[part] == 3.0).all())
        else:
            assert bool((err[part] <= bar[part]).all()), r


def many_rows(H):
    """Rows of q behind the last request that make a call large enough for two CTAs per SM (a tile per SM)."""
    return -(-torch.cuda.get_device_properties(0).multi_processor_count * 128 // H)


@pytest.mark.parametrize("act", ["f16", "bf16"])
@pytest.mark.parametrize("H,KV,hd", [x for x in GEO if x[2] <= 128])
@pytest.mark.parametrize("page,gate", [(16, False), (128, True), (256, False)])
def test_large_calls_chunks(dev, act, H, KV, hd, page, gate):
    """Two CTAs per SM: chunks of odd sizes, single tokens, requests without tokens or keys; padded rows stay."""
    lens = [40, 1, 129, 700, 0, 65, 257, 300, 20]
    new = [40, 1, 129, 33, 0, 1, 2, 100, 70]
    c = Case(dev, H, KV, hd, page, lens, new, act=act, gate=gate, seed=H + hd + page, pad=many_rows(H),
             stride_extra=16 if page == 128 else 0)
    c.run()
    c.check()


@pytest.mark.parametrize("act", ["f16", "bf16"])
@pytest.mark.parametrize("lens,new", [
    ([9], [9]), ([64], [64]), ([1000], [1000]), ([40000], [33]), ([17, 16, 15], [17, 16, 15]), ([3, 0, 40], [60, 20, 40]),
    ([2500, 31, 1], [70, 31, 1]), ([1500, 900, 700], [700, 900, 65]),
])
@pytest.mark.parametrize("H,KV,hd", [(32, 8, 128), (14, 2, 64)])
def test_large_calls_lengths(dev, act, lens, new, H, KV, hd):
    c = Case(dev, H, KV, hd, 16, lens, new, act=act, seed=sum(lens) + hd, pad=many_rows(H))
    c.run()
    c.check()
    first = c.out.clone()
    for _ in range(3):
        c.out.fill_(3.0)
        c.run()
        assert torch.equal(c.out, first)


def test_large_calls_share_the_gpu(dev):
    """Calls of every form in flight at once on streams of their own, eager and replayed."""
    mk = lambda act, hd, pad, i: Case(dev, 8, 2, hd, 16, [3000 + 77 * i, 400], [300, 70], act=act, seed=50 + i, pad=pad)
    cases = [mk("bf16", 128, many_rows(8), 0), mk("f16", 64, many_rows(8), 1), mk("f32", 128, 0, 2), mk("bf16", 256, 0, 3),
             Case(dev, 32, 8, 128, 16, [20000], [1], seed=54)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for c, s in zip(cases, streams):
        c.run(stream=s)
    torch.cuda.synchronize()
    graphs = []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.run()
        graphs.append(g)
        c.out.fill_(3.0)
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for c in cases:
        c.check()


# ------------------------------------------------------- what the calls refuse or report

def test_bad_page_reads_as_zeros_and_is_reported(dev):
    """A block table entry outside the pool: status 602, and the other requests are untouched by it."""
    from yllm_b200 import attn
    for new in ([1, 1], [40, 30]):
        c = Case(dev, 8, 2, 64, 16, [100, 90], new, seed=6)
        c.run()
        torch.cuda.synchronize()
        good = c.out.clone()
        for entry in (-1, 1 << 20, 2 ** 31 - 1, c.kp.shape[0] // 16):
            c.tables[0, 2] = entry
            c.run()
            torch.cuda.synchronize()
            assert attn.device_status() == 602
            assert torch.equal(c.out[new[0]:], good[new[0]:]) and bool(c.out[:new[0]].isfinite().all())


@pytest.mark.parametrize("new", [[1, 1, 1], [30, 1, 40]])
@pytest.mark.parametrize("what", ["cu falls", "cu past the rows", "negative length", "length past the table", "max_new"])
def test_contradicting_request_is_skipped_and_reported(dev, what, new):
    from yllm_b200 import attn
    c = Case(dev, 8, 2, 64, 16, [100, 90, 80], new, seed=7)
    want, bar = c.want(max(new) * 4 <= ROWS)
    kw = {}
    skipped = 2
    if what == "cu falls":
        c.cu[3] = int(c.cu[2]) - 1
    elif what == "cu past the rows":
        c.cu[3] = c.q.shape[0] + 1
    elif what == "negative length":
        c.kv[2] = -5
    elif what == "length past the table":
        c.kv[2] = c.tables.shape[1] * 16 + 1
    else:
        if new[2] == 1:
            return
        kw["max_new"] = new[2] - 1     # still the tiles form
    c.run(**kw)
    torch.cuda.synchronize()
    assert attn.device_status() == 603
    a, b = sum(new[:skipped]), sum(new)
    # (the others hold their bars; not bit for bit, as the work is divided anew without it)
    assert bool(((c.out[:a, :512].double() - want[:a]).abs() <= bar[:a]).all()) and bool((c.out[a:b] == 3.0).all())
    c.run(max_new=64)      # nothing of it lingers (its own lengths are still wrong for four of them)
    attn.device_status()


def test_rows_form_refuses_more_tokens_than_announced(dev):
    from yllm_b200 import attn
    c = Case(dev, 8, 2, 128, 16, [64, 200], [1, 3], seed=8)
    c.run(max_new=1)
    torch.cuda.synchronize()
    assert attn.device_status() == 603 and bool((c.out[1:, :8 * 128] == 3.0).all())
    c.run(max_new=3)
    c.check(max_new=3)


# ------------------------------------------------------------- streams, graphs, workspaces

def test_two_streams_at_once(dev):
    """Each stream has its own workspace: cut units of two calls in flight do not meet."""
    cases = [Case(dev, 32, 8, 128, 16, [20000 + 777 * i], [1], seed=20 + i) for i in range(2)]
    cases += [Case(dev, 8, 2, 128, 16, [9000 + 77 * i], [70], seed=30 + i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        for c, s in zip(cases, streams):
            c.run(stream=s)
    torch.cuda.synchronize()
    for c in cases:
        c.check()


def test_capture_and_replay_with_other_lengths(dev):
    """Lengths and tables are read at replay: one graph serves growing requests.  Two graphs replayed at once on two
    streams have workspaces of their own."""
    from yllm_b200 import attn
    H, KV, hd, page = 8, 2, 128, 16
    big = [Case(dev, H, KV, hd, page, [6000, 50, 3000], [1, 1, 1], seed=40), Case(dev, H, KV, hd, page, [5000, 40, 300], [60, 1, 7], seed=41)]
    for c in big:
        c.run()
    torch.cuda.synchronize()
    graphs = []
    for c in big:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.run()
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in big]
    for cut in (0, 17, 2900):
        for c in big:
            c.out.fill_(3.0)
        for c in big:     # shorter caches, other lengths per replay
            lens = [max(x - cut, n) for x, n in zip(c.full if hasattr(c, "full") else c.lens, c.new)]
            c.full = c.full if hasattr(c, "full") else list(c.lens)
            c.kv.copy_(torch.tensor(lens, dtype=torch.int32))
            c.rows = [r[:n] for r, n in zip(c.rows_full, lens)] if hasattr(c, "rows_full") else c.rows
            if not hasattr(c, "rows_full"):
                c.rows_full = list(c.rows)
            c.rows = [r[:n] for r, n in zip(c.rows_full, lens)]
            c.lens = lens
        torch.cuda.synchronize()
        for _ in range(3):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for c in big:
            c.check()
    assert attn.device_status() == 0


def test_own_workspace(dev):
    from yllm_b200 import attn
    c = Case(dev, 32, 8, 128, 64, [30000], [1], seed=50)
    ws = attn.paged_workspace(128)
    c.run(workspace=ws)
    c.check()
    assert bool((ws[:4096] == 0).all())      # the call leaves the counters zero
    with pytest.raises(attn._lib.YattnError, match="workspace"):
        c.run(workspace=ws[:4096])
    with pytest.raises(ValueError, match="workspace"):
        c.run(workspace=ws.cpu())


def test_wrapper_checks(dev):
    from yllm_b200 import attn
    c = Case(dev, 8, 2, 64, 16, [20, 30], [1, 1], seed=51)
    k, v = c.kp.view(-1, 16, 128), c.vp.view(-1, 16, 128)
    good = dict(out=c.out[:, :512], q=c.q, kpool=k, vpool=v, tables=c.tables, cu_new=c.cu, kv_len=c.kv, max_new=1,
                n_heads=8, n_kv_heads=2, head_dim=64)
    for change, word in [
        (dict(q=c.q.double()), "float32"), (dict(q=c.q.cpu()), "CUDA"), (dict(out=c.out[:1, :512]), "out"),
        (dict(out=c.out[:, :512].half()), "out"), (dict(kpool=k.float()), "pool"), (dict(vpool=v[:1]), "pool"),
        (dict(kpool=k[:, ::2]), "pool"), (dict(n_kv_heads=4, n_heads=8), "shorter"), (dict(tables=c.tables[:1]), "tables"),
        (dict(tables=c.tables.long()), "tables"), (dict(tables=c.tables.t()), "tables"), (dict(cu_new=c.cu[:2]), "cu_new"),
        (dict(cu_new=c.cu.long()), "cu_new"), (dict(gate=c.q[:1]), "gate"), (dict(kv_len=c.kv.cpu()), "kv_len"),
    ]:
        with pytest.raises(ValueError, match=word):
            attn.attn_paged(**dict(good, **change))
    attn.attn_paged(**dict(good, q=c.q[:0], out=c.out[:0, :512]))      # no tokens: nothing to do


def test_pool_past_32_bits(dev):
    """Pages whose elements lie beyond 2^32 of the pool's base."""
    from yllm_b200 import attn
    H, KV, hd, page = 16, 8, 128, 64
    n_pages = (2 ** 32 // (KV * hd) + 4096) // page        # 4.3 G elements a pool
    kp, vp = (torch.empty(n_pages, page, KV * hd, dtype=torch.float16, device=dev) for _ in range(2))
    L = 300
    pages = torch.tensor([n_pages - 1, 3, n_pages - 2, 0, n_pages - 3], dtype=torch.int32, device=dev)
    kp[pages.long()] = torch.randn(5, page, KV * hd, device=dev).half()
    vp[pages.long()] = torch.randn(5, page, KV * hd, device=dev).half()
    T = 40
    q, k, v = (torch.randn(T, m * hd, device=dev) for m in (H, KV, KV))
    pos = torch.arange(L - T, L, dtype=torch.int32, device=dev)
    slots = (pages[(pos // page).long()] * page + pos % page).to(torch.int32)
    qo, out, one = torch.empty_like(q), torch.empty_like(q), torch.empty_like(q[:1])
    attn.rope_store_kv_paged(qo, q, k, v, kp, vp, slots, pos, H, KV, hd, 1, 1e6)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    attn.attn_paged(out, qo, kp, vp, pages[None], i32([0, T]), i32([L]), T, H, KV, hd)
    attn.attn_paged(one, qo[-1:].contiguous(), kp, vp, pages[None], i32([0, 1]), i32([L]), 1, H, KV, hd)
    torch.cuda.synchronize()
    kk, vv = kp[pages.long()].view(-1, KV, hd)[:L].double(), vp[pages.long()].view(-1, KV, hd)[:L].double()
    assert bool((vv[L - T:].float() - v.view(T, KV, hd)).abs().max() <= 2.0 ** -11 * v.abs().max())
    qq = qo.double().view(T, KV, H // KV, hd)
    s = torch.einsum("tkgd,lkd->tkgl", qq, kk) / hd ** 0.5
    s = s.masked_fill(torch.arange(L, device=dev)[None, None, None] > pos.long()[:, None, None, None], -np.inf)
    want = torch.einsum("tkgl,lkd->tkgd", torch.softmax(s, -1), vv).reshape(T, H * hd)
    assert float((out.double() - want).abs().max()) < 2e-5 and float((one.double() - want[-1:]).abs().max()) < 2e-5
