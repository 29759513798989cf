"""The paged-cache operators as one serving step uses them, with their plain forms.

Three operators: the page step (block tables and slot maps from request lengths), the QK-norm + RoPE + KV store
into pages, and the attention of new tokens over the pages.  run(state) computes them with elementary torch
operations, or (own = True) through the library's entry points."""
from __future__ import annotations

import math

import torch

own = False

# name: (query heads, KV heads, head dim, rope kind, rotated dims, theta, per-head norms)
SHAPES = {
    "qwen2.5-0.5b": (14, 2, 64, 1, 64, 1e6, False),
    "qwen3-0.6b": (16, 8, 128, 1, 128, 1e6, True),
    "llama3-8b": (32, 8, 128, 0, 128, 5e5, False),
    "qwen3.5": (16, 2, 256, 2, 64, 1e7, True),
}
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # one user's chat: the single sequence grows by its next token
        dict(name="step_1", op="step", n_seqs=1, page=16, len_lo=511, len_hi=511, new_lo=1, new_hi=1, ended=0, spare=0),
        # a decode step of a full batch, two of its requests over
        dict(name="step_64_decode", op="step", n_seqs=64, page=16, len_lo=1024, len_hi=8192, new_lo=1, new_hi=1,
             ended=2, spare=0),
        # a busy server: 512 requests, prompts in chunks beside decoding requests, a padded token buffer
        dict(name="step_512_chunks", op="step", n_seqs=512, page=16, len_lo=0, len_hi=8192, new_lo=1, new_hi=129,
             ended=31, spare=37),
        # the layer's K and V of one decode step, engine fp32 activations
        dict(name="store_64_f32", op="store", shape="llama3-8b", tokens=64, spare=0, page=16, dtype="f32",
             pos_hi=8192),
        # a 2048-token prompt with per-head norms, fp16 activations in one fused projection output
        dict(name="store_2048_norm_f16", op="store", shape="qwen3-0.6b", tokens=2048, spare=0, page=16, dtype="f16",
             pos_hi=40960),
        # 16384 prompt tokens of the hybrid's gated attention layers: 64 of 256 dims rotate
        dict(name="store_16384_partial_bf16", op="store", shape="qwen3.5", tokens=16384, spare=21, page=64,
             dtype="bf16", pos_hi=131072),
        # one user's chat, context 512: latency counts
        dict(name="attn_1x512_f32", op="attn", shape="qwen2.5-0.5b", n_seqs=1, len_lo=511, len_hi=511, chunks=0,
             chunk_lo=1, chunk_hi=1, page=16, dtype="f32", gate=False),
        # a batched decode step, ragged contexts
        dict(name="attn_64x8k_f32", op="attn", shape="llama3-8b", n_seqs=64, len_lo=1024, len_hi=8192, chunks=0,
             chunk_lo=1, chunk_hi=1, page=16, dtype="f32", gate=False),
        # one long context
        dict(name="attn_1x131071_f16", op="attn", shape="llama3-8b", n_seqs=1, len_lo=131070, len_hi=131070, chunks=0,
             chunk_lo=1, chunk_hi=1, page=64, dtype="f16", gate=False),
        # a whole prompt
        dict(name="attn_prompt_2048_f16", op="attn", shape="qwen3-0.6b", n_seqs=1, len_lo=0, len_hi=0, chunks=1,
             chunk_lo=2048, chunk_hi=2048, page=16, dtype="f16", gate=False),
        # prompts in chunks of about 512 beside decoding requests, engine fp32 activations
        dict(name="attn_mixed_f32", op="attn", shape="llama3-8b", n_seqs=32, len_lo=100, len_hi=8192, chunks=4,
             chunk_lo=300, chunk_hi=515, page=16, dtype="f32", gate=False),
        # gated full attention of the hybrid: eight prompts' later chunks
        dict(name="attn_gated_chunks_bf16", op="attn", shape="qwen3.5", n_seqs=8, len_lo=1, len_hi=4096, chunks=8,
             chunk_lo=200, chunk_hi=1000, page=64, dtype="bf16", gate=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["step", "store", "attn", "attn", "attn"])
    page = rng.choice([16, 16, 32, 64, 128, 256])
    if op == "step":
        n = _log(rng, 1, 512)
        lo = _log(rng, 1, 8192) - 1
        return dict(op=op, n_seqs=n, page=page, len_lo=lo, len_hi=rng.randint(lo, 8192), new_lo=rng.randint(0, 1),
                    new_hi=_log(rng, 1, max(1, min(2048, 33000 // n))), ended=rng.randint(0, n // 8),
                    spare=rng.choice([0, rng.randint(1, 99)]))
    shape = rng.choice(sorted(SHAPES))
    dtype = rng.choice(sorted(DT))
    if op == "store":
        return dict(op=op, shape=shape, tokens=_log(rng, 1, 8192), spare=rng.choice([0, rng.randint(1, 99)]),
                    page=page, dtype=dtype, pos_hi=_log(rng, 64, 131072))
    gate = rng.random() < 0.3
    if rng.random() < 0.5:   # single tokens
        n = _log(rng, 1, 64)
        hi = _log(rng, 16, min(131071, 290000 // n))
        return dict(op=op, shape=shape, n_seqs=n, len_lo=rng.randint(0, hi), len_hi=hi, chunks=0, chunk_lo=1,
                    chunk_hi=1, page=page, dtype=dtype, gate=gate)
    n = _log(rng, 1, 24)
    chunks = rng.randint(1, min(n, 4))
    clo = _log(rng, 2, 400)
    hi = _log(rng, 1, 8192)
    return dict(op=op, shape=shape, n_seqs=n, len_lo=rng.randint(0, hi), len_hi=hi, chunks=chunks, chunk_lo=clo,
                chunk_hi=rng.randint(clo, 515), page=page, dtype=dtype, gate=gate)


# ------------------------------------------------------------------ inputs

def _lengths(case, seed):
    """Host lists (cached, new) of a case's requests: the case has its lengths, the seed their order."""
    g = torch.Generator().manual_seed(case["len_hi"] + 17 * case["n_seqs"])

    def ints(lo, hi, n):
        return torch.randint(lo, hi + 1, (n,), generator=g).tolist()

    n = case["n_seqs"]
    cached = ints(case["len_lo"], case["len_hi"], n)
    if case["op"] == "step":
        new = ints(case["new_lo"], case["new_hi"], n)
        for r in torch.randperm(n, generator=g)[:case["ended"]].tolist():
            new[r] = -1
    else:
        new = [1] * n
        sizes = ints(case["chunk_lo"], case["chunk_hi"], case["chunks"])
        for r, c in zip(torch.randperm(n, generator=g)[:case["chunks"]].tolist(), sizes):
            new[r] = c
    order = torch.randperm(n, generator=torch.Generator().manual_seed(seed)).tolist()
    return [cached[r] for r in order], [new[r] for r in order]


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _pages(x, page):
    return -(-x // page)


def _prepare_step(case, seed):
    cached, new = _lengths(case, seed)
    page, n = case["page"], case["n_seqs"]
    held = [_pages(c, page) for c in cached]
    width = max(_pages(c + max(m, 0), page) for c, m in zip(cached, new)) + 3
    grow = sum(_pages(c + max(m, 0), page) - h for c, m, h in zip(cached, new, held))
    n_pages = sum(held) + grow + 5
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(n_pages, generator=g).to(torch.int32)
    tables = torch.full((n, width), -1, dtype=torch.int32)
    at = 0
    for r, h in enumerate(held):
        tables[r, :h] = order[at:at + h]
        at += h
    head, count = seed % n_pages, n_pages - at
    ring = torch.full((n_pages,), -1, dtype=torch.int32)
    ring[(head + torch.arange(count)) % n_pages] = order[at:]
    total = sum(max(m, 0) for m in new)
    cap = total + case["spare"]
    e = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    return dict(op="step", page=page, kv_len=_i32(cached), new_len=_i32(new), tables=tables.cuda(), ring=ring.cuda(),
                state=_i32([head, count, 0, 0]), kv_len_out=e(n), cu_new=e(n + 1), slots=e(cap), positions=e(cap),
                state_out=e(4))


def _prepare_store(case, seed):
    h, kv, hd, kind, rot, theta, norms = SHAPES[case["shape"]]
    page, tokens = case["page"], case["tokens"]
    rows = tokens + case["spare"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn(rows, (h + 2 * kv) * hd, generator=g, device="cuda").to(DT[case["dtype"]])
    n_pages = _pages(tokens, page) + 2
    slots = torch.randperm(n_pages * page, generator=g, device="cuda")[:rows].to(torch.int32)
    positions = torch.randint(0, case["pos_hi"], (rows,), generator=g, device="cuda").to(torch.int32)
    slots[tokens:] = -1          # rows behind the last token of a padded buffer
    positions[tokens:] = 0
    pool = lambda: torch.randn(n_pages, page, kv * hd, generator=g, device="cuda").to(torch.float16)
    s = dict(op="store", shape=case["shape"], qkv=qkv, q=qkv[:, :h * hd], k=qkv[:, h * hd:(h + kv) * hd],
             v=qkv[:, (h + kv) * hd:], slots=slots, positions=positions, kpool=pool(), vpool=pool(),
             q_out=torch.zeros(rows, h * hd, dtype=qkv.dtype, device="cuda"), q_w=None, k_w=None)
    if norms:
        s["q_w"] = 1 + 0.2 * torch.randn(hd, generator=g, device="cuda")
        s["k_w"] = 1 + 0.2 * torch.randn(hd, generator=g, device="cuda")
    return s


def _prepare_attn(case, seed):
    h, kv, hd, *_ = SHAPES[case["shape"]]
    cached, new = _lengths(case, seed)
    page, n = case["page"], case["n_seqs"]
    total = [c + m for c, m in zip(cached, new)]
    need = [_pages(t, page) for t in total]
    n_pages = sum(need) + 3
    g = torch.Generator(device="cuda").manual_seed(seed)
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    tables = torch.full((n, max(need) + 1), -1, dtype=torch.int32, device="cuda")
    pool = lambda: torch.randn(n_pages, page, kv * hd, generator=g, device="cuda", dtype=torch.float16)
    kpool, vpool = pool(), pool()
    at = 0
    for r, m in enumerate(need):
        tables[r, :m] = order[at:at + m]
        at += m
    for r, m in enumerate(need):     # a last page's rows behind its sequence hold whatever was there
        if total[r] % page:
            kpool[order[sum(need[:r + 1]) - 1].long(), total[r] % page:] = float("nan")
            vpool[order[sum(need[:r + 1]) - 1].long(), total[r] % page:] = float("nan")
    rows = sum(new)
    q = torch.randn(rows, h * hd, generator=g, device="cuda").to(DT[case["dtype"]])
    gate = torch.randn(rows, h * hd, generator=g, device="cuda").to(q.dtype) if case["gate"] else None
    cu = [0]
    for m in new:
        cu.append(cu[-1] + m)
    return dict(op="attn", shape=case["shape"], page=page, q=q, gate=gate, out=torch.zeros_like(q), kpool=kpool,
                vpool=vpool, tables=tables, cu_new=_i32(cu), kv_len=_i32(total), cu=cu, total=total,
                max_new=max(new))


def prepare(case, seed):
    return {"step": _prepare_step, "store": _prepare_store, "attn": _prepare_attn}[case["op"]](case, seed)


# ------------------------------------------------------------- plain forms

def _plain_step(s):
    page, kv_len, new = s["page"], s["kv_len"], s["new_len"]
    n, cap, n_pages = kv_len.numel(), s["slots"].numel(), s["ring"].numel()
    ended = new < 0
    m = new.clamp(min=0)
    held = (kv_len + page - 1) // page
    grow = (kv_len + m + page - 1) // page - held
    freed = torch.where(ended, held, torch.zeros_like(held))
    zero = torch.zeros(1, dtype=torch.int64, device=m.device)
    cu = torch.cat([zero, m.cumsum(0)])
    cg = torch.cat([zero, grow.cumsum(0)])
    head, count = s["state"][0].long(), s["state"][1].long()
    cols = torch.arange(s["tables"].shape[1], device=m.device)
    # pages handed out in request order, then page order
    at = cols[None, :] - held[:, None]
    fresh = (at >= 0) & (at < grow[:, None])
    s["tables"].copy_(torch.where(fresh, s["ring"][(head + cg[:-1, None] + at) % n_pages], s["tables"]))
    # ended requests' pages behind the queue's tail
    back = s["tables"][cols[None, :] < freed[:, None]]
    s["ring"][(head + count + torch.arange(back.numel(), device=m.device)) % n_pages] = back
    t = torch.arange(cap, device=m.device)
    r = (torch.searchsorted(cu, t, right=True) - 1).clamp(max=n - 1)
    live = t < cu[-1]
    pos = kv_len[r] + t - cu[r]
    slot = s["tables"][r, (pos // page).clamp(max=cols.numel() - 1)].long() * page + pos % page
    s["slots"].copy_(torch.where(live, slot, -torch.ones_like(slot)))
    s["positions"].copy_(torch.where(live, pos, torch.zeros_like(pos)))
    s["cu_new"].copy_(cu)
    s["kv_len_out"].copy_(torch.where(ended, torch.zeros_like(kv_len), kv_len + m))
    s["state_out"].copy_(torch.stack([(head + cg[-1]) % n_pages, count - cg[-1] + back.numel(), 0 * head, cu[-1]]))
    return [s[k] for k in ("tables", "ring", "kv_len_out", "cu_new", "slots", "positions", "state_out")]


def _plain_store(s):
    h, kv, hd, kind, rot, theta, norms = SHAPES[s["shape"]]
    rows = s["q"].shape[0]
    live = s["slots"] >= 0
    freq = theta ** (-2.0 * torch.arange(rot // 2, device="cuda", dtype=torch.float64) / rot)
    angle = s["positions"].double()[:, None] * freq
    c, sn = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x, heads, w):
        x = x.float().reshape(rows, heads, hd)
        if norms:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        y = x.clone()
        a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if kind == 0 else (x[..., :rot // 2], x[..., rot // 2:rot])
        ra, rb = a * c - b * sn, a * sn + b * c
        if kind == 0:
            y[..., 0:rot:2], y[..., 1:rot:2] = ra, rb
        else:
            y[..., :rot // 2], y[..., rot // 2:rot] = ra, rb
        return y.reshape(rows, -1)

    at = s["slots"][live].long()
    s["q_out"][live] = turned(s["q"], h, s["q_w"])[live].to(s["q_out"].dtype)
    s["kpool"].view(-1, kv * hd)[at] = turned(s["k"], kv, s["k_w"])[live].to(torch.float16)
    s["vpool"].view(-1, kv * hd)[at] = s["v"][live].to(torch.float16)
    return [s["q_out"], s["kpool"], s["vpool"]]


def _plain_attn(s):
    h, kv, hd, *_ = SHAPES[s["shape"]]
    g = h // kv
    for r, length in enumerate(s["total"]):
        a, b = s["cu"][r], s["cu"][r + 1]
        pages = s["tables"][r, :_pages(length, s["page"])].long()
        k = s["kpool"][pages].reshape(-1, kv, hd)[:length].float().permute(1, 2, 0)     # [kv, hd, L]
        v = s["vpool"][pages].reshape(-1, kv, hd)[:length].float().transpose(0, 1)      # [kv, L, hd]
        step = max(1, (1 << 28) // (h * length))
        for t in range(a, b, step):
            u = min(b, t + step)
            q = s["q"][t:u].float().reshape(u - t, kv, g, hd).permute(1, 2, 0, 3).reshape(kv, g * (u - t), hd)
            sc = ((q @ k) / math.sqrt(hd)).reshape(kv, g, u - t, length)
            pos = length - (b - a) + torch.arange(t - a, u - a, device="cuda")
            sc = sc.masked_fill(torch.arange(length, device="cuda")[None, :] > pos[:, None], float("-inf"))
            p = (sc - sc.amax(-1, keepdim=True)).exp()
            o = (p.reshape(kv, -1, length) @ v).reshape(kv, g, u - t, hd) / p.sum(-1, keepdim=True)
            o = o.permute(2, 0, 1, 3).reshape(u - t, h * hd)
            if s["gate"] is not None:
                o = o / (1 + (-s["gate"][t:u].float()).exp())
            s["out"][t:u] = o.to(s["out"].dtype)
    return s["out"]


# ----------------------------------------------------------- library calls

def _own_step(s):
    from yllm_b200 import attn
    attn.page_step(s["kv_len_out"], s["cu_new"], s["slots"], s["positions"], s["state_out"], s["tables"], s["ring"],
                   s["state"], s["kv_len"], s["new_len"], s["page"])
    return [s[k] for k in ("tables", "ring", "kv_len_out", "cu_new", "slots", "positions", "state_out")]


def _own_store(s):
    from yllm_b200 import attn
    h, kv, hd, kind, rot, theta, norms = SHAPES[s["shape"]]
    norm = attn.qk_norm(s["q_w"], s["k_w"], EPS) if norms else None
    attn.rope_store_kv_paged(s["q_out"], s["q"], s["k"], s["v"], s["kpool"], s["vpool"], s["slots"], s["positions"],
                             h, kv, hd, kind, theta, n_rope_dims=rot, norm=norm)
    return [s["q_out"], s["kpool"], s["vpool"]]


def _own_attn(s):
    from yllm_b200 import attn
    h, kv, hd, *_ = SHAPES[s["shape"]]
    attn.attn_paged(s["out"], s["q"], s["kpool"], s["vpool"], s["tables"], s["cu_new"], s["kv_len"], s["max_new"],
                    h, kv, hd, gate=s["gate"])
    return s["out"]


def run(state):
    forms = (_own_step, _own_store, _own_attn) if own else (_plain_step, _plain_store, _plain_attn)
    return forms[("step", "store", "attn").index(state["op"])](state)


# -------------------------------------------------------- what it cannot do without

def work(case):
    if case["op"] == "store":
        h, kv, hd, kind, rot, theta, norms = SHAPES[case["shape"]]
        act = DT[case["dtype"]].itemsize
        t = case["tokens"]
        return {"bytes": t * ((2 * h + 2 * kv) * hd * act + 2 * kv * hd * 2 + 4) + 4 * (t + case["spare"]),
                "flops": t * (h + kv) * (3 * rot + (4 * hd if norms else 0))}
    cached, new = _lengths(case, 1)
    if case["op"] == "step":
        page = case["page"]
        total = sum(max(m, 0) for m in new)
        touched = sum(_pages(c + m, page) - c // page for c, m in zip(cached, new) if m > 0)
        grow = sum(_pages(c + max(m, 0), page) - _pages(c, page) for c, m in zip(cached, new))
        freed = sum(_pages(c, page) for c, m in zip(cached, new) if m < 0)
        return {"bytes": 16 * case["n_seqs"] + 8 * (total + case["spare"]) + 4 * touched + 4 * grow + 8 * freed + 36,
                "flops": 0}
    h, kv, hd, *_ = SHAPES[case["shape"]]
    act = DT[case["dtype"]].itemsize
    rows = sum(new)
    keys = sum(c + m for c, m in zip(cached, new))
    pages = sum(_pages(c + m, case["page"]) for c, m in zip(cached, new))
    pairs = sum(c * m + m * (m + 1) // 2 for c, m in zip(cached, new))
    return {"bytes": keys * kv * hd * 4 + rows * h * hd * act * (3 if case["gate"] else 2) + 4 * pages + 8 * len(new),
            "flops": 4 * hd * h * pairs}


# ------------------------------------------------------------ 64-bit results

def _exact_step(case, seed):
    s = prepare(case, seed)
    page, cap = case["page"], s["slots"].numel()
    lens, new, tables = s["kv_len"].tolist(), s["new_len"].tolist(), s["tables"].tolist()
    ring = s["ring"].tolist()
    head, count = s["state"].tolist()[:2]
    free = [ring[(head + i) % len(ring)] for i in range(count)]
    freed, slots, positions, out_len, cu, taken = [], [], [], [], [0], 0
    for r, (c, m) in enumerate(zip(lens, new)):
        if m < 0:
            freed += tables[r][:_pages(c, page)]
            out_len.append(0)
        else:
            for p in range(c, c + m):
                if p % page == 0:
                    tables[r][p // page] = free[taken]
                    taken += 1
                slots.append(tables[r][p // page] * page + p % page)
                positions.append(p)
            out_len.append(c + m)
        cu.append(len(slots))
    for i, x in enumerate(freed):
        ring[(head + count + i) % len(ring)] = x
    total = len(slots)
    slots += [-1] * (cap - total)
    positions += [0] * (cap - total)
    state = [(head + taken) % len(ring), count - taken + len(freed), 0, total]
    return [_i32(x) for x in (tables, ring, out_len, cu, slots, positions, state)]


def _exact_store(case, seed):
    s = prepare(case, seed)
    h, kv, hd, kind, rot, theta, norms = SHAPES[case["shape"]]
    n = case["tokens"]
    half = rot // 2
    j = torch.arange(half, dtype=torch.float64, device="cuda")
    first = (2 * j if kind == 0 else j).long()
    second = first + (1 if kind == 0 else half)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       torch.outer(s["positions"][:n].double(), torch.exp(-j / half * math.log(theta))))

    def rows(x, heads, w):
        x = x[:n].double().reshape(n, heads, hd)
        if norms:
            x = w.double() * x / (x.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt()
        z = torch.complex(x[..., first], x[..., second]) * turn[:, None, :]
        y = x.clone()
        y[..., first] = z.real
        y[..., second] = z.imag
        return y.reshape(n, heads * hd)

    q_out = s["q_out"].double()
    q_out[:n] = rows(s["q"], h, s["q_w"])
    at = s["slots"][:n].long()
    kpool, vpool = s["kpool"].double(), s["vpool"].double()
    kpool.view(-1, kv * hd)[at] = rows(s["k"], kv, s["k_w"])
    vpool.view(-1, kv * hd)[at] = s["v"][:n].double()
    return [q_out, kpool, vpool]


def _exact_attn(case, seed):
    s = prepare(case, seed)
    h, kv, hd, *_ = SHAPES[case["shape"]]
    page = case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    kp, vp = s["kpool"].view(-1, kv, hd), s["vpool"].view(-1, kv, hd)
    for r, length in enumerate(s["total"]):
        a, b = s["cu"][r], s["cu"][r + 1]
        key = torch.arange(length, device="cuda")
        row = s["tables"][r].long()[key // page] * page + key % page
        seen = length - (b - a) + torch.arange(b - a, device="cuda")     # each token's last key
        for head in range(h):
            k, v = kp[row, head * kv // h].double(), vp[row, head * kv // h].double()
            cols = slice(head * hd, (head + 1) * hd)
            for t in range(0, b - a, 2048):
                sc = s["q"][a + t:min(b, a + t + 2048), cols].double() @ k.T * hd ** -0.5
                sc = torch.where(key <= seen[t:t + 2048, None], sc, -math.inf)
                out[a + t:min(b, a + t + 2048), cols] = torch.softmax(sc, -1) @ v
    if s["gate"] is not None:
        out *= torch.sigmoid(s["gate"].double())
    return out


def exact(case, seed):
    return {"step": _exact_step, "store": _exact_store, "attn": _exact_attn}[case["op"]](case, seed)
