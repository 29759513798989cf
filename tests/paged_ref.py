"""Plain 64-bit forms of the paged-cache operators (numpy), for the tests."""
import numpy as np


def page_step(tables, ring, head, count, kv_len, new_len, page, max_tokens, max_pages=None):
    """Returns dict(tables, ring, cu, slots, positions, kv_len, state) after one step (verdicts included)."""
    tables, ring = tables.copy(), ring.copy()
    n_pages = ring.size
    max_pages = tables.shape[1] if max_pages is None else max_pages
    pages = lambda x: -(-int(x) // page)
    denied = dict(tables=tables.copy(), ring=ring.copy(), cu=np.zeros(len(kv_len) + 1, np.int32),
                  slots=np.full(max_tokens, -1, np.int32), positions=np.zeros(max_tokens, np.int32),
                  kv_len=np.array(kv_len, np.int32))

    def deny(code):
        return dict(denied, state=[head, count, code, 0])

    if not (0 <= head < n_pages and 0 <= count <= n_pages):
        return deny(-3)
    for c, m in zip(kv_len, new_len):
        if c < 0 or m < -1 or pages(c) > max_pages:
            return deny(-3)
    back = sum(pages(c) for c, m in zip(kv_len, new_len) if m < 0)
    if count + back > n_pages:
        return deny(-3)
    if any(m >= 0 and pages(c + m) > max_pages for c, m in zip(kv_len, new_len)):
        return deny(-2)
    total = sum(max(int(m), 0) for m in new_len)
    if total > max_tokens:
        return deny(-1)
    need = sum(pages(int(c) + int(m)) - pages(c) for c, m in zip(kv_len, new_len) if m >= 0)
    if need > count:
        return deny(need - count)
    free = [ring[(head + i) % n_pages] for i in range(count)]
    freed, slots, positions, cu, out = [], [], [], [0], []
    for r, (c, m) in enumerate(zip(kv_len, new_len)):
        if m < 0:
            freed += list(tables[r, :pages(c)])
            out.append(0)
        else:
            for p in range(pages(c), pages(int(c) + int(m))):
                tables[r, p] = free.pop(0)
            for p in range(int(c), int(c) + int(m)):
                slots.append(int(tables[r, p // page]) * page + p % page)
                positions.append(p)
            out.append(int(c) + int(m))
        cu.append(len(slots))
    for i, x in enumerate(freed):
        ring[(head + count + i) % n_pages] = x
    pad = max_tokens - total
    return dict(tables=tables, ring=ring, cu=np.array(cu, np.int32), slots=np.array(slots + [-1] * pad, np.int32),
                positions=np.array(positions + [0] * pad, np.int32), kv_len=np.array(out, np.int32),
                state=[(head + need) % n_pages, count - need + len(freed), 0, total])


def rope_rows(x, positions, heads, hd, kind, n_dims, theta, w=None, eps=0.0):
    """QK-norm (w) and RoPE of x [T, heads*hd] in 64 bits."""
    x = np.asarray(x, np.float64).reshape(len(positions), heads, hd).copy()
    if w is not None:
        x = x * np.asarray(w, np.float64) / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    n = n_dims if kind == 2 else hd
    j = np.arange(n // 2)
    e0, e1 = (2 * j, 2 * j + 1) if kind == 0 else (j, j + n // 2)
    ang = np.asarray(positions, np.float64)[:, None] * float(theta) ** (-2.0 * j / n)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    a, b = x[..., e0].copy(), x[..., e1].copy()
    x[..., e0], x[..., e1] = a * c - b * s, a * s + b * c
    return x.reshape(len(positions), heads * hd)


def attn(q, k_rows, v_rows, tables, cu, kv_len, page, n_heads, n_kv, hd, gate=None):
    """Attention over pages in 64 bits: k_rows, v_rows [rows, kv_dim]; rows past cu[-1] come back as zeros."""
    q = np.asarray(q, np.float64)
    out = np.zeros_like(q)
    for r in range(len(kv_len)):
        a, b, L = int(cu[r]), int(cu[r + 1]), int(kv_len[r])
        t = np.arange(L)
        rows = tables[r, t // page].astype(np.int64) * page + t % page
        for h in range(n_heads):
            g = h * n_kv // n_heads
            k = np.asarray(k_rows[rows, g * hd:(g + 1) * hd], np.float64)
            v = np.asarray(v_rows[rows, g * hd:(g + 1) * hd], np.float64)
            for i in range(a, b):
                last = L - (b - a) + (i - a)
                if last < 0:
                    continue
                s = k[:last + 1] @ q[i, h * hd:(h + 1) * hd] / np.sqrt(hd)
                p = np.exp(s - s.max())
                out[i, h * hd:(h + 1) * hd] = (p @ v[:last + 1]) / p.sum()
    if gate is not None:
        out = out / (1 + np.exp(-np.asarray(gate, np.float64)))
    return out
