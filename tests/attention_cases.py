"""Plain 64-bit forms of the rotary / paged attention operators, inputs and error bounds shared by their tests."""
import math

import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}             # largest relative error of a rounding to the type


def tokens(pos, counts):
    """[(sequence, position)] of every row"""
    return [(b, p + t) for b, (p, n) in enumerate(zip(pos, counts)) for t in range(n)]


def visible(p, window, sinks):
    return [j for j in range(p + 1) if not window or j > p - window or j < sinks] if p >= 0 else []


def rotate(x, p, inv_freq, interleaved, mscale):
    """x (heads, dim) float64 at position p"""
    half = inv_freq.numel()
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    ang = p * inv_freq.double()
    y = x.clone()
    y[:, a] = (x[:, a] * torch.cos(ang) - x[:, b] * torch.sin(ang)) * mscale
    y[:, b] = (x[:, b] * torch.cos(ang) + x[:, a] * torch.sin(ang)) * mscale
    return y


def rotate_bound(x, inv_freq, interleaved, mscale, u):
    """Largest error of a rotation of x (heads, dim) made in fp32 and rounded once: u of the result, of which cos and sin carry
    2^-22 each (the angle's rounding to fp32 half turns, pi 2^-24, and sincospif's own two units) and three operations 2^-24"""
    half = inv_freq.numel()
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    size = (x[:, a].abs() + x[:, b].abs()) * abs(mscale)
    t = torch.zeros_like(x)
    t[:, a] = t[:, b] = size * (u * 1.001 + 2.0 ** -21)
    return t + 2.0 ** -24                                              # (fp16: half a step below its normal range)


def attention(q, k_cache, v_cache, table, pos, counts, window, sinks, scale):
    """(out, lse, bound of out's error, bound of lse's error), all float64; rows behind the last sequence: zero and not meant.

    The bound, by element: the scores carry (dim + 3) roundings of 2^-24 of sum |q k| scale, and exp2 2^-21, which is the
    relative error d of a weight (twice: above and below the fraction); a weight is rounded to the type for the product (u; fp16
    below its normal range: 2^-25 of the largest weight, and a part's largest may be 2^8 times smaller than the range's end); sums in
    fp32 over n keys; the result is rounded (u)."""
    P = k_cache.shape[1]
    hq, hkv, d = q.shape[1], k_cache.shape[2], q.shape[2]
    group = hq // hkv
    u = U[q.dtype]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    tab = table.tolist()
    for row, (b, p) in enumerate(tokens(pos, counts)):
        js = visible(p, window, sinks)
        if not js:
            continue
        pages = torch.tensor([tab[b][j // P] for j in js], device=q.device)
        rows = torch.tensor([j % P for j in js], device=q.device)
        k, v = k_cache[pages, rows].double(), v_cache[pages, rows].double()       # (n, hkv, d)
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        x = q[row].double()
        s = torch.einsum("hd,nhd->hn", x, k) * scale
        size = torch.einsum("hd,nhd->hn", x.abs(), k.abs()).amax(1) * abs(scale)
        m = s.amax(1, keepdim=True)
        e = torch.exp(s - m)
        l = e.sum(1)
        out[row] = torch.einsum("hn,nhd->hd", e, v) / l[:, None]
        lse[row] = m[:, 0] + torch.log(l)
        n = len(js)
        delta = size * (d + 3) * 2.0 ** -24 + 2.0 ** -21 + s.abs().amax(1) * 2.0 ** -23
        mean = torch.einsum("hn,nhd->hd", e, v.abs()) / l[:, None]
        tol[row] = u * out[row].abs() + mean * (u + 2 * delta + (n + 64) * 2.0 ** -23)[:, None] * 1.01 + 2.0 ** -24
        if q.dtype == torch.float16:
            tol[row] += n * 2.0 ** -25 * v.abs().amax(0) / l[:, None]
        ltol[row] = delta + (n + 64) * 2.0 ** -23 + lse[row].abs() * 2.0 ** -22
    return out, lse, tol, ltol


def paged(pos, counts, page, hkv, d, dtype, window=0, sinks=0, seed=0, spare=3, wide=0, device="cuda", per_head=False):
    """Caches and a table in which every page that no row can see is poisoned: its entry lies outside the pool, and the rows of the
    pool behind a sequence's end, the spare pages and the first rows a window has left hold NaN and infinities. (k, v, table)"""
    g = torch.Generator().manual_seed(seed)
    ends = [max(0, p + n) for p, n in zip(pos, counts)]
    width = max([1] + [-(-e // page) for e in ends]) + wide
    seen = []
    for p, n in zip(pos, counts):
        seen.append(sorted({j for t in range(n) for j in visible(p + t, window, sinks)}))
    need = [(b, x) for b, js in enumerate(seen) for x in sorted({j // page for j in js})]
    pool = len(need) + spare
    order = torch.randperm(pool, generator=g).tolist()
    table = torch.randint(0, 2, (len(pos), width), generator=g, dtype=torch.int32) * 2000000000 - 1000000000
    shape = (pool, page, hkv, d)
    bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).min])[torch.randint(0, 4, shape, generator=g)]
    k, v = bad.clone(), bad.clone()
    for (b, x), at in zip(need, order):
        table[b, x] = at
        rows = [j % page for j in seen[b] if j // page == x]
        k[at, rows] = torch.randn((len(rows), hkv, d), generator=g)
        v[at, rows] = torch.randn((len(rows), hkv, d), generator=g)
    k, v = k.to(dtype), v.to(dtype)
    if per_head:                                                        # stored as (pages, kv_heads, page_size, dim)
        k, v = (t.transpose(1, 2).contiguous().to(device).transpose(1, 2) for t in (k, v))
    return k.to(device), v.to(device), table.to(device)
