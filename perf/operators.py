"""Performance cases of the operators between the q|k|v projections and o: rotary positions with the write into a paged
key-value cache, attention over that cache (new tokens of running sequences, prompt chunks, sliding windows whose first tokens
stay visible), and the copies that fork sequences and compact the cache.

Kinds of case:
  rope    rotary positions of q and k, k and v written to the cache's pages
  decode  attention of one token (or a few drafted ones) per sequence
  prompt  attention of prompt chunks
  copy    pages copied to other pages, in all layers

Sequence lengths, chunk sizes and page lists follow from the case alone (`spread` seeds them), values and the order of the pages in
the pool from the seed of prepare(). Entries of a page table that no token of the call can see are -1, as in a cache that frees
what a window has left behind."""
import math
import random

import torch

own = False
DEV = "cuda:0"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one decoded token of the 32-layer stack: the smallest call, latency counts
        dict(name="rope_m1", kind="rope", seqs=1, tokens=1, lo=8191, hi=8191, hq=32, hkv=8, d=128, rot=128, interleaved=False,
             scaling="llama3", page=16, dtype="f16", spread=1),
        # a prefill chunk packed from the prompts of several users, half of each head rotated in pairs
        dict(name="rope_chunk_2047", kind="rope", seqs=5, tokens=2047, ragged=True, lo=1, hi=100000, hq=48, hkv=8, d=128, rot=64,
             interleaved=True, scaling="yarn", page=64, dtype="bf16", spread=2),
        # the first answer tokens of one user
        dict(name="decode_m1_77", kind="decode", seqs=1, tokens=1, lo=76, hi=76, hq=32, hkv=8, d=128, page=16, window=0, sinks=0,
             dtype="f16", spread=3),
        # one user far into a long document: the whole device on one sequence
        dict(name="decode_m1_131071", kind="decode", seqs=1, tokens=1, lo=131070, hi=131070, hq=32, hkv=8, d=128, page=64, window=0,
             sinks=0, dtype="f16", spread=4),
        # a batch of users in mid conversation, two slots of the captured batch unused
        dict(name="decode_b32", kind="decode", seqs=32, unused=2, tokens=1, lo=100, hi=8192, hq=32, hkv=8, d=128, page=16, window=0,
             sinks=0, dtype="f16", spread=5),
        # a tensor-parallel shard (six query heads on one key-value head) of a windowed model, long conversations
        dict(name="decode_b48_window", kind="decode", seqs=48, tokens=1, lo=500, hi=100000, hq=6, hkv=1, d=128, page=64, window=1024,
             sinks=4, dtype="bf16", spread=6),
        # two drafted tokens verified behind each sequence's own, wide heads, pages of an odd size
        dict(name="decode_b7_t3_wide", kind="decode", seqs=7, tokens=3, lo=1000, hi=30000, hq=16, hkv=2, d=256, page=24, window=0,
             sinks=0, dtype="bf16", spread=7),
        # a whole prompt from its first token
        dict(name="prompt_8192", kind="prompt", seqs=1, tokens=8192, lo=0, hi=0, hq=32, hkv=8, d=128, page=64, window=0, sinks=0,
             dtype="f16", spread=8),
        # a prefill chunk with an odd number of tokens behind a long context
        dict(name="prompt_511_on_16k", kind="prompt", seqs=1, tokens=511, lo=16001, hi=16001, hq=48, hkv=8, d=128, page=16, window=0,
             sinks=0, dtype="bf16", spread=9),
        # the short prompts of several users packed together, narrow heads, a sliding window with sinks
        dict(name="prompt_b6_window", kind="prompt", seqs=6, tokens=2333, ragged=True, lo=0, hi=2000, hq=64, hkv=8, d=64, page=32,
             window=128, sinks=4, dtype="bf16", spread=10),
        # a sequence is forked: its last, half-filled page gets a copy of its own in each of 32 layers
        dict(name="copy_fork", kind="copy", layers=32, pages=64, pairs=1, hkv=8, d=128, page=16, dtype="f16", spread=11),
        # a fragmented cache is compacted
        dict(name="copy_compact", kind="copy", layers=16, pages=256, pairs=101, hkv=8, d=128, page=64, dtype="f16", spread=12),
    ]


def _log(rng, lo, hi):
    """Log-uniform whole number in [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("rope", "decode", "decode", "decode", "prompt", "prompt", "copy"))
    d = rng.choice((64, 128, 128, 128, 256))
    hkv = rng.choice((1, 2, 4, 8, 8))
    group = rng.choice((1, 2, 3, 4, 4, 5, 6, 7, 8, 8, 16))
    c = dict(kind=kind, hkv=hkv, d=d, page=rng.choice((1, 8, 16, 16, 24, 32, 64, 64, 100, 128, 256)), dtype=rng.choice(("f16", "bf16")),
             spread=rng.randint(100, 1 << 30))
    if kind == "copy":
        c["layers"] = rng.randint(1, 24)
        c["page"] = rng.choice((8, 16, 16, 24, 32, 64, 64, 100, 128))
        c["pages"] = rng.randint(16, 200)
        c["pairs"] = _log(rng, 1, c["pages"] // 2)
        while work(c)["bytes"] > 8e8:
            c["layers"] = -(-c["layers"] // 2)
        return c
    c["hq"] = hkv * group
    if kind == "rope":
        c["d"] = d = rng.choice((64, 80, 96, 128, 128, 256))
        c["rot"] = rng.choice((d, d, d // 2, 2 * rng.randint(1, d // 2)))
        c["interleaved"] = rng.random() < 0.5
        c["scaling"] = rng.choice(("none", "linear", "ntk", "llama3", "yarn"))
        c["ragged"] = rng.random() < 0.5
        c["seqs"] = _log(rng, 1, 64)
        c["tokens"] = max(c["seqs"], _log(rng, 1, 4096)) if c["ragged"] else _log(rng, 1, max(1, 4096 // c["seqs"]))
        c["lo"], c["hi"] = 1, rng.choice((2000, 30000, 200000))
        if not c["ragged"] and rng.random() < 0.3:
            c["unused"] = rng.randint(0, c["seqs"] - 1)
        return c
    window = rng.choice((0, 0, 0, _log(rng, 16, 4096)))
    c["window"], c["sinks"] = window, rng.choice((0, 1, 4, 16)) if window else 0
    if kind == "decode":
        c["tokens"] = rng.choice((1, 1, 1, 1, 2, 3, 4, rng.randint(5, 16)))
        c["seqs"] = _log(rng, 1, 128)
        c["unused"] = rng.choice((0, 0, rng.randint(0, c["seqs"] - 1)))
        most = 2 ** 28 // (c["seqs"] * hkv * d)                        # at most 1 GB of keys and values
        c["lo"], c["hi"] = 1, max(1, min(131000, most))
    else:
        c["seqs"] = _log(rng, 1, 8)
        c["tokens"] = max(c["seqs"], _log(rng, 17, 3500))
        c["ragged"] = True
        c["lo"], c["hi"] = 0, rng.choice((0, 0, 1000, max(1, min(16000, int(2e7 / c["tokens"])))))
        while work(c)["flops"] > 3e11 and c["tokens"] > 2 * c["seqs"]:
            c["tokens"] //= 2
    return c


def _sequences(c):
    """[(position of the first new token, number of new tokens)] of the case's sequences"""
    r = random.Random(c["spread"])
    n, total = c["seqs"], c["tokens"]
    if c.get("ragged"):
        cuts = sorted(r.sample(range(1, total), n - 1)) if n > 1 else []
        counts = [b - a for a, b in zip([0] + cuts, cuts + [total])]
    else:
        counts = [total] * n
    out = []
    for i in range(n):
        first = c["lo"] if c["lo"] == c["hi"] else (_log(r, c["lo"], c["hi"]) if c["lo"] else r.randint(0, c["hi"]))
        out.append((first, counts[i]))
    for i in r.sample(range(n), c.get("unused", 0)):
        out[i] = (-counts[i], counts[i])                                # a slot without a sequence: its tokens stand before position 0
    return out


def _visible(first, count, window, sinks):
    """Positions that some token of a chunk sees: [0, a) and [lo, end)"""
    end = max(0, first + count)
    lo = max(0, first - window + 1) if window else 0
    return min(sinks if window else 0, lo), lo, end


def _pairs(first, count, window, sinks):
    """(query, key) pairs with the key visible"""
    total = 0
    for p in range(max(0, first), first + count):
        total += p + 1 if not window or p < window else window + min(sinks, p + 1 - window)
    return total


def _page_pairs(c):
    r = random.Random(c["spread"])
    order = r.sample(range(c["pages"]), 2 * c["pairs"])
    return order[:c["pairs"]], order[c["pairs"]:]


def work(c):
    if c["kind"] == "copy":
        return dict(bytes=2 * 2 * c["layers"] * c["pairs"] * c["page"] * c["hkv"] * c["d"] * 2, flops=0)
    seqs = _sequences(c)
    rows = sum(n for _, n in seqs)
    if c["kind"] == "rope":
        live = sum(n for p, n in seqs if p >= 0)
        return dict(bytes=(2 * rows * c["hq"] + 2 * 2 * live * c["hkv"]) * c["d"] * 2 + 2 * c["rot"] + 8 * c["seqs"],
                    flops=3 * (rows * c["hq"] + live * c["hkv"]) * c["rot"])
    keys = pairs = 0
    for first, n in seqs:
        a, lo, end = _visible(first, n, c["window"], c["sinks"])
        keys += a + max(0, end - lo)
        pairs += _pairs(first, n, c["window"], c["sinks"])
    return dict(bytes=(2 * keys * c["hkv"] + 2 * rows * c["hq"]) * c["d"] * 2 + 4 * -(-keys // c["page"]) + 4 * c["seqs"],
                flops=4 * pairs * c["hq"] * c["d"])


# ---- inputs ---------------------------------------------------------------------------------


def _frequencies(c):
    """(inverse frequencies as float32 values, factor of cos and sin) of the case's scaling"""
    r, base, kind = c["rot"], 500000.0 if c["scaling"] == "llama3" else 10000.0, c["scaling"]
    if kind == "ntk" and r > 2:
        base *= 4.0 ** (r / (r - 2))
    freq = [base ** (-2.0 * i / r) for i in range(r // 2)]
    factor = 1.0
    if kind == "linear":
        freq = [f / 4 for f in freq]
    elif kind == "llama3":                                              # long waves slowed down eightfold, a ramp in between
        for i, f in enumerate(freq):
            turns = 8192 * f / (2 * math.pi)
            mix = min(1.0, max(0.0, (turns - 1.0) / (4.0 - 1.0)))
            freq[i] = mix * f + (1 - mix) * f / 8
    elif kind == "yarn":                                                # 16 times the context, the fast dimensions kept
        def dim(rotations):
            return r * math.log(4096 / (rotations * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(0, math.floor(dim(32))), min(r - 1, math.ceil(dim(1)))
        for i, f in enumerate(freq):
            keep = 1 - min(1.0, max(0.0, (i - low) / max(high - low, 0.001)))
            freq[i] = keep * f + (1 - keep) * f / 16
        factor = 0.1 * math.log(16) + 1.0
    return freq, factor


def _pool(c, g, seqs, needed):
    """Page table (seqs, most pages) int32 with the needed entries drawn from a pool in random order, and the pool's size"""
    width = max(1, max(-(-(p + n) // c["page"]) for p, n in seqs))
    count = sum(len(x) for x in needed)
    pool = count + 3
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    flat = [b * width + x for b, xs in enumerate(needed) for x in xs]
    table = torch.full((len(seqs) * width,), -1, dtype=torch.int32, device=DEV)
    table[torch.tensor(flat, dtype=torch.int64, device=DEV)] = order[:count]
    return table.view(len(seqs), width), pool


def prepare(c, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt = DTYPES[c["dtype"]]

    def randn(*shape):
        return torch.randn(shape, device=DEV, generator=g).to(dt)

    if c["kind"] == "copy":
        shape = (c["layers"], c["pages"], c["page"], c["hkv"], c["d"])
        src, dst = _page_pairs(c)
        return dict(case=c, k=randn(*shape), v=randn(*shape), src=src, dst=dst)
    seqs = _sequences(c)
    rows = sum(n for _, n in seqs)
    P = c["page"]
    s = dict(case=c, seqs=seqs, pos=torch.tensor([p for p, _ in seqs], dtype=torch.int32, device=DEV))
    if c.get("ragged"):
        cu = [0]
        for _, n in seqs:
            cu.append(cu[-1] + n)
        s["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEV)
    needed = []
    for first, n in seqs:
        if c["kind"] == "rope":
            spans = [(max(0, first), max(0, first + n))]
        else:
            a, lo, end = _visible(first, n, c["window"], c["sinks"])
            spans = [(0, a), (lo, end)]
        needed.append(sorted({x for lo, hi in spans if hi > lo for x in range(lo // P, -(-hi // P))}))
    s["table"], pool = _pool(c, g, seqs, needed)
    s["k"], s["v"] = randn(pool, P, c["hkv"], c["d"]), randn(pool, P, c["hkv"], c["d"])
    s["q"] = randn(rows, c["hq"], c["d"])
    if c["kind"] == "rope":
        s["new_k"], s["new_v"] = randn(rows, c["hkv"], c["d"]), randn(rows, c["hkv"], c["d"])
        freq, s["factor"] = _frequencies(c)
        s["freq"] = torch.tensor(freq, dtype=torch.float32, device=DEV)
    return s


# ---- one pass -------------------------------------------------------------------------------


def run(s):
    c = s["case"]
    if c["kind"] == "copy":
        return _copy_own(s) if own else _copy_plain(s)
    if c["kind"] == "rope":
        return _rope_own(s) if own else _rope_plain(s)
    return _attention_own(s) if own else _attention_plain(s)


def _copy_own(s):
    import ampstein_b200 as amp
    amp.copy_pages([s["k"], s["v"]], s["src"], s["dst"])
    return s["k"], s["v"]


def _rope_own(s):
    import ampstein_b200 as amp
    q = amp.rope_append(s["q"], s["new_k"], s["new_v"], s["pos"], s["freq"], s["k"], s["v"], s["table"], cu=s.get("cu"),
                        interleaved=s["case"]["interleaved"], mscale=s["factor"])
    return q, s["k"], s["v"]


def _attention_own(s):
    import ampstein_b200 as amp
    c = s["case"]
    return amp.paged_attention(s["q"], s["k"], s["v"], s["table"], s["pos"], cu=s.get("cu"), window=c["window"], sinks=c["sinks"])


def _copy_plain(s):
    src, dst = (torch.tensor(s[x], dtype=torch.int64, device=DEV) for x in ("src", "dst"))
    for x in (s["k"], s["v"]):
        x.index_copy_(1, dst, x.index_select(1, src))
    return s["k"], s["v"]


def _rotate_plain(x, cos, sin, rot, interleaved):
    x = x.float()
    a, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        x0, x1 = a[..., 0::2], a[..., 1::2]
        turned = torch.stack((x0 * cos - x1 * sin, x1 * cos + x0 * sin), -1).flatten(-2)
    else:
        x0, x1 = a[..., :rot // 2], a[..., rot // 2:]
        turned = torch.cat((x0 * cos - x1 * sin, x1 * cos + x0 * sin), -1)
    return torch.cat((turned, rest), -1)


def _rope_plain(s):
    c, P = s["case"], s["case"]["page"]
    p = torch.cat([torch.arange(first, first + n, device=DEV) for first, n in s["seqs"]])
    seq = torch.cat([torch.full((n,), b, dtype=torch.int64, device=DEV) for b, (_, n) in enumerate(s["seqs"])])
    angle = p.double()[:, None] * s["freq"].double()
    cos, sin = ((f(angle) * s["factor"]).float()[:, None] for f in (torch.cos, torch.sin))
    q = _rotate_plain(s["q"], cos, sin, c["rot"], c["interleaved"]).to(s["q"].dtype)
    k = _rotate_plain(s["new_k"], cos, sin, c["rot"], c["interleaved"]).to(s["q"].dtype)
    v = s["new_v"]
    if c.get("unused"):
        live = torch.cat([torch.arange(first, first + n) >= 0 for first, n in s["seqs"]]).nonzero()[:, 0].to(DEV)
        p, seq, k, v = p[live], seq[live], k[live], v[live]
    page = s["table"][seq, p // P].long()
    s["k"][page, p % P] = k
    s["v"][page, p % P] = v
    return q, s["k"], s["v"]


def _attention_plain(s):
    c, P = s["case"], s["case"]["page"]
    hq, hkv, d, W, S = c["hq"], c["hkv"], c["d"], c["window"], c["sinks"]
    G = hq // hkv
    out = torch.zeros_like(s["q"])
    at = 0
    for b, (first, n) in enumerate(s["seqs"]):
        q = s["q"][at:at + n].view(n, hkv, G, d)
        o = out[at:at + n].view(n, hkv, G, d)
        at += n
        a, lo, end = _visible(first, n, W, S)
        if end <= 0:
            continue
        j = torch.cat((torch.arange(a, device=DEV), torch.arange(lo, end, device=DEV)))
        page = s["table"][b][j // P].long()
        p = torch.arange(first, first + n, device=DEV)[:, None]
        seen = j <= p
        if W:
            seen &= (j > p - W) | (j < S)
        keys, values = s["k"][page, j % P], s["v"][page, j % P]
        for h in range(hkv):
            x = torch.matmul(q[:, h].float(), keys[:, h].float().t()) / math.sqrt(d)          # (n, G, keys)
            x = x.masked_fill_(~seen[:, None], float("-inf"))
            e = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-3e38))
            total = e.sum(-1, keepdim=True)
            o[:, h] = (torch.matmul(e, values[:, h].float()) / total.masked_fill(total == 0, 1.0)).to(o.dtype)
    return out


# ---- the definition in 64 bits --------------------------------------------------------------


def exact(c, seed):
    s = prepare(c, seed)
    if c["kind"] == "copy":
        new = []
        for x in (s["k"], s["v"]):
            y = x.double()
            for a, b in zip(s["src"], s["dst"]):
                y[:, b] = x[:, a].double()
            new.append(y)
        return tuple(new)
    if c["kind"] == "rope":
        return _exact_rope(c, s)
    return _exact_attention(c, s)


def _exact_rope(c, s):
    q, k = s["q"].double(), s["k"].double()
    v = s["v"].double()
    half, at = c["rot"] // 2, 0
    i = torch.arange(half, device=DEV)
    first_of, second_of = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
    table = s["table"].tolist()
    for b, (first, n) in enumerate(s["seqs"]):
        p = torch.arange(first, first + n, device=DEV, dtype=torch.float64)
        turn = torch.polar(torch.full((), s["factor"], dtype=torch.float64, device=DEV).expand(n, 1, half),
                           torch.outer(p, s["freq"].double())[:, None].contiguous())

        def rotated(x):
            x = x.double().clone()
            z = torch.complex(x[..., first_of], x[..., second_of]) * turn
            x[..., first_of], x[..., second_of] = z.real, z.imag
            return x

        q[at:at + n] = rotated(s["q"][at:at + n])
        nk, nv = rotated(s["new_k"][at:at + n]), s["new_v"][at:at + n].double()
        t = 0
        while t < n:                                                    # page by page
            where = first + t
            if where < 0:
                t += 1
                continue
            take = min(n - t, c["page"] - where % c["page"])
            page = table[b][where // c["page"]]
            span = slice(where % c["page"], where % c["page"] + take)
            k[page, span], v[page, span] = nk[t:t + take], nv[t:t + take]
            t += take
        at += n
    return q, k, v


def _exact_attention(c, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    W, S, P, at = c["window"], c["sinks"], c["page"], 0
    group = c["hq"] // c["hkv"]
    table = s["table"].tolist()
    for b, (first, n) in enumerate(s["seqs"]):
        end = first + n
        if end > 0:
            pages = [x if x >= 0 else 0 for x in table[b][:-(-end // P)]]
            keys = s["k"][pages].flatten(0, 1)[:end]
            values = s["v"][pages].flatten(0, 1)[:end]
            place = torch.arange(first, end, device=DEV)
            age = place[:, None] - torch.arange(end, device=DEV)[None]                  # of a key, seen from a query
            hidden = age < 0
            if W:
                hidden |= (age >= W) & (torch.arange(end, device=DEV) >= S)
            none = hidden.all(1)
            used = (~hidden).any(0).nonzero()[:, 0]                                     # (a window leaves most of a long sequence unseen)
            hidden = hidden[:, used]
            for h in range(c["hq"]):
                x = s["q"][at:at + n, h].double() @ keys[used, h // group].double().T * c["d"] ** -0.5
                x[hidden] = -math.inf
                y = torch.softmax(x, 1) @ values[used, h // group].double()
                y[none] = 0.0
                out[at:at + n, h] = y
        at += n
    return out
