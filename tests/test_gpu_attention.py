"""Paged attention against its plain 64-bit form, by element and with derived bounds: lengths from nothing to long, odd sizes, head
layouts, windows with sinks, strides, poisoned surroundings, streams and graphs."""
import math

import pytest

torch = pytest.importorskip("torch")
import attention_cases as ac  # noqa: E402

pytestmark = pytest.mark.gpu
H, B = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def amp():
    import ampstein_b200
    return ampstein_b200


def make(pos, counts, hq, hkv, d, page, dtype, window=0, sinks=0, seed=1, **kw):
    k, v, table = ac.paged(pos, counts, page, hkv, d, dtype, window, sinks, seed, **kw)
    g = torch.Generator().manual_seed(seed + 1000)
    q = torch.randn((sum(counts), hq, d), generator=g).to(dtype).cuda()
    return q, k, v, table


def cu_of(counts):
    c = [0]
    for n in counts:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int32, device="cuda")


def check(amp, pos, counts, hq, hkv, d, page, dtype, window=0, sinks=0, ragged=False, scale=None, pos_dtype=torch.int32, seed=1, **kw):
    q, k, v, table = make(pos, counts, hq, hkv, d, page, dtype, window, sinks, seed, **kw)
    lse = torch.full((q.shape[0], hq), 7.0, device="cuda")
    out = amp.paged_attention(q, k, v, table, torch.tensor(pos, dtype=pos_dtype, device="cuda"), cu=cu_of(counts) if ragged else None,
                              window=window, sinks=sinks, scale=scale, lse=lse)
    want, wlse, tol, ltol = ac.attention(q, k, v, table, pos, counts, window, sinks, d ** -0.5 if scale is None else scale)
    assert torch.isfinite(out).all()
    over = (out.double() - want).abs() - tol
    assert over.max() <= 0, (float(over.max()), int(over.argmax()))
    assert torch.equal(torch.isinf(lse), torch.isinf(wlse))
    live = ~torch.isinf(wlse)
    assert ((lse.double() - wlse)[live].abs() <= ltol[live]).all()
    return out


@pytest.mark.parametrize("dtype,wide", [(H, 0), (B, 0), (H, 200)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 8), (8, 2), (6, 1), (5, 1), (14, 2), (16, 1), (40, 2)])
def test_one_token(amp, dtype, d, hq, hkv, wide):
    """Every group size, rows that fill a row tile and rows that do not; lengths 1, 2, around the units' ends, none"""
    pos = [0, 1, 14, 15, 16, 62, 63, 64, 127, 128, -1, 700]
    check(amp, pos, [1] * len(pos), hq, hkv, d, 16, dtype, wide=wide)


@pytest.mark.parametrize("page", [1, 3, 16, 24, 64, 100, 256, 1000])
def test_pages_that_end_inside_a_unit(amp, page):
    check(amp, [0, 99, 517, 64], [1] * 4, 8, 2, 128, page, H, wide=2)
    check(amp, [0, 99, 517, 64], [1] * 4, 8, 2, 128, page, H, wide=-(-2500 // page))
    for wide in (2, -(-2500 // page)):
        check(amp, [0, 117], [70, 70], 8, 2, 128, page, B, wide=wide)


@pytest.mark.parametrize("length", [1, 63, 64, 65, 255, 256, 257, 1000, 9001])
def test_one_sequence_over_the_whole_device(amp, length):
    check(amp, [length - 1], [1], 4, 1, 128, 64, B, pos_dtype=torch.int64)


@pytest.mark.parametrize("wide", [0, 200])                              # (long tables: equal ranges instead of clusters)
@pytest.mark.parametrize("count", [2, 3, 4, 5, 7, 16, 33])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (6, 1, 64), (3, 3, 256), (32, 2, 128)])
def test_several_tokens_per_sequence(amp, count, hq, hkv, d, wide):
    """Drafted tokens: each sees the ones in front of it; sequences that begin with the call, and one that begins inside it"""
    pos = [0, 100, 300, 1, -1, -count]
    check(amp, pos, [count] * len(pos), hq, hkv, d, 16, B, wide=wide)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 4), (16, 0), (64, 4), (100, 1), (100, 200), (5000, 3)])
@pytest.mark.parametrize("count", [1, 3, 20])
def test_windows_and_sinks(amp, window, sinks, count):
    """Windows of one key, longer than the sequence, sinks beyond the window; pages left behind are not read"""
    check(amp, [0, 5, 17, 90, 400, 1000, -1], [count] * 7, 4, 2, 64, 16, H, window, sinks)


def test_sinks_without_a_window_change_nothing(amp):
    q, k, v, table = make([200, 50], [1, 1], 4, 2, 64, 16, H)
    pos = torch.tensor([200, 50], dtype=torch.int32, device="cuda")
    assert torch.equal(amp.paged_attention(q, k, v, table, pos), amp.paged_attention(q, k, v, table, pos, sinks=4))


@pytest.mark.parametrize("d,dtype,wide", [(64, B, 0), (128, H, 0), (128, B, 100), (256, H, 0), (64, H, 100)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
def test_mixed_ragged(amp, d, dtype, window, sinks, wide):
    """Single tokens, drafts, prompts, empty sequences in one call"""
    counts = [1, 200, 0, 3, 77, 1, 0, 129]
    pos = [900, 0, 5, 63, 64, -1, 0, 31]
    check(amp, pos, counts, 8, 2, d, 16, dtype, window, sinks, ragged=True, wide=wide)


@pytest.mark.parametrize("wide", [0, 200])                              # (long tables: two row tiles per CTA instead of one)
@pytest.mark.parametrize("count,first", [(64, 0), (300, 0), (257, 1000), (130, 7)])
@pytest.mark.parametrize("hq,hkv,d,dtype", [(8, 2, 128, H), (5, 1, 64, B), (4, 4, 128, B), (2, 1, 256, B), (32, 2, 64, H)])
def test_prompt_chunks(amp, count, first, hq, hkv, d, dtype, wide):
    check(amp, [first], [count], hq, hkv, d, 24, dtype, wide=wide)


def test_a_prompt_of_many_tiles(amp):
    """Whole waves of CTAs, no slices; every eleventh row is checked"""
    n, hq, hkv, d = 2600, 8, 8, 128
    q, k, v, table = make([0], [n], hq, hkv, d, 64, H)
    out = amp.paged_attention(q, k, v, table, torch.tensor([0], device="cuda"))
    rows = list(range(0, n, 11)) + [n - 1]
    for r0 in range(0, len(rows), 60):
        part = rows[r0:r0 + 60]
        pos = part
        want, _, tol, _ = ac.attention(q[part], k, v, table.expand(len(part), -1), pos, [1] * len(part), 0, 0, d ** -0.5)
        assert ((out[part].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("scale", [0.0, -0.5, 1.0, 0.003])
@pytest.mark.parametrize("wide", [0, 200])
def test_scales_of_prompts(amp, scale, wide):
    check(amp, [40], [90], 4, 2, 128, 16, H, scale=scale, wide=wide)


def test_many_sequences_of_different_lengths(amp):
    """More segments than CTAs, more sequences than a warp counts by itself: ranges over all of them"""
    g = torch.Generator().manual_seed(6)
    pos = torch.randint(-1, 120, (220,), generator=g).tolist()
    pos[7], pos[100], pos[219] = 2500, 1900, 3000
    check(amp, pos, [1] * 220, 8, 2, 128, 16, H)
    check(amp, pos, [1] * 220, 4, 4, 64, 16, B)
    check(amp, pos[:40], [1] * 40, 4, 2, 256, 64, B)


@pytest.mark.parametrize("counts", [[1, 60, 0, 3], [64, 0, 0, 0], [0, 0, 0, 0], [16, 16, 16, 16]])
def test_captured_ragged_calls_replay_with_other_cuts(amp, counts):
    rows = 64
    q, k, v, table = make([300] * 4, [rows] * 4, 4, 2, 128, 16, H)
    k, v = torch.nan_to_num(k, 1.0, 1.0, -1.0), torch.nan_to_num(v, 1.0, 1.0, -1.0)
    table = table.clamp(0, k.shape[0] - 1)
    q = q[:rows].contiguous()
    pos, cu, out = torch.tensor([5, 5, 5, 5], device="cuda"), cu_of([16, 16, 16, 16]), torch.zeros_like(q)
    amp.paged_attention(q, k, v, table, pos, cu=cu, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        amp.paged_attention(q, k, v, table, pos, cu=cu, out=out)
    pos.copy_(torch.tensor([200, 17, -1, 90]))
    cu.copy_(cu_of(counts))
    out.fill_(5.0)
    graph.replay()
    want = amp.paged_attention(q, k, v, table, pos, cu=cu, out=torch.full_like(q, 5.0))
    assert torch.equal(out, want) and (out[sum(counts):] == 5.0).all()
    ref, _, tol, _ = ac.attention(q, k, v, table, [200, 17, -1, 90], counts, 0, 0, 128 ** -0.5)
    n = sum(counts)
    assert ((out[:n].double() - ref[:n]).abs() <= tol[:n]).all()


@pytest.mark.parametrize("window,sinks", [(1, 0), (30, 4), (128, 4), (200, 500)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_prompt_chunks_in_a_window(amp, window, sinks, d):
    check(amp, [0, 600], [260, 260], 8, 2, d, 16, B, window, sinks)


@pytest.mark.parametrize("d", [64, 128])
def test_prompt_chunks_in_a_long_window(amp, d):
    """Windows long enough for two row tiles per CTA, in a context longer than they are"""
    check(amp, [2300], [140], 4, 1, d, 16, H, 1700, 5)


def test_scales(amp):
    for scale in (0.0, -0.5, 1.0, 0.003):
        check(amp, [40, 300], [2, 2], 4, 2, 64, 16, H, scale=scale)


def test_peaked_scores(amp):
    """Scores far apart: every other weight vanishes, and the running maximum moves late"""
    q, k, v, table = make([1500], [1], 4, 1, 128, 64, H)
    q *= 8
    k = torch.where(torch.isfinite(k), k * torch.linspace(0.5, 4, k.shape[0], device="cuda").to(H)[:, None, None, None], k)
    out = amp.paged_attention(q, k, v, table, torch.tensor([1500], device="cuda"))
    want, _, tol, _ = ac.attention(q, k, v, table, [1500], [1], 0, 0, 128 ** -0.5)
    assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("count,extra", [(2, 0), (2, 200), (90, 0), (90, 200)])
def test_strides(amp, count, extra):
    """q out of a packed q|k|v row, caches stored per head, caches that are one layer of a larger tensor, out inside a larger one"""
    pos, counts, hq, hkv, d = [333, 20], [count] * 2, 8, 2, 128
    n = 2 * count
    q, k, v, table = make(pos, counts, hq, hkv, d, 16, H, wide=extra)
    want = amp.paged_attention(q, k, v, table, torch.tensor(pos, device="cuda"))
    packed = torch.randn((n, (hq + 2 * hkv) * d), device="cuda").to(H)
    packed[:, :hq * d] = q.view(n, -1)
    qs = packed[:, :hq * d].view(n, hq, d)
    kh, vh = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    both = torch.stack((k, v), 1)                                       # (pages, 2, page_size, ...)
    wide = torch.zeros((n, 2 * hq, d), dtype=H, device="cuda")
    tab = torch.cat((table, table), 1)[:, :table.shape[1]]
    for kk, vv in ((kh, vh), (k, vh), (both[:, 0], both[:, 1])):
        got = amp.paged_attention(qs, kk, vv, tab, torch.tensor(pos, device="cuda"), out=wide[:, hq:])
        assert torch.equal(got, want) and not wide[:, :hq].any()


def test_same_bits_every_time(amp):
    q, k, v, table = make([5000, 70, 900], [1, 1, 1], 8, 2, 128, 16, H)
    pos = torch.tensor([5000, 70, 900], device="cuda")
    first = amp.paged_attention(q, k, v, table, pos)
    for _ in range(5):
        assert torch.equal(first, amp.paged_attention(q, k, v, table, pos))


@pytest.mark.parametrize("counts", [[1, 1, 1], [3, 3, 3], [140, 2, 70]])
def test_rows_behind_the_last_sequence_are_left(amp, counts):
    pos = [10, 200, 0]
    q, k, v, table = make(pos, counts, 4, 2, 128, 16, H)
    q = torch.cat((q, torch.full((9, 4, 128), math.nan, dtype=H, device="cuda")))
    out = torch.full_like(q, 3.0)
    lse = torch.full(q.shape[:2], 5.0, device="cuda")
    amp.paged_attention(q, k, v, table, torch.tensor(pos, device="cuda"), cu=cu_of(counts), out=out, lse=lse)
    n = sum(counts)
    assert (out[n:] == 3.0).all() and (lse[n:] == 5.0).all() and torch.isfinite(out[:n]).all()


@pytest.mark.parametrize("wide", [0, 200])
@pytest.mark.parametrize("count", [1, 3, 200])
def test_pages_outside_the_pool_give_nan_in_their_rows_alone(amp, count, wide):
    """A table that names no page, or ends too early, is not read from; the other sequences keep their bits"""
    pos = [500, 500, 500, 1 << 40]
    q, k, v, table = make([500] * 4, [count] * 4, 4, 2, 128, 16, H, wide=wide)
    p = torch.tensor([500] * 4, dtype=torch.int64, device="cuda")
    want = amp.paged_attention(q, k, v, table, p)
    broken = table.clone()
    broken[1, 3] = -1
    broken[2, 30] = k.shape[0]
    got = amp.paged_attention(q, k, v, broken, torch.tensor(pos, dtype=torch.int64, device="cuda"))
    assert torch.equal(got[:count], want[:count]) and got[count:].isnan().all()
    short = amp.paged_attention(q, k, v, table[:, :4].contiguous(), p)
    assert short.isnan().all()
    none = amp.paged_attention(q, k, v, table[:, :0], torch.tensor([-count, 0, -1, 5], device="cuda"))
    assert (none[:count] == 0).all() and none[count:2 * count].isnan().all()


@pytest.mark.parametrize("wide", [0, 200])
@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 3)])
@pytest.mark.parametrize("count", [2, 5, 16, 40, 150])
@pytest.mark.parametrize("hq,hkv,d,dtype", [(8, 2, 128, H), (3, 1, 64, B), (4, 2, 256, H)])
def test_infinities_and_nan_reach_the_rows_that_see_them_alone(amp, hq, hkv, d, dtype, count, window, sinks, wide):
    """A padded batch's spare rows, a token whose projections overflowed: other tokens of the call do not see those keys"""
    pos, page = [300, 0], 16
    q, k, v, table = make(pos, [count] * 2, hq, hkv, d, page, dtype, window, sinks, wide=wide)
    odd = torch.zeros_like(v, dtype=torch.bool)
    inf, nan = math.inf, math.nan

    def put(b, j, head, values):
        if j < 0 or not any(j in ac.visible(pos[b] + t, window, sinks) for t in range(count)):
            return
        at = int(table[b, j // page]), j % page, head
        for c, x in values.items():
            v[at][c % d] = x
            odd[at][c % d] = True

    for b in range(2):
        last = pos[b] + count - 1
        put(b, last, 0, {0: inf, 1: -inf, 2: nan, 33: inf, d - 1: -inf})
        put(b, last - 1, 0, {0: inf, 33: -inf, 40: nan, 63: inf})
        put(b, last, hkv - 1, {5: nan})
        put(b, pos[b] + count // 2, hkv - 1, {c: inf for c in range(d // 2, d)})
        put(b, pos[b] - window + 2, 0, {7: inf, 8: -inf, 62: nan})          # the window leaves it behind soon
        put(b, pos[b] + 1, 0, {9: nan})
    clean = torch.where(odd, torch.zeros_like(v), v)
    lse = torch.zeros((2 * count, hq), device="cuda")
    out = amp.paged_attention(q, k, v, table, torch.tensor(pos, device="cuda"), window=window, sinks=sinks, lse=lse)
    want, wlse, tol, ltol = ac.attention(q, k, clean, table, pos, [count] * 2, window, sinks, d ** -0.5)
    up, down = torch.zeros_like(out, dtype=torch.bool), torch.zeros_like(out, dtype=torch.bool)
    kinds = [(odd & ~(v < 0)).repeat_interleave(hq // hkv, 2), (odd & ~(v > 0)).repeat_interleave(hq // hkv, 2)]
    for row, (b, p) in enumerate(ac.tokens(pos, [count] * 2)):
        js = torch.tensor(ac.visible(p, window, sinks), device="cuda")
        pages, rows = table[b, js // page].long(), js % page
        up[row], down[row] = (x[pages, rows].any(0) for x in kinds)
    fine = ~up & ~down
    assert fine.any() and up.any() and down.any() and ((out.double() - want).abs() <= tol)[fine].all()
    assert (out[up & ~down] == inf).all() and (out[down & ~up] == -inf).all() and out[up & down].isnan().all()
    assert ((lse.double() - wlse).abs() <= ltol).all()


def test_far_positions_of_a_large_cache(amp):
    """Offsets that pass 32 bits: 5 GB of keys"""
    page, hkv, d = 64, 8, 128
    pages = 40000
    k = torch.zeros((pages, page, hkv, d), dtype=H, device="cuda")
    v = torch.zeros_like(k)
    table = torch.arange(pages - 1, pages - 9, -1, dtype=torch.int32, device="cuda").view(1, 8)
    g = torch.Generator(device="cuda").manual_seed(3)
    for t in (k, v):
        t[pages - 8:] = torch.randn((8, page, hkv, d), device="cuda", generator=g).to(H)
    small = torch.arange(7, -1, -1, dtype=torch.int32, device="cuda").view(1, 8)
    for n in (1, 90):
        q = torch.randn((n, 16, d), device="cuda", generator=g).to(H)
        pos = torch.tensor([511 - n], device="cuda")
        out = amp.paged_attention(q, k, v, table, pos)
        assert torch.equal(out, amp.paged_attention(q, k[pages - 8:].clone(), v[pages - 8:].clone(), small, pos))


def test_many_sequences(amp):
    g = torch.Generator().manual_seed(5)
    pos = torch.randint(-1, 90, (700,), generator=g).tolist()
    check(amp, pos, [1] * 700, 2, 1, 64, 16, H)


def test_captured_calls_replay_with_other_lengths_and_beside_each_other(amp):
    """Two graphs with their own workspaces, replayed on two streams at once; the lengths change between replays"""
    sets = []
    for seed in (1, 2):
        pos = [3000, 40, 1200, -1]
        q, k, v, table = make(pos, [1] * 4, 8, 2, 128, 16, H, seed=seed, wide=3)
        k, v = torch.nan_to_num(k, 1.0, 1.0, -1.0), torch.nan_to_num(v, 1.0, 1.0, -1.0)
        table = table.clamp(0, k.shape[0] - 1)
        p = torch.tensor(pos, device="cuda")
        out = torch.empty_like(q)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            amp.paged_attention(q, k, v, table, p, out=out)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                amp.paged_attention(q, k, v, table, p, out=out)
        sets.append((q, k, v, table, p, out, graph, stream))
    torch.cuda.synchronize()
    for lengths in ([3000, 40, 1200, -1], [17, 2999, -1, 3020], [0, 0, 0, 0]):
        for s in sets:
            s[4].copy_(torch.tensor(lengths))
        torch.cuda.synchronize()
        for _ in range(20):
            for s in sets:
                with torch.cuda.stream(s[7]):
                    s[6].replay()
        torch.cuda.synchronize()
        for q, k, v, table, p, out, _, _ in sets:
            assert torch.equal(out, amp.paged_attention(q, k, v, table, p))


def test_two_streams_at_once(amp):
    a, b = make([4000], [1], 8, 2, 128, 16, H, seed=1), make([3000, 77], [1, 1], 8, 2, 128, 16, H, seed=2)
    pa, pb = torch.tensor([4000], device="cuda"), torch.tensor([3000, 77], device="cuda")
    wa, wb = amp.paged_attention(*a, pa), amp.paged_attention(*b, pb)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(30):
        for s, args, p in zip(streams, (a, b), (pa, pb)):
            with torch.cuda.stream(s):
                got.append(amp.paged_attention(*args, p))
    torch.cuda.synchronize()
    assert all(torch.equal(x, wa if i % 2 == 0 else wb) for i, x in enumerate(got))


def test_empty_calls(amp):
    q, k, v, table = make([5], [1], 4, 2, 64, 16, H)
    e = amp.paged_attention(q[:0], k, v, table[:0], torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert e.shape == (0, 4, 64)
    amp.paged_attention(q[:0], k, v, table, torch.zeros(1, dtype=torch.int32, device="cuda"))
    out = amp.paged_attention(q, k, v, table[:0], torch.zeros(0, dtype=torch.int32, device="cuda"), cu=cu_of([]), out=torch.full_like(q, 2.0))
    assert (out == 2.0).all()


def test_refusals(amp):
    q, k, v, table = make([5, 9], [1, 1], 4, 2, 64, 16, H)
    pos = torch.tensor([5, 9], device="cuda")
    f = amp.paged_attention
    bad = [
        (RuntimeError, lambda: f(q.cpu(), k, v, table, pos)),
        (RuntimeError, lambda: f(q, k, v, table.cpu(), pos)),
        (TypeError, lambda: f(q.float(), k, v, table, pos)),
        (TypeError, lambda: f(q, k.to(B), v, table, pos)),
        (TypeError, lambda: f(q, k, v, table.long(), pos)),
        (TypeError, lambda: f(q, k, v, table, pos.float())),
        (TypeError, lambda: f(q, k, v, table, pos, cu=torch.zeros(2, dtype=torch.int32, device="cuda"))),
        (TypeError, lambda: f(q, k, v, table[:1], pos)),
        (ValueError, lambda: f(q[:, :3], k, v, table, pos)),
        (ValueError, lambda: f(q[:, :, :32], k[..., :32], v[..., :32], table, pos)),
        (ValueError, lambda: f(q, k, v[:1], table, pos)),
        (ValueError, lambda: f(torch.cat((q, q[:1])), k, v, table, pos)),
        (ValueError, lambda: f(q, k, v, table, pos, window=-1)),
        (ValueError, lambda: f(q, k, v, table, pos, scale=math.nan)),
        (ValueError, lambda: f(q, k, v, table, pos, scale=3e38)),
        (ValueError, lambda: f(q, k, v, table, pos, out=q)),
        (ValueError, lambda: f(q, k, v, table, pos, lse=torch.zeros((2, 3), device="cuda"))),
        (ValueError, lambda: f(q.transpose(1, 2).contiguous().transpose(1, 2), k, v, table, pos)),
        (RuntimeError, lambda: f(torch.zeros(2 * 4 * 64 + 1, dtype=H, device="cuda")[1:].view(2, 4, 64), k, v, table, pos)),
        (ValueError, lambda: f(q, k, v, table, pos, out=q[:1].clone().expand(2, 4, 64))),
        (ValueError, lambda: f(q, k, v, torch.zeros((2, 1 << 27), dtype=torch.int32, device="cuda"), pos)),
    ]
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            pytest.fail("call %d was taken" % i)


@pytest.mark.parametrize("seqs", [33, 150, 700])
def test_prompts_among_many_sequences(amp, seqs):
    """Row tiles of prompts found behind hundreds of single tokens and empty sequences"""
    g = torch.Generator().manual_seed(seqs)
    counts = torch.randint(0, 2, (seqs,), generator=g).tolist()
    pos = torch.randint(-1, 60, (seqs,), generator=g).tolist()
    for b, n in ((0, 70), (31, 40), (32, 129), (seqs - 2, 33), (seqs - 1, 90)):
        counts[b], pos[b] = n, b % 7
    check(amp, pos, counts, 4, 2, 64, 16, H, ragged=True)


def test_no_wait_was_lost(amp):
    assert amp.attention_status() == 0


def test_calls_without_the_tensor_table(amp, monkeypatch):
    """The checks in Python and the ones on DLPack descriptions make the same calls"""
    from ampstein_b200 import attention as at
    assert at._calls()                                                  # this torch has the table
    pos, counts = [40, 700], [3, 3]
    q, k, v, table = make(pos, counts, 8, 2, 128, 16, B, window=100, sinks=3)
    p, cu = torch.tensor(pos, device="cuda"), cu_of(counts)
    inv_freq, m = amp.rope_frequencies(128, scaling=dict(kind="yarn", factor=4.0))
    new = torch.randn((6, 4, 128), device="cuda").to(B)

    def run():
        a, b = k.clone(), v.clone()
        lse = torch.zeros((6, 8), device="cuda")
        r = amp.rope_append(q, new[:, :2], new[:, 2:], p, inv_freq, a, b, table, cu=cu, interleaved=True, mscale=m)
        o = amp.paged_attention(r, a, b, table, p, cu=cu, window=100, sinks=3, scale=0.1, lse=lse)
        w = amp.paged_attention(q, k, v, table, p, window=100, sinks=3)
        amp.copy_pages([a, b], [0, 1], [2, 3])
        return r, o, w, lse, a, b, amp.rope(q, p, inv_freq)

    want = run()
    monkeypatch.setattr(at, "_direct", {})
    for x, y in zip(want, run()):
        assert torch.equal(torch.nan_to_num(x), torch.nan_to_num(y))
    monkeypatch.undo()
    par = torch.nn.Parameter(q, requires_grad=False)                    # another type than a plain tensor
    assert torch.equal(amp.paged_attention(par, k, v, table, p, window=100, sinks=3), want[2])
