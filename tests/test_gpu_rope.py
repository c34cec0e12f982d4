"""Rotary positions, the write into the paged cache and page copies against their plain forms."""
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


def rand(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def expect(x, place, inv_freq, interleaved, mscale):
    out, tol = torch.empty(x.shape, dtype=torch.float64, device="cuda"), torch.empty(x.shape, dtype=torch.float64, device="cuda")
    for row, (_, p) in enumerate(place):
        out[row] = ac.rotate(x[row].double(), p, inv_freq, interleaved, mscale)
        tol[row] = ac.rotate_bound(x[row].double(), inv_freq, interleaved, mscale, ac.U[x.dtype])
    return out, tol


def run(amp, pos, counts, hq, hkv, d, rot, page, dtype, interleaved, mscale=1.0, ragged=False, extra=0, pos_dtype=torch.int32, theta=10000.0, in_place=False):
    n = sum(counts)
    q, k, v = rand((n + extra, hq, d), dtype, 1), rand((n + extra, hkv, d), dtype, 2), rand((n + extra, hkv, d), dtype, 3)
    inv_freq, _ = amp.rope_frequencies(rot, theta) if rot else (torch.zeros(0, device="cuda"), 1.0)
    place = ac.tokens(pos, counts)
    width = max([1] + [p // page + 1 for _, p in place])
    pool = len(pos) * width + 2
    table = torch.randperm(pool, generator=torch.Generator().manual_seed(4))[:len(pos) * width].to(torch.int32).view(len(pos), width).cuda()
    kc, vc = rand((pool, page, hkv, d), dtype, 5), rand((pool, page, hkv, d), dtype, 6)
    k0, v0 = kc.clone(), vc.clone()
    cu = None
    if ragged:
        cu = torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 9.0)
    src = q.clone()
    if in_place:
        out = q
    got = amp.rope_append(q, k, v, torch.tensor(pos, dtype=pos_dtype, device="cuda"), inv_freq, kc, vc, table, cu=cu, interleaved=interleaved,
                          mscale=mscale, out=out)
    assert got is out
    want, tol = expect(src[:n], place, inv_freq, interleaved, mscale)
    assert ((got[:n].double() - want).abs() <= tol).all()
    assert torch.equal(got[:n, :, rot:], src[:n, :, rot:])
    assert torch.equal(got[n:], src[n:]) if in_place else (got[n:] == 9.0).all()
    want, tol = expect(k[:n], place, inv_freq, interleaved, mscale)
    for row, (b, p) in enumerate(place):
        if p < 0:
            continue
        at = int(table[b, p // page])
        assert ((kc[at, p % page].double() - want[row]).abs() <= tol[row]).all()
        assert torch.equal(vc[at, p % page], v[row])
        k0[at, p % page], v0[at, p % page] = kc[at, p % page], v[row]
    assert torch.equal(kc, k0) and torch.equal(vc, v0)                  # nothing else was written


@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hq,hkv,d,rot", [(32, 8, 128, 128), (8, 2, 128, 64), (6, 1, 64, 64), (5, 5, 256, 32), (4, 2, 80, 80), (4, 2, 96, 48), (3, 1, 72, 72),
                                          (2, 1, 128, 2), (2, 2, 128, 126), (1, 1, 8, 6), (2, 1, 1024, 1024), (40, 20, 16, 16), (2, 1, 64, 0)])
def test_heads_and_rotated_parts(amp, dtype, interleaved, hq, hkv, d, rot):
    run(amp, [0, 1, 77, 1000, -1, -3], [2] * 6, hq, hkv, d, rot, 16, dtype, interleaved)


@pytest.mark.parametrize("page", [1, 3, 16, 100])
@pytest.mark.parametrize("in_place", [False, True])
def test_ragged_rows(amp, page, in_place):
    """Empty sequences, rows behind the last one"""
    run(amp, [7, 0, 99, 3, 1], [1, 0, 33, 5, 0], 8, 2, 64, 64, page, B, False, ragged=True, extra=4, mscale=1.25, in_place=in_place)
    run(amp, [7, 0, 99, 3, 1], [1, 0, 33, 5, 0], 8, 2, 64, 30, page, B, True, ragged=True, extra=4, in_place=in_place)


@pytest.mark.parametrize("seqs", [32, 33, 300])
def test_rows_of_many_sequences(amp, seqs):
    """Sequences found by a warp, and by the block"""
    counts = torch.randint(0, 3, (seqs,), generator=torch.Generator().manual_seed(seqs)).tolist()
    counts[-1] = 2
    run(amp, [(7 * b) % 50 for b in range(seqs)], counts, 4, 2, 64, 64, 16, H, False, ragged=True, extra=3)


@pytest.mark.parametrize("p", [131071, (1 << 20) - 1, (1 << 30) - 2])
def test_far_positions(amp, p):
    """The angle is exact where an fp32 product is off by radians"""
    d = 128
    for theta in (10000.0, 500000.0):
        inv_freq, _ = amp.rope_frequencies(d, theta)
        q = rand((2, 4, d), H, 8)
        got = amp.rope(q, torch.tensor([p], dtype=torch.int64, device="cuda"), inv_freq)
        want, tol = expect(q, [(0, p), (0, p + 1)], inv_freq, False, 1.0)
        assert ((got.double() - want).abs() <= tol).all()


def test_strides_and_alignment(amp):
    """q, k, v out of a packed row; the same at an odd address (value by value); caches kept per head; rope_append == rope"""
    hq, hkv, d = 4, 2, 64
    inv_freq, _ = amp.rope_frequencies(d)
    pos = torch.tensor([30, 5], device="cuda")
    table = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device="cuda")
    flat = rand((4 * (hq + 2 * hkv) * d + 8,), H, 9)
    results = []
    for shift in (0, 1, 8):
        packed = torch.empty_like(flat)[shift:shift + 4 * (hq + 2 * hkv) * d].view(4, -1, d)
        packed.copy_(flat[:packed.numel()].view(packed.shape))
        for per_head in (False, True):
            kc, vc = (torch.zeros((6, 16, hkv, d), dtype=H, device="cuda") for _ in range(2))
            if per_head:
                kc, vc = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (kc, vc))
            q = amp.rope_append(packed[:, :hq], packed[:, hq:hq + hkv], packed[:, hq + hkv:], pos, inv_freq, kc, vc, table)
            results.append((q, kc, vc))
            assert torch.equal(q, amp.rope(packed[:, :hq], pos, inv_freq))
    for r in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, results[0]))
    assert results[0][1].any() and results[0][2].any()


def test_tokens_without_a_place_are_not_stored(amp):
    inv_freq, _ = amp.rope_frequencies(64)
    q, k, v = rand((5, 2, 64), H, 1), rand((5, 1, 64), H, 2), rand((5, 1, 64), H, 3)
    kc, vc = (torch.zeros((3, 16, 1, 64), dtype=H, device="cuda") for _ in range(2))
    table = torch.tensor([[0, 9], [-1, 0], [3, 3], [2, 2], [1, 1]], dtype=torch.int32, device="cuda")
    pos = torch.tensor([16, 0, 5, 32, 1 << 50], dtype=torch.int64, device="cuda")
    got = amp.rope_append(q, k, v, pos, inv_freq, kc, vc, table)
    assert not kc.any() and not vc.any() and torch.isfinite(got).all()
    amp.rope_append(q, k, v, pos, inv_freq, kc, vc, table[:, :0])
    assert not kc.any()


def test_refusals(amp):
    inv_freq, _ = amp.rope_frequencies(64)
    q, k, v = rand((2, 4, 64), H, 1), rand((2, 2, 64), H, 2), rand((2, 2, 64), H, 3)
    kc, vc = (torch.zeros((3, 16, 2, 64), dtype=H, device="cuda") for _ in range(2))
    table, pos = torch.zeros((2, 3), dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    f = amp.rope_append
    bad = [
        (RuntimeError, lambda: f(q.cpu(), k, v, pos, inv_freq, kc, vc, table)),
        (RuntimeError, lambda: f(q, k, v, pos, inv_freq.cpu(), kc, vc, table)),
        (TypeError, lambda: f(q.float(), k, v, pos, inv_freq, kc, vc, table)),
        (TypeError, lambda: f(q, k.to(B), v, pos, inv_freq, kc, vc, table)),
        (ValueError, lambda: f(q, k, v, pos, inv_freq.half(), kc, vc, table)),
        (ValueError, lambda: f(q, k, v, pos, torch.zeros(33, device="cuda"), kc, vc, table)),
        (ValueError, lambda: f(q, k[:, :1], v, pos, inv_freq, kc, vc, table)),
        (ValueError, lambda: f(q, k[:, :1], v[:, :1], pos, inv_freq, kc, vc, table)),
        (ValueError, lambda: f(q[:1], k, v, pos[:1], inv_freq, kc, vc, table[:1])),
        (ValueError, lambda: f(q, k, v, pos, inv_freq, kc, vc[:2], table)),
        (TypeError, lambda: f(q, k, v, pos, inv_freq, kc, vc, table[:1])),
        (ValueError, lambda: amp.rope(q, torch.zeros(3, dtype=torch.int32, device="cuda"), inv_freq)),
        (ValueError, lambda: amp.rope(q, pos, inv_freq, out=q.new_empty((2, 4, 32)))),
        (ValueError, lambda: amp.rope(q[:, :2], pos, inv_freq, out=q.view(-1)[:2 * 2 * 64].view(2, 2, 64))),
        (ValueError, lambda: amp.rope(q, pos, inv_freq, out=q[:, :1].clone().expand(2, 4, 64))),
        (ValueError, lambda: f(q, k, v, pos, inv_freq, kc[:1].expand(3, 16, 2, 64), vc, table)),
        (RuntimeError, lambda: amp.rope(rand((1, 1, 1040), H, 1), pos[:1], inv_freq)),
    ]
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            pytest.fail("call %d was taken" % i)


@pytest.mark.parametrize("layers", [None, 1, 5])
@pytest.mark.parametrize("page,hkv,d,dtype", [(1, 1, 8, H), (16, 2, 64, H), (16, 8, 128, B), (100, 3, 128, H), (256, 8, 256, H), (7, 1, 8, torch.float32)])
def test_copy_pages(amp, layers, page, hkv, d, dtype):
    pages = 40
    shape = (pages, page, hkv, d) if layers is None else (layers, pages, page, hkv, d)
    a, b = rand(shape, dtype, 1), rand(shape, dtype, 2)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(3)).tolist()
    src, dst = order[:17] + [order[0]], order[17:34] + [order[39]]      # one source twice
    wa, wb = a.clone(), b.clone()
    for w in (wa, wb):
        for s, t in zip(src, dst):
            w.select(0 if layers is None else 1, t).copy_(w.select(0 if layers is None else 1, s))
    caches = [a, b]
    assert amp.copy_pages(caches, torch.tensor(src), dst) is caches
    assert torch.equal(a, wa) and torch.equal(b, wb)
    amp.copy_pages([a], [5], [5])
    amp.copy_pages([a], [], [])
    amp.copy_pages([], [1], [2])
    assert torch.equal(a, wa)


def test_copy_many_pages_of_many_caches(amp):
    """More pages and caches than one launch takes"""
    caches = [rand((700, 1, 1, 8), H, i) for i in range(40)]
    want = [c.clone() for c in caches]
    for w in want:
        w[350:] = w[:350]
    amp.copy_pages(caches, list(range(350)), list(range(350, 700)))
    assert all(torch.equal(a, b) for a, b in zip(caches, want))


def test_copy_pages_layouts(amp):
    """Pages kept per head, caches interleaved in one tensor, layers inside a page's stride"""
    base = rand((10, 2, 3, 4, 16, 64), H, 1)                             # (pages, k/v, layers, kv_heads, page_size, dim)
    caches = [base[:, i].transpose(0, 1).transpose(2, 3) for i in range(2)]
    want = base.clone()
    want[7] = want[2]
    amp.copy_pages(caches, [2], [7])
    assert torch.equal(base, want)


def test_copy_refusals(amp):
    a = rand((4, 10, 16, 2, 64), H, 1)
    before = a.clone()
    f = amp.copy_pages
    bad = [
        (RuntimeError, lambda: f([a], [0], [10])),
        (RuntimeError, lambda: f([a], [-1], [1])),
        (RuntimeError, lambda: f([a], [0, 1], [5, 5])),
        (RuntimeError, lambda: f([a], [0, 1], [1, 2])),
        (RuntimeError, lambda: f([a], [0, 1], [1, 0])),
        (RuntimeError, lambda: f([a], [3, 3], [3, 4])),
        (ValueError, lambda: f([a], [0, 1], [2])),
        (TypeError, lambda: f([a], torch.tensor([0], device="cuda"), [1])),
        (TypeError, lambda: f([a], [0.5], [1])),
        (TypeError, lambda: f([a], [1 << 40], [1])),
        (RuntimeError, lambda: f([a.cpu()], [0], [1])),
        (ValueError, lambda: f([a, a[:2]], [0], [1])),
        (ValueError, lambda: f([a[:, :, ::2]], [0], [1])),
        (ValueError, lambda: f([a[0, 0]], [0], [1])),
        (RuntimeError, lambda: f([a[:, :1].expand(4, 10, 16, 2, 64)], [0], [1])),
        (RuntimeError, lambda: f([a[..., :4].contiguous()[:, :, :1, :1]], [0], [1])),
    ]
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            pytest.fail("call %d was taken" % i)
    assert torch.equal(a, before)
