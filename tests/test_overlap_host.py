"""CPU-only: which arrays of a call may share memory. The C entries refuse before any CUDA call (a call that gets through ends with a CUDA
error here, a positive code); the checks of the Python layer are compared with the places themselves."""
import ctypes
import random

import pytest
import torch

from ampstein_b200 import attention

H = torch.float16


def _lib():
    from ampstein_b200 import _lib
    return _lib, _lib.lib()


def strides(t):
    return [s if n > 1 else 0 for n, s in zip(t.shape[:-1], t.stride()[:-1])]


def run_attention(q, k, v, out, lse=None):
    mod, L = _lib()
    pos = torch.zeros(q.shape[0], dtype=torch.int32)
    args = [q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(), pos.data_ptr(), pos.data_ptr(), 0, 0, 0,
            *strides(q), *strides(out), *strides(k), *strides(v), 1, q.shape[0], q.shape[0], q.shape[1], k.shape[2], q.shape[2], k.shape[0], k.shape[1], 1, 0, 0,
            0, 0, 1.0]
    rc = L.amp_b200_attention(attention._ATTENTION.pack(*args), None)
    return rc < 0 and "overlap" in mod.last_error()


def run_rope(q, k, v, out, kc=None, vc=None):
    mod, L = _lib()
    pos, f = torch.zeros(q.shape[0], dtype=torch.int32), torch.zeros(q.shape[2] // 2)
    ptr = lambda t: 0 if t is None else t.data_ptr()                    # noqa: E731
    two = lambda t: [0, 0] if t is None else strides(t)                 # noqa: E731
    cache = [0] * 6 if kc is None else strides(kc) + strides(vc)
    args = [q.data_ptr(), ptr(k), ptr(v), out.data_ptr(), ptr(kc), ptr(vc), 0 if kc is None else pos.data_ptr(), pos.data_ptr(), 0, f.data_ptr(),
            *strides(q), *two(k), *two(v), *strides(out), *cache, 1, q.shape[0], q.shape[0], q.shape[1], 0 if k is None else k.shape[1], q.shape[2], q.shape[2], 0,
            *((0, 0, 0) if kc is None else (kc.shape[0], kc.shape[1], 1)), 0, 0, 1.0]
    rc = L.amp_b200_rope(attention._ROPE.pack(*args), None)
    return rc < 0 and "overlap" in mod.last_error()


def test_attention():
    n, h, d = 6, 4, 64
    buf = torch.zeros(1 << 16, dtype=H)
    q = buf[:n * h * d].view(n, h, d)
    both = torch.zeros((5, 2, 16, 2, d), dtype=H)
    rows = torch.zeros((5, 16, 2, 2, d), dtype=H)
    k, v = both[:, 0], both[:, 1]
    fine = torch.zeros_like(q)
    wide = torch.zeros((n, 3 * h, d), dtype=H)
    assert not run_attention(q, k, v, fine) and not run_attention(q, rows[:, :, 0], rows[:, :, 1], fine)
    assert not run_attention(q, k, v, buf[n * h * d:2 * n * h * d].view(n, h, d))                         # behind q
    assert not run_attention(wide[:, :h], k, v, wide[:, h:2 * h]) and not run_attention(wide[:, 2 * h:], k, v, wide[:, :h])
    heads = torch.zeros((n, h, 3, d), dtype=H)
    assert not run_attention(heads[:, :, 0], k, v, heads[:, :, 2])                                        # between q's heads
    every = torch.zeros((2 * n, h, d), dtype=H)
    assert not run_attention(every[0::2], k, v, every[1::2])                                              # between q's rows
    for shift in (0, 8, d, h * d, (n - 1) * h * d, n * h * d - 8):
        assert run_attention(q, k, v, buf[shift:shift + n * h * d].view(n, h, d)), shift                  # shifted in q
    assert run_attention(wide[:, :h], k, v, wide[:, h - 1:2 * h - 1])
    for c in (k, v):
        assert run_attention(q, k, v, c.reshape(-1)[:0].new_empty(0).set_(c.untyped_storage(), c.storage_offset(), (n, h, d), (h * d, d, 1)))
    lse = lambda t: t.view(-1).view(torch.float32)[:n * h].view(n, h)   # noqa: E731
    assert not run_attention(q, k, v, fine, torch.zeros((n, h)))
    for t in (fine, buf, both):
        assert run_attention(q, k, v, fine, lse(t))


def test_rope():
    n, h, d = 6, 4, 64
    packed = torch.zeros((n + 1, 4 * h, d), dtype=H)
    q, k, v, rest = (packed[:n, i * h:(i + 1) * h] for i in range(4))
    kc, vc = torch.zeros((5, 16, h, d), dtype=H), torch.zeros((5, 16, h, d), dtype=H)
    assert not run_rope(q, None, None, q) and not run_rope(q, None, None, rest) and not run_rope(q, None, None, torch.zeros((n, h, d), dtype=H))
    assert not run_rope(q, k, v, q, kc, vc) and not run_rope(q, k, v, rest, kc, vc) and not run_rope(q, k, k, q, kc, vc)
    assert run_rope(q, None, None, packed[1:, :h])                                                        # a row further
    assert run_rope(q, None, None, packed[:n, 1:h + 1])
    assert run_rope(q, k, v, k, kc, vc) and run_rope(q, k, v, v, kc, vc)
    assert run_rope(q, k, v, q, kc, kc) and run_rope(q, k, v, q, kc[:4], kc[1:])
    for inside in (kc, vc):
        t = inside[1:2].reshape(16, h, d)[:n]
        assert run_rope(t, k, v, q, kc, vc) and run_rope(q, t, v, q, kc, vc) and run_rope(q, k, t, q, kc, vc) and run_rope(q, k, v, t, kc, vc)


def test_copies():
    mod, L = _lib()

    def run(caches):
        arr = lambda t, xs: (t * len(xs))(*xs)                          # noqa: E731
        c = caches[0]
        return L.amp_b200_copy_pages(arr(ctypes.c_void_p, [t.data_ptr() for t in caches]), arr(ctypes.c_long, [t.stride(0) * 2 for t in caches]),
                                     arr(ctypes.c_long, [t.stride(1) * 2 for t in caches]), len(caches), c.shape[0], c.shape[1], c[0, 0].numel() * 2,
                                     arr(ctypes.c_int, [0]), arr(ctypes.c_int, [1]), 1, None) < 0 and "overlap" in mod.last_error()
    pool = torch.zeros((3, 9, 2, 4, 1, 8), dtype=H)
    k, v = pool[:, :, 0], pool[:, :, 1]
    assert not run([k, v]) and not run([k, k]) and not run([k[:, :4], v[:, 2:6], k[:, 4:8]]) and not run([k[:1], k[1:2], k[2:]])
    assert run([k[:, :5], k[:, 3:8]]) and run([k, v, k[:, :1].expand(3, 9, 4, 1, 8)][:2] + [pool.view(3, 18, 4, 1, 8)[:, 1:10]])


def test_the_python_checks_against_the_places_themselves():
    rng = random.Random(7)
    places = torch.arange(4000)
    shared = refused = 0
    for _ in range(4000):
        def view():
            shape = [rng.choice((1, 2, 3, 5)), rng.choice((1, 2, 4)), rng.choice((1, 4, 8))]
            inner = shape[2]
            a, b = sorted((inner * rng.randint(1, 6), inner * rng.choice((4, 8, 12, 24, 30))))
            st = rng.choice(((b, a, 1), (a, b, 1), (0, a, 1)))
            return torch.as_strided(places, shape, st, rng.randint(0, 200))
        t, u = view(), view()
        truth = bool(set(t.reshape(-1).tolist()) & set(u.reshape(-1).tolist()))
        got = attention._share(t, u)
        assert got or not truth, (t.shape, t.stride(), t.storage_offset(), u.shape, u.stride(), u.storage_offset())
        shared += truth
        refused += got and not truth
    assert shared > 500 and refused < 800
    assert not attention._share(places[:0], places)


@pytest.mark.parametrize("n", [1, 6])
def test_layouts_that_do_not_share(n):
    packed = torch.zeros((n, 12, 64), dtype=H)
    heads = torch.zeros((n, 4, 3, 64), dtype=H)
    pages = torch.zeros((5, 2, 16, 2, 64), dtype=H)
    for a, b in ((packed[:, :4], packed[:, 4:]), (heads[:, :, 0], heads[:, :, 1]), (pages[:, 0], pages[:, 1]), (pages[0], pages[1:]),
                 (packed[:, ::2], packed[:, 1::2]), (pages[:, 0].transpose(1, 2), pages[:, 1].transpose(1, 2))):
        assert not attention._share(a, b) and not attention._share(b, a) and attention._share(a, a)
