"""CPU-only: bookkeeping of the paged cache (page copies done by torch), and what the attention operators refuse before any launch."""
import ctypes
import random

import pytest
import torch

from ampstein_b200 import attention, models


@pytest.fixture
def cache(monkeypatch):
    def copy(caches, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        for c in caches:
            c[:, dst] = c[:, src]
        return caches
    monkeypatch.setattr(attention, "copy_pages", copy)
    return models.PagedCache(2, 12, 4, 1, 8, 5, 6, dtype=torch.float32, device="cpu")


def write(c, slot, tokens, value):
    """What rope_append does: the new tokens' values into the pages that the table names"""
    at = c.extend(slot, tokens)
    for p in range(at, at + tokens):
        page = int(c.table[slot, p // 4])
        assert page >= 0
        c.k[:, page, p % 4] = value
        c.v[:, page, p % 4] = -value
    return at


def read(c, slot):
    return [float(c.k[1, int(c.table[slot, p // 4]), p % 4, 0, 0]) for p in range(c.length(slot)) if c.table[slot, p // 4] >= 0]


def test_pages_come_and_go(cache):
    a, b = cache.add(), cache.add()
    assert (a, b) == (0, 1) and cache.length(a) == 0 and cache.free_pages == 12
    assert write(cache, a, 5, 1.0) == 0 and write(cache, a, 3, 2.0) == 5 and cache.free_pages == 10
    assert write(cache, b, 4, 3.0) == 0 and write(cache, b, 0, 0.0) == 4
    assert read(cache, a) == [1.0] * 5 + [2.0] * 3 and read(cache, b) == [3.0] * 4
    assert (cache.table[a, 2:] == -1).all()
    cache.free(a)
    assert cache.free_pages == 11 and (cache.table[a] == -1).all()
    with pytest.raises(ValueError):
        cache.length(a)
    assert cache.add() == a


def test_forks_share_until_they_write(cache):
    a = cache.add()
    write(cache, a, 6, 1.0)
    b = cache.fork(a)
    assert cache.free_pages == 10 and torch.equal(cache.table[a], cache.table[b])
    write(cache, b, 1, 2.0)                                             # into the half-filled page: b's own from here on
    assert cache.free_pages == 9 and cache.table[a, 0] == cache.table[b, 0] and cache.table[a, 1] != cache.table[b, 1]
    write(cache, a, 1, 3.0)                                             # a's page is its own again: no copy
    assert cache.free_pages == 9
    assert read(cache, a) == [1.0] * 6 + [3.0] and read(cache, b) == [1.0] * 6 + [2.0]
    write(cache, a, 1, 3.0)
    c = cache.fork(a)                                                   # whole pages: nothing to copy
    write(cache, c, 2, 4.0)
    assert cache.free_pages == 8 and read(cache, a) == [1.0] * 6 + [3.0] * 2 and read(cache, c)[-2:] == [4.0] * 2
    cache.free(a)
    cache.free(b)
    assert read(cache, c) == [1.0] * 6 + [3.0] * 2 + [4.0] * 2
    cache.free(c)
    assert cache.free_pages == 12


def test_no_room_changes_nothing(cache):
    a, b = cache.add(), cache.add()
    write(cache, a, 24, 1.0)
    with pytest.raises(RuntimeError):
        cache.extend(a, 1)                                              # the table's row is full
    write(cache, b, 22, 2.0)
    c = cache.fork(b)
    before = cache.table.clone()
    with pytest.raises(RuntimeError):
        cache.extend(c, 1)                                              # no page for the copy
    assert torch.equal(before, cache.table) and cache.length(c) == 22 and cache.free_pages == 0
    with pytest.raises(ValueError):
        cache.extend(c, -1)
    cache.fork(c)
    cache.fork(c)
    with pytest.raises(RuntimeError):
        cache.fork(c)                                                   # no slot


def test_windows_give_pages_up(cache):
    a = cache.add()
    write(cache, a, 19, 1.0)
    cache.leave_behind(a, window=6, sinks=1)                            # the next token, at 19, sees 14 .. 19 and 0
    assert cache.table[a].tolist().count(-1) == 3 and cache.table[a, 0] >= 0 and cache.table[a, 3] >= 0 and (cache.table[a, 1:3] == -1).all()
    b = cache.fork(a)
    cache.leave_behind(b, window=1)                                     # sees itself alone: position 19 and its page
    assert cache.table[b, 0] == -1 and cache.table[a, 0] >= 0 and cache.table[b, 4] >= 0
    with pytest.raises(ValueError):
        cache.leave_behind(a, window=0)
    cache.free(a)
    cache.free(b)
    assert cache.free_pages == 12


def test_rejected_drafts_are_taken_back(cache):
    a = cache.add()
    write(cache, a, 7, 1.0)
    write(cache, a, 3, 2.0)
    cache.truncate(a, 8)
    assert cache.length(a) == 8 and cache.free_pages == 10 and cache.table[a, 2] == -1
    cache.truncate(a, 8)
    with pytest.raises(ValueError):
        cache.truncate(a, 9)
    cache.truncate(a, 0)
    assert cache.free_pages == 12


def test_compaction_keeps_the_sequences(cache):
    a, b, c = cache.add(), cache.add(), cache.add()
    for i in range(3):
        for s in (a, b, c):
            write(cache, s, 4, 10.0 * s + i)
    d = cache.fork(b)
    cache.free(a)
    want = {s: read(cache, s) for s in (b, c, d)}
    assert cache.compact() == 6
    assert {s: read(cache, s) for s in want} == want and cache.table.max() == 5 and cache.free_pages == 6
    write(cache, d, 1, 7.0)
    assert read(cache, b) == want[b] and cache.compact() == 7


def test_any_order_of_calls(cache):
    """Against a plain list per sequence"""
    rng, model = random.Random(1), {}
    for step in range(1500):
        op = rng.choice(("add", "write", "write", "write", "fork", "free", "truncate", "compact"))
        slot = rng.choice(list(model)) if model else None
        try:
            if op == "add":
                model[cache.add()] = []
            elif slot is None:
                continue
            elif op == "write":
                n = rng.randint(0, 7)
                write(cache, slot, n, float(step))
                model[slot] += [float(step)] * n
            elif op == "fork":
                model[cache.fork(slot)] = list(model[slot])
            elif op == "free":
                cache.free(slot)
                del model[slot]
            elif op == "truncate":
                n = rng.randint(0, len(model[slot]))
                cache.truncate(slot, n)
                del model[slot][n:]
            else:
                cache.compact()
        except RuntimeError:
            pass
        for s, want in model.items():
            assert read(cache, s) == want, (step, op)
        pages = {int(p) for s in model for p in cache.table[s] if p >= 0}
        assert cache.free_pages == 12 - len(pages) and len(set(cache._free)) == len(cache._free) and not pages & set(cache._free)


def test_sizes_are_checked():
    with pytest.raises(ValueError):
        models.PagedCache(1, 0, 4, 1, 8, 1, 1, device="cpu")


def test_frequencies():
    f, m = attention.rope_frequencies(8, 10000.0, device="cpu")
    assert m == 1.0 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001]))
    f4, _ = attention.rope_frequencies(8, scaling=dict(kind="linear", factor=4.0), device="cpu")
    assert torch.allclose(f4 * 4, f)
    n, _ = attention.rope_frequencies(8, scaling=dict(kind="ntk", factor=4.0), device="cpu")
    assert n[0] == 1.0 and abs(float(n[-1]) * 4 / 0.001 - 1) < 1e-5      # the slowest is stretched by the whole factor
    l, _ = attention.rope_frequencies(128, 500000.0, dict(kind="llama3", factor=8.0), device="cpu")
    base, _ = attention.rope_frequencies(128, 500000.0, device="cpu")
    assert l[0] == base[0] and abs(float(l[-1] * 8 / base[-1]) - 1) < 1e-5 and ((l <= base) & (l * 8.00001 >= base)).all()
    y, m = attention.rope_frequencies(128, scaling=dict(kind="yarn", factor=16.0), device="cpu")
    base, _ = attention.rope_frequencies(128, device="cpu")
    assert y[0] == base[0] and abs(float(y[-1] * 16 / base[-1]) - 1) < 1e-5 and abs(m - 1.2772588722239782) < 1e-12
    for bad in (dict(rot=7), dict(rot=0), dict(rot=8, theta=0.0), dict(rot=8, scaling=dict(kind="spiral")), dict(rot=8, scaling=dict(kind="linear", factor=0.0)),
                dict(rot=8, scaling=dict(kind="linear", factor=2.0, beta_fast=3.0)), dict(rot=8, scaling=dict(kind="yarn", factor=2.0, beta_fast=1.0, beta_slow=2.0)),
                dict(rot=8, scaling=dict(kind="llama3", factor=2.0, high_freq_factor=1.0))):
        with pytest.raises(ValueError):
            attention.rope_frequencies(device="cpu", **bad)


def _lib():
    from ampstein_b200 import _lib
    return _lib, _lib.lib()


def test_entries_refuse_before_any_cuda_call():
    """(no GPU here: an argument that got through would end with a CUDA error, a positive code)"""
    mod, L = _lib()
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(buf)
    p += (-p) % 16
    rope = dict(q=p, k=p, v=p, q_out=p, k_cache=p, v_cache=p, table=p, pos=p, cu=0, inv_freq=p, strides=[64] * 15, tokens=4, seqs=2, heads=2, kv_heads=1,
                dim=64, rot=64, interleaved=0, pages=4, page_size=16, max_pages=3, bf16=0, pos64=0, mscale=1.0)
    att = dict(q=p, k_cache=p, v_cache=p, out=p, lse=0, table=p, pos=p, cu=0, workspace=0, workspace_bytes=0, strides=[64] * 11, tokens=4, seqs=2, heads=2,
               kv_heads=1, dim=64, pages=4, page_size=16, max_pages=3, window=0, sinks=0, bf16=0, pos64=0, scale=1.0)

    def run(name, pack, args, **change):
        a = dict(args, **change)
        flat = [x for v in a.values() for x in (v if isinstance(v, list) else [v])]
        return getattr(L, name)(pack.pack(*flat), None), mod.last_error()

    for change in (dict(q=0), dict(q_out=0), dict(pos=0), dict(inv_freq=0), dict(tokens=-1), dict(tokens=5), dict(tokens=1 << 25), dict(seqs=-1), dict(dim=0), dict(dim=2048),
                   dict(rot=65), dict(rot=63), dict(rot=128), dict(heads=0), dict(k=0), dict(v_cache=0), dict(table=0), dict(page_size=0), dict(pages=0), dict(max_pages=1 << 28),
                   dict(q=p + 1)):
        rc, text = run("amp_b200_rope", attention._ROPE, rope, **change)
        assert rc < 0 and text.startswith("rope"), (change, rc, text)
    for change in (dict(q=0), dict(out=0), dict(table=0), dict(pos=0), dict(tokens=-3), dict(tokens=5), dict(seqs=1 << 21, tokens=1 << 21), dict(heads=3, kv_heads=2),
                   dict(kv_heads=0), dict(dim=96), dict(pages=0), dict(page_size=0), dict(max_pages=1 << 28), dict(window=-1), dict(sinks=-1), dict(q=p + 2),
                   dict(strides=[64] * 4 + [60] + [64] * 6), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=-3e38)):
        rc, text = run("amp_b200_attention", attention._ATTENTION, att, **change)
        assert rc < 0 and text.startswith("attention"), (change, rc, text)
    assert run("amp_b200_rope", attention._ROPE, rope, tokens=0)[0] == 0 and run("amp_b200_attention", attention._ATTENTION, att, seqs=0)[0] == 0
    assert L.amp_b200_attention(None, None) < 0 and L.amp_b200_rope(None, None) < 0

    def copy(src, dst, pages=8, page_bytes=64, ls=512, ps=64, n_caches=1, base=p, layers=1):
        n = len(src)
        arr = lambda t, xs: (t * max(1, len(xs)))(*xs)                  # noqa: E731
        return L.amp_b200_copy_pages(arr(ctypes.c_void_p, [base]), arr(ctypes.c_long, [ls]), arr(ctypes.c_long, [ps]), n_caches, layers, pages, page_bytes,
                                     arr(ctypes.c_int, src), arr(ctypes.c_int, dst), n, None)
    for bad in (dict(src=[0], dst=[8]), dict(src=[-1], dst=[1]), dict(src=[0, 1], dst=[2, 2]), dict(src=[0, 1], dst=[1, 2]), dict(src=[0], dst=[1], page_bytes=72),
                dict(src=[0], dst=[1], ps=48), dict(src=[0], dst=[1], base=p + 8), dict(src=[0], dst=[1], base=0), dict(src=[0], dst=[1], pages=-1),
                dict(src=[0], dst=[1], layers=2, ls=256)):
        assert copy(**bad) < 0 and mod.last_error().startswith("copy_pages"), bad
    assert copy([], []) == 0 and copy([3, 4], [3, 4]) == 0 and copy([1], [2], n_caches=0) == 0
