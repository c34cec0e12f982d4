"""CPU-only: pages that a window gives up, beside tokens that have still to run and drafts that are taken back."""
import random

import pytest
import torch

from ampstein_b200 import attention, models

PAGE = 4


@pytest.fixture
def cache(monkeypatch):
    def copy(caches, src, dst):
        for c in caches:
            c[:, dst] = c[:, src]
        return caches
    monkeypatch.setattr(attention, "copy_pages", copy)
    return models.PagedCache(1, 80, PAGE, 1, 8, 3, 40, dtype=torch.float32, device="cpu")


def check(cache, slot, first, count, window, sinks):
    """Every announced token's page that one of the tokens first .. first + count - 1 sees is in the table"""
    for p in range(first, first + count):
        for j in range(min(p + 1, cache.length(slot))):
            if j > p - window or j < sinks:
                assert cache.table[slot, j // PAGE] >= 0, (p, j)


@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 1), (6, 1), (8, 0), (9, 5), (40, 3)])
@pytest.mark.parametrize("prompt", [1, 2, 5, 19, 37])
def test_single_tokens_in_both_orders(cache, prompt, window, sinks):
    """Pages given up between the announcement of a token and its run, and behind its run; over more than four pages"""
    before, after = cache.add(), cache.add()
    for slot in (before, after):
        cache.extend(slot, prompt)
    for _ in range(4 * PAGE + 3):
        at = cache.extend(before, 1)
        cache.leave_behind(before, window, sinks)
        check(cache, before, at, 1, window, sinks)
        at = cache.extend(after, 1)
        check(cache, after, at, 1, window, sinks)
        cache.leave_behind(after, window, sinks, pending=0)
        check(cache, after, at + 1, 1, window, sinks)
        kept = lambda slot: int((cache.table[slot] >= 0).sum())         # noqa: E731
        need = len({j // PAGE for j in range(at + 1) if j > at - window or j < sinks})
        assert kept(after) <= need + 1 and kept(before) <= need + 1


@pytest.mark.parametrize("window,sinks", [(1, 0), (6, 1), (9, 5), (17, 0)])
def test_drafts_that_are_taken_back(cache, window, sinks):
    rng = random.Random(window)
    slot = cache.add()
    cache.extend(slot, 21)
    for step in range(40):
        n = rng.randint(1, 4)
        at = cache.extend(slot, n)
        if step % 2:
            cache.leave_behind(slot, window, sinks)
        check(cache, slot, at, n, window, sinks)
        if step % 3:
            cache.leave_behind(slot, window, sinks)
        cache.truncate(slot, at + rng.randint(0, n))
        check(cache, slot, cache.length(slot), 1, window, sinks)


def test_tokens_that_are_named_as_pending(cache):
    slot = cache.add()
    cache.extend(slot, 30)
    cache.leave_behind(slot, 6, pending=30)                             # the prompt has still to run
    check(cache, slot, 0, 30, 6, 0)
    cache.extend(slot, 2)
    cache.leave_behind(slot, 6, pending=5)                              # announced by two calls
    check(cache, slot, 27, 5, 6, 0)
    assert cache.table[slot, 4] == -1 and cache.table[slot, 5] >= 0
    for bad in (-1, 33):
        with pytest.raises(ValueError):
            cache.leave_behind(slot, 6, pending=bad)


def test_no_truncation_to_where_given_up_pages_are_seen(cache):
    a = cache.add()
    cache.extend(a, 30)
    cache.leave_behind(a, 6, 1, pending=0)                              # pages 1 .. 5 (positions 4 .. 23): from 29 on none is seen
    table, free = cache.table.clone(), cache.free_pages
    b = cache.fork(a)
    for slot in (a, b):
        for tokens in (28, 24, 20, 5):
            with pytest.raises(ValueError):
                cache.truncate(slot, tokens)
    assert torch.equal(cache.table[a], table[a]) and cache.length(a) == 30 and cache.free_pages == free
    cache.truncate(a, 29)
    check(cache, a, cache.extend(a, 1), 1, 6, 1)
    cache.truncate(a, 4)                                                # in front of all that was given up: nothing is missing
    check(cache, a, cache.extend(a, 9), 9, 6, 1)
    cache.truncate(a, 5)
    cache.leave_behind(b, 20, pending=0)                                # a longer window looks back to more of them
    cache.truncate(b, 29)
    assert cache.length(a) == 5 and cache.length(b) == 29


def test_an_extension_by_nothing_leaves_the_pending_tokens(cache):
    slot = cache.add()
    cache.extend(slot, 21)
    at = cache.extend(slot, 9)
    assert cache.extend(slot, 0) == 30
    cache.leave_behind(slot, 6)
    check(cache, slot, at, 9, 6, 0)
