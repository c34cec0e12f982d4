"""CPU-only: a page copy that fails leaves the paged cache as it was."""
import pytest
import torch

from ampstein_b200 import attention, models


def test_a_failed_copy_changes_nothing(monkeypatch):
    cache = models.PagedCache(2, 6, 4, 1, 8, 3, 6, dtype=torch.float32, device="cpu")
    a, hole = cache.add(), cache.add()
    cache.extend(hole, 4)
    cache.extend(a, 6)
    b = cache.fork(a)
    cache.free(hole)
    table, free = cache.table.clone(), cache.free_pages

    def fails(caches, src, dst):
        raise RuntimeError("copy_pages failed")

    monkeypatch.setattr(attention, "copy_pages", fails)
    for call in (lambda: cache.extend(b, 1), lambda: cache.extend(b, 9), cache.compact) * 2:
        with pytest.raises(RuntimeError, match="copy_pages failed"):
            call()
        assert cache.free_pages == free and torch.equal(cache.table, table) and cache.length(b) == 6
    monkeypatch.setattr(attention, "copy_pages", lambda caches, src, dst: [c[:, dst].copy_(c[:, src]) for c in caches])
    assert cache.extend(b, 1) == 6 and cache.free_pages == free - 1
    cache.free(a)
    cache.free(b)
    assert cache.free_pages == 6 and len(set(cache._free)) == 6
