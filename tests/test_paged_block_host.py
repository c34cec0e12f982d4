"""CPU-only: what the attention block refuses before anything runs."""
import pytest
import torch

from ampstein_b200 import models


class Linear:
    def __init__(self, n):
        self.in_features = self.out_features = n


class Bundle:
    def __init__(self, *widths):
        self.linears = [Linear(n) for n in widths]


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_widths_that_fit(dim):
    cache = models.PagedCache(2, 2, 16, 2, dim, 1, 2, device="cpu")
    block = models.PagedAttention(Bundle(4 * dim, 2 * dim, 2 * dim), Linear(4 * dim), cache, 1, dim, None)
    assert block.k.data_ptr() == cache.k[1].data_ptr()


@pytest.mark.parametrize("dim", [32, 80, 96, 192, 512])
def test_heads_that_the_attention_cannot_read(dim):
    cache = models.PagedCache(1, 2, 16, 2, dim, 1, 2, device="cpu")
    with pytest.raises(ValueError, match="heads of %d" % dim):
        models.PagedAttention(Bundle(4 * dim, 2 * dim, 2 * dim), Linear(4 * dim), cache, 0, dim, None)
