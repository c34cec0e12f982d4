"""CPU-only: bundles add the biases of their linears, and only those (the launches stood in for by products in torch)."""
import pytest
import torch

from ampstein_b200 import exl3, models


@pytest.fixture
def launches(monkeypatch):
    """Every launch leaves 1 in all outputs"""
    ones = []
    monkeypatch.setattr(exl3, "ptr_array", lambda values, device=None: torch.tensor(list(values), dtype=torch.int64))
    for name in ("mgemm", "mgemm_rms_norm_res", "mgemm_normed"):
        monkeypatch.setattr(exl3, name, lambda *a, **k: [t.fill_(1.0) for t in ones])
    return ones


def linear(n, bias):
    return models.LinearEXL3(torch.zeros((16, n // 16, 64), dtype=torch.int16), torch.ones(256), torch.ones(n),
                             bias=None if bias is None else torch.full((n,), bias, dtype=torch.float16))


@pytest.mark.parametrize("biases", [(None, None, None), (2.0, None, -3.0), (0.5, 1.5, 2.5)])
def test_sliced(launches, biases):
    outs = [torch.zeros((1, 2, n), dtype=torch.float16) for n in (256, 128, 128)]
    launches.extend(outs)
    bundle = models.Sliced([linear(n, b) for n, b in zip((256, 128, 128), biases)], outs)
    x = torch.zeros((1, 2, 256), dtype=torch.float16)
    for got in (bundle.run(x), bundle.run_norm(x, x, None, 1e-5, x), bundle.run_normed(x, None, None, 1e-5)):
        assert [t.unique().tolist() for t in got] == [[1.0 + (b or 0.0)] for b in biases]
        assert all(a.data_ptr() == b.data_ptr() for a, b in zip(got, outs))


@pytest.mark.parametrize("biases", [(None, None), (None, -3.0), (0.5, 1.5)])
def test_multi(launches, biases):
    out = torch.zeros((2, 2, 128), dtype=torch.float16)
    launches.append(out)
    bundle = models.Multi([linear(128, b) for b in biases], out)
    x = torch.zeros((1, 2, 256), dtype=torch.float16)
    for got in (bundle.run(x), bundle.run_norm(x, x, None, 1e-5, x), bundle.run_normed(x, None, None, 1e-5)):
        assert [t.unique().tolist() for t in got] == [[1.0 + (b or 0.0)] for b in biases] and got.data_ptr() == out.data_ptr()
