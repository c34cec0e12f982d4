"""CPU-only: a bundle takes any number of rows up to that of its buffers (the launches stood in for by fills of what they are given)."""
import pytest
import torch

from ampstein_b200 import exl3, models


@pytest.fixture
def seen(monkeypatch):
    seen = []
    monkeypatch.setattr(exl3, "ptr_array", lambda values, device=None: torch.tensor(list(values), dtype=torch.int64))
    monkeypatch.setattr(exl3, "mgemm", lambda x, B, C, *a: seen.append((x.shape, C)) or C.fill_(1.0))
    monkeypatch.setattr(exl3, "mgemm_rms_norm_res", lambda x, res, w, eps, y, B, C, *a: seen.append((x.shape, C)) or C.fill_(1.0))
    monkeypatch.setattr(exl3, "mgemm_normed", lambda y, ssq, w, eps, B, C, *a: seen.append((y.shape, C)) or C.fill_(1.0))
    return seen


def linear(n):
    return models.LinearEXL3(torch.zeros((16, n // 16, 64), dtype=torch.int16), torch.ones(256), torch.ones(n))


def calls(bundle, x):
    yield bundle.run(x)
    yield bundle.run_norm(x, x, None, 1e-5, x)
    yield bundle.run_normed(x, None, None, 1e-5)


@pytest.mark.parametrize("rows", [1, 3, 6, 7])
def test_sliced(seen, rows):
    outs = [torch.zeros((1, 7, n), dtype=torch.float16) for n in (256, 128, 128)]
    bundle = models.Sliced([linear(n) for n in (256, 128, 128)], outs)
    for got in calls(bundle, torch.zeros((1, rows, 256), dtype=torch.float16)):
        shape, carrier = seen[-1]
        assert shape[1] == rows and carrier.shape == (4, rows, 128) and carrier.is_contiguous()
        assert [t.shape for t in got] == [(1, rows, n) for n in (256, 128, 128)] and all(t.is_contiguous() for t in got)
        assert all(a.data_ptr() == b.data_ptr() for a, b in zip(got, outs))


@pytest.mark.parametrize("rows", [1, 3, 6, 7])
def test_multi(seen, rows):
    out = torch.zeros((2, 7, 128), dtype=torch.float16)
    bundle = models.Multi([linear(128) for _ in range(2)], out)
    for got in calls(bundle, torch.zeros((1, rows, 256), dtype=torch.float16)):
        assert seen[-1][0][1] == rows and seen[-1][1] is got
        assert got.shape == (2, rows, 128) and got.is_contiguous() and got.data_ptr() == out.data_ptr() and (got == 1.0).all()
        assert int(out.sum()) == 2 * rows * 128
        out.zero_()


@pytest.mark.parametrize("rows", [0, 8])
def test_more_rows_than_the_buffers_hold_are_refused(seen, rows):
    x = torch.zeros((1, rows, 256), dtype=torch.float16)
    for bundle in (models.Multi([linear(128) for _ in range(2)], torch.zeros((2, 7, 128), dtype=torch.float16)),
                   models.Sliced([linear(128), linear(256)], [torch.zeros((1, 7, n), dtype=torch.float16) for n in (128, 256)])):
        for call in (lambda: bundle.run(x), lambda: bundle.run_norm(x, x, None, 1e-5, x), lambda: bundle.run_normed(x, None, None, 1e-5)):
            with pytest.raises(ValueError):
                call()
    assert not seen
