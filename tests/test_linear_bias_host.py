"""CPU-only: where a linear's bias ends up (the launches stood in for by products in torch)."""
import pytest
import torch

from ampstein_b200 import exl3, models


@pytest.fixture
def lin(monkeypatch):
    monkeypatch.setattr(exl3, "exl3_gemm", lambda x, t, out, *a: out.fill_(1.0))
    monkeypatch.setattr(exl3, "exl3_gemm_silu_mul", lambda g, u, t, out, *a: out.fill_(1.0))
    monkeypatch.setattr(exl3, "exl3_gemm_recon", lambda x, *a: torch.ones((x.shape[0], 128), dtype=torch.float16))
    monkeypatch.setattr(exl3.GemmPlan, "__init__", lambda self, *a: None)
    monkeypatch.setattr(exl3.GemmPlan, "matches", lambda self, *a: True)
    monkeypatch.setattr(exl3.GemmPlan, "run", lambda self, x, *a: None if x.shape[0] == 3 else torch.ones((x.shape[0], 128), dtype=torch.float16))
    return models.LinearEXL3(torch.zeros((16, 8, 64), dtype=torch.int16), torch.ones(256), torch.ones(128))


@pytest.mark.parametrize("rows", [1, 3, 200])
@pytest.mark.parametrize("bias", [None, 2.0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_the_buffer_that_the_caller_gave_holds_the_result(lin, rows, bias, dtype):
    lin.bias = None if bias is None else torch.full((128,), bias, dtype=torch.float16)
    x, want = torch.zeros((rows, 256), dtype=torch.float16), 1.0 + (bias or 0.0)
    for call in (lin.forward, lambda x, out=None: lin.forward_silu_mul(x, x, out)):
        got = call(x)
        assert got.dtype == torch.float16 and (got == want).all()
        out = torch.zeros((rows, 128), dtype=dtype)
        got = call(x, out)
        assert got is out and (out == want).all()


def test_the_fused_residual_add_refuses_a_bias(lin, monkeypatch):
    monkeypatch.setattr(exl3, "exl3_gemm_add_res", lambda *a: "launched")
    x = torch.zeros((1, 256), dtype=torch.float16)
    assert lin.forward_add_res(x, x, x, None) == "launched"
    lin.bias = torch.ones(128, dtype=torch.float16)
    with pytest.raises(ValueError):
        lin.forward_add_res(x, x, x, None)


def test_shards_have_their_part_of_the_bias(lin):
    lin = models.LinearEXL3(torch.zeros((32, 32, 64), dtype=torch.int16), torch.ones(512), torch.ones(512), bias=torch.arange(512.0).half())
    parts = [models.cols(lin, [(0, 128), (384, 128)]), models.cols(lin, [(128, 256)])]
    assert torch.equal(torch.cat([p.bias for p in parts]), torch.cat((lin.bias[:128], lin.bias[384:], lin.bias[128:384])))
    parts = [models.rows(lin, k0, 256) for k0 in (0, 256)]
    assert torch.equal(sum(p.bias for p in parts if p.bias is not None), lin.bias)      # (once, whatever the number of shards)
    lin.bias = None
    assert models.cols(lin, [(0, 128)]).bias is None and models.rows(lin, 0, 128).bias is None
