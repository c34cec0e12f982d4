"""One key far above a long context: what the many small weights add up to."""
import math

import pytest

torch = pytest.importorskip("torch")
import attention_cases as ac  # noqa: E402

pytestmark = pytest.mark.gpu
H, B = torch.float16, torch.bfloat16


@pytest.mark.parametrize("nats", [10.0, 15.0, 17.0, 17.4])
@pytest.mark.parametrize("dtype", [H, B])
@pytest.mark.parametrize("seqs,count,hkv", [(1, 1, 1), (150, 1, 4), (1, 70, 1), (150, 70, 4)])
def test_a_sink(nats, dtype, seqs, count, hkv):
    """Key 0 has the score `nats`, the others 0 (exactly: one term each); the sequences share their pages. Both forms, one sequence over
    the whole device (every part has a maximum of its own) and many (one maximum for all keys).

    Bounds, of the largest weight's 1: a rounded weight is off by u of itself, with fp16 at least by 2^-25 over 2^7, the lift of the prompt
    form (2^15 in the few-token form); the weights are added up in steps of 32 keys at least over 4 groups of warps, 2^-24 each time and
    64 within a step; exp2 2^-21 and its argument 2^-19.
    The products with the values: fp32 sums of n terms, whose error is n 2^-23 of the sum at most, each term cut to what fits beside it (a matrix
    instruction that brought its 16 products together first would be off by a sixteenth of that; this one does not promise it: at
    17.4 nats each product, 2^-25.1, is less than half a unit in the last place, 2^-24, of a sum of 1, and nothing of it is left there. That is the
    arithmetic of any sum in fp32, term by term. In the columns without a value of the sink the sum is small and keeps them, which is where
    a weight that was lost in its rounding shows)."""
    import ampstein_b200 as amp
    d, page, n = 64, 256, 131072
    first = n - count
    q = torch.zeros((seqs * count, hkv, d), dtype=dtype, device="cuda")
    q[:, :, 0] = 8.0
    k, v = (torch.zeros((n // page, page, hkv, d), dtype=dtype, device="cuda") for _ in range(2))
    k[0, 0, :, 0] = nats
    x = float(k[0, 0, 0, 0])                                            # 8 x / 8
    v[:] = 1.0
    v[0, 0, :, d // 2:] = 0.0                                           # (columns in which the sink has no value)
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").view(1, -1).expand(seqs, -1).contiguous()
    lse = torch.zeros((seqs * count, hkv), device="cuda")
    out = amp.paged_attention(q, k, v, table, torch.full((seqs,), first, device="cuda"), scale=0.125, lse=lse).double()
    u = ac.U[dtype]
    for t in (0, count - 1):
        others = first + t
        tail = others * math.exp(-x)
        got, glse = out[t::count], lse[t::count].double()
        for cols, want, top in ((slice(0, d // 2), 1.0, 1.0), (slice(d // 2, d), tail / (1 + tail), 0.0)):
            weights = tail * max(u, 2.0 ** -32 / math.exp(-x) if dtype == H else 0.0)      # roundings of the small weights
            tol = (weights + (top + tail) * (n * 2.0 ** -23 + 2.0 ** -18)) / (1 + tail) + want * (n / 128 * 2.0 ** -24 + 2.0 ** -17 + u) + 2.0 ** -24
            assert (got[..., cols] - want).abs().max() <= tol, (t, want, float((got[..., cols] - want).abs().max()), tol)
        assert (glse - x - math.log1p(tail)).abs().max() <= n / 128 * 2.0 ** -24 + 2.0 ** -17 + abs(x) * 2.0 ** -22
