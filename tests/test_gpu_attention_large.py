"""Scores of large magnitude: finite inputs whose softmax is a mean over the keys of the largest score."""
import math

import pytest

torch = pytest.importorskip("torch")
import attention_cases as ac  # noqa: E402

pytestmark = pytest.mark.gpu
H, B = torch.float16, torch.bfloat16


@pytest.mark.parametrize("wide", [0, 200])
@pytest.mark.parametrize("count", [1, 6, 150])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype,power,sign", [(H, 13, 1), (H, 13, -1), (H, 8, 1), (B, 13, 1), (B, 24, 1), (B, 24, -1), (B, 50, 1)]
                         + [(H, p, s) for p in (9, 10, 11, 12) for s in (1, -1)])
def test_far_scores(dtype, power, sign, d, count, wide):
    """q = 2^power everywhere, key j sign * 2^power (1 + c_j / 64) everywhere: the scores, 2^(2 power) d / 8 (1 + c_j / 64), are exact in fp32 and
    64-bit numbers and lie so far apart that all weights but those of the largest are 0 (2^(2 power - 9) d / 8 > 100 from power 8 on)"""
    import ampstein_b200 as amp
    hq, hkv, page, first = 4, 2, 16, 300
    g = torch.Generator().manual_seed(power + d + count)
    n = first + count
    c = torch.randint(0, 12, (n,), generator=g)
    c[n // 2:] += 3                                                     # the maximum moves late
    width = -(-n // page)
    k = (sign * 2.0 ** power * (1 + c / 64)).view(n, 1, 1).expand(n, hkv, d)
    v = torch.randn((n, hkv, d), generator=g)
    pad = width * page - n
    kc, vc = (torch.cat((t, torch.zeros((pad, hkv, d)))).view(width, page, hkv, d).to(dtype).cuda() for t in (k, v))
    table = torch.cat((torch.arange(width), torch.full((wide,), -1))).to(torch.int32).view(1, -1).cuda()
    q = torch.full((count, hq, d), 2.0 ** power, dtype=dtype, device="cuda")
    lse = torch.zeros((count, hq), device="cuda")
    out = amp.paged_attention(q, kc, vc, table, torch.tensor([first], device="cuda"), scale=0.125, lse=lse)
    u, vd = ac.U[dtype], vc.view(-1, hkv, d)[:n].double()
    for t in range(count):
        seen = sign * c[:first + t + 1]
        best = (seen == seen.max()).nonzero()[:, 0].cuda()
        want = vd[best].mean(0).repeat_interleave(hq // hkv, 0)
        # (equal weights, each off by u beside the sum; sums of so many values in fp32; the result is rounded)
        tol = u * want.abs() + vd[best].abs().mean(0).repeat_interleave(hq // hkv, 0) * (u + (len(best) + 64) * 2.0 ** -23) * 1.01 + 2.0 ** -24
        assert ((out[t].double() - want).abs() <= tol).all(), t
        score = 2.0 ** (2 * power) * d / 8 * sign * (1 + float(seen.max() * sign) / 64)
        # (score, its product with the scale in powers of two and back: three roundings)
        assert ((lse[t].double() - score - math.log(len(best))).abs() <= abs(score) * 2.0 ** -22 + 2.0 ** -20).all(), t
