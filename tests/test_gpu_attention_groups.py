"""Many query heads on one key-value head: a single token has more rows than the few-token form takes."""
import pytest

torch = pytest.importorskip("torch")
import attention_cases as ac  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("wide", [0, 200])
@pytest.mark.parametrize("hq,hkv,d,dtype", [(64, 1, 64, torch.float16), (65, 1, 128, torch.bfloat16), (128, 1, 128, torch.float16), (200, 1, 64, torch.bfloat16),
                                            (260, 2, 64, torch.float16), (129, 1, 256, torch.bfloat16)])
@pytest.mark.parametrize("counts", [[1, 1, 1, 1, 1], [2, 2, 2, 2, 2], [1, 0, 3, 1, 20]])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
def test_large_groups(counts, hq, hkv, d, dtype, wide, window, sinks):
    import ampstein_b200 as amp
    pos = [0, 70, 300, -1, 129]
    k, v, table = ac.paged(pos, counts, 16, hkv, d, dtype, window, sinks, seed=hq, wide=wide)
    q = torch.randn((sum(counts), hq, d), generator=torch.Generator().manual_seed(d)).to(dtype).cuda()
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    ragged = len(set(counts)) > 1
    for cuts in ([True] if ragged else [False, True]):
        lse = torch.zeros((q.shape[0], hq), device="cuda")
        out = amp.paged_attention(q, k, v, table, torch.tensor(pos, device="cuda"), cu=torch.tensor(cu, dtype=torch.int32, device="cuda") if cuts else None,
                                  window=window, sinks=sinks, lse=lse)
        want, wlse, tol, ltol = ac.attention(q, k, v, table, pos, counts, window, sinks, d ** -0.5)
        assert torch.isfinite(out).all() and ((out.double() - want).abs() <= tol).all()
        live = ~torch.isinf(wlse)
        assert torch.equal(torch.isinf(lse), ~live) and ((lse.double() - wlse)[live].abs() <= ltol[live]).all()
