"""The attention block with linears that have biases."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
from conftest import make_linear  # noqa: E402

pytestmark = pytest.mark.gpu

HIDDEN, HQ, HKV, D = 512, 4, 2, 128


def linear(k, n, seed, bias):
    from ampstein_b200.models import LinearEXL3
    trellis, suh, svh, _ = make_linear(k, n, 4, seed=seed)
    svh = (svh.astype(np.float32) / (1.2437 * k ** 0.5)).astype(np.float16)
    b = torch.randn(n, generator=torch.Generator().manual_seed(seed)).to(torch.float16).cuda() if bias else None
    return LinearEXL3(torch.from_numpy(trellis.view(np.int16)).cuda(), torch.from_numpy(suh).cuda(), torch.from_numpy(svh).cuda(), bias=b)


@pytest.mark.parametrize("rows", [1, 3, 33])
def test_biases_of_q_k_v(oracle, rows):
    """The block against its linears one by one, which add their biases themselves"""
    import ampstein_b200 as amp
    from ampstein_b200.models import PagedAttention, PagedCache, Sliced
    lins = [linear(HIDDEN, n * D, i, True) for i, n in enumerate((HQ, HKV, HKV))]
    o = linear(HQ * D, HIDDEN, 9, True)
    inv_freq, _ = amp.rope_frequencies(D)
    x = torch.randn((1, rows, HIDDEN), generator=torch.Generator().manual_seed(3)).to(torch.float16).cuda()
    caches = [PagedCache(1, 8, 16, HKV, D, 1, 8) for _ in range(2)]
    pos = [torch.tensor([c.extend(c.add(), rows)], device="cuda") for c in caches][0]
    outs = [torch.zeros((1, rows, w.out_features), dtype=torch.float16, device="cuda") for w in lins]
    got = PagedAttention(Sliced(lins, outs), o, caches[0], 0, D, inv_freq).run(x, pos, caches[0].table).float()
    q, k, v = (w.forward(x[0]).view(rows, -1, D) for w in lins)
    q = amp.rope_append(q, k, v, pos, inv_freq, caches[1].k[0], caches[1].v[0], caches[1].table)
    a = amp.paged_attention(q, caches[1].k[0], caches[1].v[0], caches[1].table, pos)
    want = o.forward(a.view(rows, -1)).float()
    # (two chains of linears within 1e-2 of the largest value each, the framework's bound for a linear)
    assert (got - want).abs().max() <= 2e-2 * want.abs().max()


def test_the_bias_of_o_reaches_the_buffer_of_a_captured_step(oracle):
    import ampstein_b200 as amp
    from ampstein_b200.models import DecodeGraph, PagedAttention, PagedCache, Sliced
    lins = [linear(HIDDEN, n * D, i, True) for i, n in enumerate((HQ, HKV, HKV))]
    o = linear(HQ * D, HIDDEN, 9, True)
    inv_freq, _ = amp.rope_frequencies(D)
    x = torch.randn((1, 1, HIDDEN), generator=torch.Generator().manual_seed(3)).to(torch.float16).cuda()
    cache = PagedCache(1, 8, 16, HKV, D, 1, 8)
    pos = torch.tensor([cache.extend(cache.add(), 1)], device="cuda")
    block = PagedAttention(Sliced(lins, [torch.zeros((1, 1, w.out_features), dtype=torch.float16, device="cuda") for w in lins]), o, cache, 0, D, inv_freq)
    out = torch.zeros((1, HIDDEN), dtype=torch.float16, device="cuda")
    graph = DecodeGraph(lambda: block.run(x, pos, cache.table, out=out))
    want = block.run(x, pos, cache.table)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    # (one linear, in its two calls)
    assert (out.float() - want.float()).abs().max() <= 1e-2 * want.float().abs().max()
