"""Bundles and the attention block with fewer rows than their buffers have."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
from conftest import make_linear  # noqa: E402

pytestmark = pytest.mark.gpu


def linear(k, n, seed):
    from ampstein_b200.models import LinearEXL3
    trellis, suh, svh, _ = make_linear(k, n, 4, seed=seed)
    svh = (svh.astype(np.float32) / (1.2437 * k ** 0.5)).astype(np.float16)
    return LinearEXL3(torch.from_numpy(trellis.view(np.int16)).cuda(), torch.from_numpy(suh).cuda(), torch.from_numpy(svh).cuda())


@pytest.mark.parametrize("rows", [1, 2, 4, 5, 9, 16, 17, 40])
def test_rows_of_a_larger_bundle(rows):
    """The same bits as a bundle of its own size; what lies behind the rows stays"""
    from ampstein_b200.models import Multi, Sliced
    k, most = 512, 40
    x = torch.randn((1, rows, k), generator=torch.Generator().manual_seed(rows)).to(torch.float16).cuda()
    lins = [linear(k, n, i) for i, n in enumerate((512, 256, 256))]

    def sliced(m):
        outs = [torch.full((1, m, w.out_features), 7.0, dtype=torch.float16, device="cuda") for w in lins]
        return Sliced(lins, outs).run(x), outs

    (want, _), (got, buffers) = sliced(rows), sliced(most)
    for a, b, t in zip(got, want, buffers):
        assert torch.equal(a, b) and (t[:, rows:] == 7.0).all()

    def multi(m):
        out = torch.full((2, m, 256), 7.0, dtype=torch.float16, device="cuda")
        return Multi(lins[1:], out).run(x), out

    (want, _), (got, out) = multi(rows), multi(most)
    assert torch.equal(got, want) and (out.view(-1)[2 * rows * 256:] == 7.0).all()


def test_one_block_for_prompts_drafts_and_single_tokens(oracle):
    """One bundle and one block for every call, a captured single-token step among them"""
    import ampstein_b200 as amp
    from ampstein_b200.models import DecodeGraph, PagedAttention, PagedCache, Sliced
    hidden, hq, hkv, d = 512, 4, 2, 128
    lins = [linear(hidden, n * d, i) for i, n in enumerate((hq, hkv, hkv))]
    o = linear(hq * d, hidden, 9)
    inv_freq, _ = amp.rope_frequencies(d)
    x = torch.randn((1, 42, hidden), generator=torch.Generator().manual_seed(3)).to(torch.float16).cuda()
    caches = [PagedCache(1, 8, 16, hkv, d, 1, 8) for _ in range(2)]
    slots = [c.add() for c in caches]
    outs = [torch.zeros((1, 42, w.out_features), dtype=torch.float16, device="cuda") for w in lins]
    bundle = Sliced(lins, outs)
    blocks = [PagedAttention(bundle, o, c, 0, d, inv_freq) for c in caches]

    def run(i, at, n):
        pos = torch.tensor([caches[i].extend(slots[i], n)], device="cuda")
        return blocks[i].run(x[:, at:at + n].contiguous(), pos, caches[i].table[:1])

    whole = run(0, 0, 42).float()
    parts = [run(1, at, n) for at, n in ((0, 33), (33, 3), (36, 1), (37, 4))]
    x1, out = x[:, 41:].contiguous(), torch.zeros((1, hidden), dtype=torch.float16, device="cuda")
    pos = torch.tensor([caches[1].extend(slots[1], 1)], device="cuda")
    graph = DecodeGraph(lambda: blocks[1].run(x1, pos, caches[1].table[:1], out=out))
    graph.replay()
    torch.cuda.synchronize()
    parts = torch.cat(parts + [out]).float()
    # (two chains of linears within 1e-2 of the largest value each, the framework's bound for a linear)
    assert (whole - parts).abs().max() <= 2e-2 * whole.abs().max()
    with pytest.raises(ValueError):
        blocks[0].run(torch.zeros((1, 43, hidden), dtype=torch.float16, device="cuda"), pos, caches[0].table[:1])
