"""The attention operators as a model uses them: prompts, captured single-token steps, drafts, forks, windows, compaction over one paged
cache, against the plain 64-bit forms at every step; and the block with real EXL3 linears."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
import attention_cases as ac  # noqa: E402
from conftest import make_linear  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def amp():
    import ampstein_b200
    return ampstein_b200


class Columns:
    """q|k|v as columns of the hidden state: exact, whatever the number of rows"""

    class Width:
        def __init__(self, n):
            self.out_features = self.in_features = n

    def __init__(self, *widths):
        self.linears = [self.Width(n) for n in widths]

    def run(self, x):
        out, at = [], 0
        for w in self.linears:
            out.append(x[:, :, at:at + w.out_features].contiguous())
            at += w.out_features
        return out


class Same:
    def __init__(self, n):
        self.in_features = n

    def forward(self, x, out=None):
        return x if out is None else out.copy_(x)


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
@pytest.mark.parametrize("hq,hkv,d,rot,dtype", [(8, 2, 128, 128, torch.float16), (6, 1, 64, 32, torch.bfloat16), (4, 2, 256, 256, torch.bfloat16)])
def test_a_conversation(amp, window, sinks, hq, hkv, d, rot, dtype):
    from ampstein_b200.models import DecodeGraph, PagedAttention, PagedCache
    rng = torch.Generator().manual_seed(11)
    inv_freq, mscale = amp.rope_frequencies(rot, scaling=dict(kind="yarn", factor=4.0))
    cache = PagedCache(2, 70, 16, hkv, d, 5, 24, dtype=dtype)
    width = (hq + 2 * hkv) * d
    blocks = [PagedAttention(Columns(hq * d, hkv * d, hkv * d), Same(hq * d), cache, layer, d, inv_freq, mscale, window=window, sinks=sinks) for layer in range(2)]
    history = {}                                                        # slot -> hidden states of its tokens, per layer

    def tokens(n):
        return torch.randn((2, n, width), generator=rng).to(dtype).cuda()

    def verify(out, layer, x, slots, pos, counts):
        """The cache against the rotated history, the output against attention over the cache as it is"""
        k, v = cache.k[layer], cache.v[layer]
        q = torch.empty((x.shape[0], hq, d), dtype=dtype, device="cuda")
        for row, (b, p) in enumerate(ac.tokens(pos, counts)):
            mine = x[row, :hq * d].view(hq, d)
            want = ac.rotate(mine.double(), p, inv_freq, False, mscale)
            q[row] = want.to(dtype)
        got = amp.rope(x[:, :hq * d].view(-1, hq, d), torch.tensor(pos, device="cuda"), inv_freq, mscale=mscale,
                       cu=torch.tensor(np.concatenate(([0], np.cumsum(counts))), dtype=torch.int32, device="cuda"))
        assert ((got.double() - q.double()).abs() <= 2 * ac.U[dtype] * q.double().abs() + 2.0 ** -18).all()
        for b, (slot, p0, n) in enumerate(zip(slots, pos, counts)):
            for p in range(max(0, p0 - 2), p0 + n):
                page = int(cache.table[slot, p // 16])
                if page < 0:
                    continue
                row = history[slot][layer, p, hq * d:]
                want, tol = row[:hkv * d].view(hkv, d).double(), None
                tol = ac.rotate_bound(want, inv_freq, False, mscale, ac.U[dtype])
                want = ac.rotate(want, p, inv_freq, False, mscale)
                assert ((k[page, p % 16].double() - want).abs() <= tol).all()
                assert torch.equal(v[page, p % 16].reshape(-1), row[hkv * d:])
        want, _, tol, _ = ac.attention(got, k, v, cache.table[slots], pos, counts, window, sinks, d ** -0.5)
        assert ((out.view(-1, hq, d).double() - want).abs() <= tol).all()

    def feed(slots, counts):
        """A ragged chunk through both layers"""
        x = tokens(sum(counts))
        pos, at = [], 0
        for slot, n in zip(slots, counts):
            pos.append(cache.extend(slot, n))
            history[slot] = torch.cat((history[slot], x[:, at:at + n]), 1) if slot in history else x[:, at:at + n]
            at += n
        cu = torch.tensor(np.concatenate(([0], np.cumsum(counts))), dtype=torch.int32, device="cuda")
        table = cache.table[slots].contiguous()
        for layer, block in enumerate(blocks):
            out = block.run(x[layer:layer + 1], torch.tensor(pos, device="cuda"), table, cu=cu)
            verify(out, layer, x[layer], slots, pos, counts)

    a, b = cache.add(), cache.add()
    feed([a, b], [100, 37])                                             # two prompts in one call
    feed([b, a], [1, 3])                                                # a single token and a draft
    cache.truncate(a, 101)                                              # two drafted tokens rejected
    history[a] = history[a][:, :101]
    feed([a], [2])
    c = cache.fork(a)
    history[c] = history[a]
    feed([c, a], [1, 1])                                                # both write on: one of them in a copy of its own
    assert int(cache.table[a, 6]) != int(cache.table[c, 6])

    # single-token steps of a captured batch of four slots, one unused
    slots = [a, b, c]
    x = torch.zeros((2, 1, 4, width), dtype=dtype, device="cuda")
    pos = torch.full((4,), -1, dtype=torch.int64, device="cuda")
    table = torch.full((4, 24), -1, dtype=torch.int32, device="cuda")
    outs = [torch.zeros((4, hq * d), dtype=dtype, device="cuda") for _ in blocks]
    graph = DecodeGraph(lambda: [block.run(x[i], pos, table, out=outs[i]) for i, block in enumerate(blocks)])
    for _ in range(12):
        new = tokens(3)
        at = [cache.extend(s, 1) for s in slots]
        if window:
            for s in slots:
                cache.leave_behind(s, window, sinks)
        for i, s in enumerate(slots):
            history[s] = torch.cat((history[s], new[:, i:i + 1]), 1)
        x[:, 0, :3] = new
        pos[:3] = torch.tensor(at)
        table[:3] = cache.table[slots]
        graph.replay()
        for layer in range(2):
            verify(outs[layer][:3], layer, new[layer], slots, at, [1, 1, 1])
            assert not outs[layer][3].any()
    cache.free(b)                                                       # its pages are filled up by the others
    free = cache.free_pages
    assert cache.compact() == 70 - free
    feed([c, a], [30, 1])                                               # (tables have changed)
    assert int(cache.table.max()) < 70 - cache.free_pages + 1


def test_block_with_exl3_linears(amp, oracle):
    """Prompt and next token of a small layer: as the same tokens in one call, within the linears' tolerance"""
    from ampstein_b200.models import LinearEXL3, PagedAttention, PagedCache, Sliced
    hidden, hq, hkv, d = 512, 4, 2, 128

    def linear(k, n, seed):
        trellis, suh, svh, _ = make_linear(k, n, 4, seed=seed)
        svh = (svh.astype(np.float32) / (1.2437 * k ** 0.5)).astype(np.float16)
        return LinearEXL3(torch.from_numpy(trellis.view(np.int16)).cuda(), torch.from_numpy(suh).cuda(), torch.from_numpy(svh).cuda())

    lins = [linear(hidden, n * d, i) for i, n in enumerate((hq, hkv, hkv))]
    o = linear(hq * d, hidden, 9)
    inv_freq, _ = amp.rope_frequencies(d)
    x = torch.randn((1, 41, hidden), generator=torch.Generator().manual_seed(3)).to(torch.float16).cuda()

    def run(chunks):
        cache = PagedCache(1, 8, 16, hkv, d, 1, 8)
        slot, got, at = cache.add(), [], 0
        for n in chunks:
            outs = [torch.zeros((1, n, w.out_features), dtype=torch.float16, device="cuda") for w in lins]
            block = PagedAttention(Sliced(lins, outs), o, cache, 0, d, inv_freq)
            pos = torch.tensor([cache.extend(slot, n)], device="cuda")
            got.append(block.run(x[:, at:at + n].contiguous(), pos, cache.table[:1]))
            at += n
        return torch.cat(got).float()

    whole, parts = run([41]), run([33, 3, 1, 4])
    # (two chains of linears within 1e-2 of the largest value each, the framework's bound for a linear)
    assert (whole - parts).abs().max() <= 2e-2 * whole.abs().max()
    with pytest.raises(ValueError):
        PagedAttention(Sliced(lins, [torch.zeros((1, 1, w.out_features), dtype=torch.float16, device="cuda") for w in lins]), o, PagedCache(1, 2, 16, 4, d, 1, 2), 0, d, inv_freq)
