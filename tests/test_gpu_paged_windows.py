"""A windowed conversation that gives up pages, beside one that keeps all of them: the same keys in other pages, so the same bits."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 3), (40, 3), (33, 0)])
@pytest.mark.parametrize("drafts", [1, 4])
def test_pages_are_given_up_while_tokens_are_pending(window, sinks, drafts):
    import ampstein_b200 as amp
    from ampstein_b200.models import PagedCache
    page, hq, hkv, d, prompt = 16, 4, 2, 64, 45
    g = torch.Generator().manual_seed(window + drafts)
    inv_freq, _ = amp.rope_frequencies(d)
    caches = [PagedCache(1, 40, page, hkv, d, 2, 12) for _ in range(2)]
    slots = [c.add() for c in caches]
    other = caches[0].add()                                             # takes what the first sequence gives up
    length = 0

    def run(n):
        nonlocal length
        x = [torch.randn((n, h, d), generator=g).to(torch.float16).cuda() for h in (hq, hkv, hkv)]
        outs = []
        for i, (c, slot) in enumerate(zip(caches, slots)):
            at = c.extend(slot, n)
            assert at == length
            if i == 0 and length:
                c.leave_behind(slot, window, sinks)
                if c.length(other) < 10 * page:
                    taken = c.extend(other, page) // page
                    c.k[0, int(c.table[other, taken])] = float("nan")
            pos, table = torch.tensor([at], device="cuda"), c.table[slot:slot + 1]
            q = amp.rope_append(*x, pos, inv_freq, c.k[0], c.v[0], table)
            outs.append(amp.paged_attention(q, c.k[0], c.v[0], table, pos, window=window, sinks=sinks))
        assert torch.isfinite(outs[0]).all() and torch.equal(*outs), length
        length += n

    run(prompt)
    for step in range(70 // drafts):
        run(drafts)
        if drafts > 1:                                                  # some are rejected
            length -= step % drafts
            for c, slot in zip(caches, slots):
                c.truncate(slot, length)
