"""Positions, cuts and tokens that change on the device between the calls of one captured graph: rope_append, then attention of mixed calls,
several times over, with nothing in between that would wait for the launches in front."""
import pytest

torch = pytest.importorskip("torch")
import attention_cases as ac  # noqa: E402

pytestmark = pytest.mark.gpu
H = torch.float16


@pytest.mark.parametrize("counts", [[1, 1, 1, 1, 1], [1, 3, 0, 40, 1], [2, 150, 1, 0, 70], [300]])
@pytest.mark.parametrize("wide", [0, 150])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
def test_steps_of_one_graph(counts, wide, window, sinks):
    """Every step turns the tokens, moves the positions on and rotates the cuts by launches of its own; each replay is compared with the same
    steps made one by one, and the last step with the 64-bit form"""
    import ampstein_b200 as amp
    hq, hkv, d, page, steps, seqs = 8, 2, 128, 16, 3, len(counts)
    rows = sum(counts)
    g = torch.Generator().manual_seed(rows + wide)
    first = [int(x) for x in torch.randint(0, 200, (seqs,), generator=g)]
    width = -(-(max(first) + 8 * (max(counts) + 8)) // page) + wide
    used = -(-(max(first) + 8 * (max(counts) + 8)) // page)
    table = torch.full((seqs, width), -1, dtype=torch.int32)
    table[:, :used] = torch.randperm(seqs * used, generator=g).view(seqs, used).to(torch.int32)
    table = table.cuda()
    shape = (seqs * used, page, hkv, d)
    k0, v0 = (torch.randn(shape, generator=g).to(H).cuda() for _ in range(2))
    x0 = torch.randn((rows, hq + 2 * hkv, d), generator=g).to(H).cuda()
    c0 = torch.tensor(counts, dtype=torch.int32).cuda()
    p0 = torch.tensor(first, dtype=torch.int32).cuda()
    inv_freq, _ = amp.rope_frequencies(d)
    x, c, p, k, v = x0.clone(), c0.clone(), p0.clone(), k0.clone(), v0.clone()
    cu = torch.zeros(seqs + 1, dtype=torch.int32, device="cuda")
    outs = [torch.zeros((rows, hq, d), dtype=H, device="cuda") for _ in range(steps)]
    qs = [torch.zeros((rows, hq, d), dtype=H, device="cuda") for _ in range(steps)]
    lses = [torch.zeros((rows, hq), device="cuda") for _ in range(steps)]

    def step(i):
        p.add_(c)                                                       # the tokens of the step in front are behind us
        c.copy_(c.roll(1))
        torch.cumsum(c, 0, dtype=torch.int32, out=cu[1:])
        x.copy_(x.roll(1, 0))
        amp.rope_append(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], p, inv_freq, k, v, table, cu=cu, out=qs[i])
        amp.paged_attention(qs[i], k, v, table, p, cu=cu, window=window, sinks=sinks, out=outs[i], lse=lses[i])

    def reset():
        for a, b in ((x, x0), (c, c0), (p, p0), (k, k0), (v, v0)):
            a.copy_(b)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step(0)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            for i in range(steps):
                step(i)
    torch.cuda.synchronize()
    reset()
    want = []
    for i in range(steps):
        step(i)
        torch.cuda.synchronize()
        want.append((outs[i].clone(), lses[i].clone()))
    ends, cuts, ks, vs = p.tolist(), c.tolist(), k.clone(), v.clone()
    for _ in range(10):
        reset()
        for t in outs:
            t.fill_(9.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for i in range(steps):
            assert torch.equal(outs[i], want[i][0]) and torch.equal(lses[i], want[i][1]), i
    assert torch.equal(k, ks) and torch.equal(v, vs)
    ref, _, tol, _ = ac.attention(qs[-1], k, v, table, ends, cuts, window, sinks, d ** -0.5)
    assert ((outs[-1].double() - ref).abs() <= tol).all()
