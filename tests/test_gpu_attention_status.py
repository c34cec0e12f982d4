"""attention_status: it waits for what it asks about, and the prompt form loses no wait."""
import pytest

torch = pytest.importorskip("torch")
import attention_cases as ac  # noqa: E402

pytestmark = pytest.mark.gpu


def prompt(n, dtype=torch.float16):
    k, v, table = ac.paged([0], [n], 16, 2, 64, dtype, seed=n)
    return torch.randn((n, 8, 64), device="cuda").to(dtype), k, v, table, torch.tensor([0], device="cuda")


def test_it_waits_for_other_streams():
    import ampstein_b200 as amp
    args = prompt(90)
    amp.paged_attention(*args)
    torch.cuda.synchronize()
    side, done = torch.cuda.Stream(), torch.cuda.Event()
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)                                  # (about 0.2 s in front of the call)
        out = amp.paged_attention(*args)
        done.record(side)
    assert not done.query()
    assert amp.attention_status() == 0 and done.query()
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("n", [70, 300, 2600])
def test_no_wait_is_lost(n):
    import ampstein_b200 as amp
    args, side = prompt(n), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(stream):
            for _ in range(5):
                amp.paged_attention(*args)
    assert amp.attention_status() == 0 and amp.attention_status(torch.device("cuda:0")) == 0


def test_a_capture_refuses_it_and_goes_on():
    import ampstein_b200 as amp
    args = prompt(70)
    want, out = amp.paged_attention(*args), torch.zeros((70, 8, 64), dtype=torch.float16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="capture"):
            amp.attention_status()
        amp.paged_attention(*args, out=out)
    graph.replay()
    assert amp.attention_status() == 0 and torch.equal(out, want)
