"""Calls whose outputs overlap what they read are refused, through both kinds of checks; layouts side by side are not."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
H = torch.float16


@pytest.fixture(params=[True, False], ids=["descriptions", "python"])
def amp(request, monkeypatch):
    import ampstein_b200
    from ampstein_b200 import attention
    if not request.param:
        monkeypatch.setattr(attention, "_direct", {})
    return ampstein_b200


@pytest.mark.parametrize("n", [2, 150])
def test_shared_memory_is_refused(amp, n):
    h, hkv, d = 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    flat = torch.randn((n + 1) * h * d, device="cuda", generator=g).to(H)
    q = flat[:n * h * d].view(n, h, d)
    caches = torch.randn((12, 2, 16, hkv, d), device="cuda", generator=g).to(H)
    k, v = caches[:, 0], caches[:, 1]
    table = torch.arange(12, dtype=torch.int32, device="cuda").view(1, 12)
    pos = torch.tensor([20], device="cuda")
    inv_freq, _ = amp.rope_frequencies(d)
    before = flat.clone(), caches.clone()
    for shift in (8, d, h * d):
        with pytest.raises(ValueError, match="overlaps"):
            amp.paged_attention(q, k, v, table, pos, out=flat[shift:shift + n * h * d].view(n, h, d))
        with pytest.raises(ValueError, match="overlaps"):
            amp.rope(q, pos, inv_freq, out=flat[shift:shift + n * h * d].view(n, h, d))
    inside = k.as_strided((n, h, d), (h * d, d, 1)) if n == 2 else None
    lse = flat[:2 * n * h].view(torch.float32).view(n, h)
    new = torch.randn((n, 2 * hkv, d), device="cuda", generator=g).to(H)
    bad = [lambda: amp.paged_attention(q, k, v, table, pos, lse=lse),
           lambda: amp.rope_append(q, new[:, :hkv], new[:, hkv:], pos, inv_freq, k, k, table),
           lambda: amp.rope_append(q[:, :hkv], new[:, :hkv], new[:, hkv:], pos, inv_freq, k, v, table, out=new[:, :hkv])]
    if n == 2:
        bad += [lambda: amp.paged_attention(q, k, v, table, pos, out=inside), lambda: amp.rope_append(q, new[:, :hkv], new[:, hkv:], pos, inv_freq, k, v, table, out=inside)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError, match="overlaps"):
            call()
            pytest.fail("call %d was taken" % i)
    with pytest.raises(RuntimeError, match="overlap"):
        amp.copy_pages([k, v, caches.view(24, 16, hkv, d)[1:13]], [0], [1])
    assert torch.equal(flat, before[0]) and torch.equal(caches, before[1])

    want = amp.paged_attention(q, k, v, table, pos)
    packed = torch.zeros((n, 3 * h, d), dtype=H, device="cuda")
    packed[:, h:2 * h] = q
    amp.paged_attention(packed[:, h:2 * h], k, v, table, pos, out=packed[:, 2 * h:])
    assert torch.equal(packed[:, 2 * h:], want) and torch.equal(packed[:, h:2 * h], q) and not packed[:, :h].any()
    want = amp.rope(q, pos, inv_freq)
    assert torch.equal(amp.rope(packed[:, h:2 * h], pos, inv_freq, out=packed[:, :h]), want)
    assert torch.equal(amp.rope(packed[:, h:2 * h], pos, inv_freq, out=packed[:, h:2 * h]), want)
