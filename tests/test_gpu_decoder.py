"""A decoder layer on the serving operators: prompts and single tokens against the layer in 64 bits, page
bookkeeping, and a captured step."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oxionnx_amd import _lib as L  # noqa: E402
from tests import _serving_ref as R  # noqa: E402


class _Cache:
    pages, page, device = 5, 16, 0


def test_pages_on_the_host(monkeypatch):
    """Slots, positions and tables of growing sequences; refusals leave everything as it was."""
    from oxionnx_amd import decoder
    real = torch.device
    monkeypatch.setattr(torch, "device", lambda *a: real("cpu"))
    p = decoder.Pages(_Cache, 2, 3)
    slots, positions = p.extend([17, 3])
    assert positions.tolist() == list(range(17)) + [0, 1, 2]
    assert slots.tolist() == list(range(16)) + [16, 32, 33, 34]
    assert p.lens.tolist() == [17, 3] and p.table.tolist() == [[0, 1, 0], [2, 0, 0]]
    with pytest.raises(MemoryError):
        p.extend([40, 0])          # more than the table's three entries
    with pytest.raises(MemoryError):
        p.extend([31, 45])         # three pages more, two are free
    assert p.lens.tolist() == [17, 3] and len(p.free) == 2
    slots, positions = p.extend([0, 14])
    assert positions.tolist() == list(range(3, 17)) and slots.tolist() == list(range(35, 48)) + [48]
    p.release(0)
    assert p.lens.tolist() == [0, 17] and len(p.free) == 3
    assert p.extend([1, 0])[0].tolist() == [0]


def _layer64(layer, dense, x, sees_lens, held):
    """The layer in 64 bits on rows x, their attention over `held` (keys, values [kv, tokens, dim])."""
    heads, kv, dim = layer.heads, layer.cache.kv_heads, layer.cache.dim

    def norm(t, scale):
        return t * (t.square().mean(-1, keepdim=True) + layer.eps).rsqrt() * R.f64(scale)

    qkv = (norm(x, layer.norm1) @ dense[0]).view(-1, heads + 2 * kv, dim)
    pos = torch.tensor(sees_lens) - 1
    q = R.rotate(qkv[:, :heads], layer.cos.cpu()[pos], layer.sin.cpu()[pos], False)[0]
    y = torch.zeros_like(q)
    for i, n in enumerate(sees_lens):
        for h in range(heads):
            s = torch.softmax(held[0][h // (heads // kv), :n] @ q[i, h] * dim ** -0.5, 0)
            y[i, h] = s @ held[1][h // (heads // kv), :n]
    x = x + y.flatten(1) @ dense[1]
    gate, up = (norm(x, layer.norm2) @ dense[2]).chunk(2, -1)
    return x + (torch.nn.functional.silu(gate) * up) @ dense[3]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [L.F16, L.BF16], ids=["f16", "bf16"])
def test_layer_prompts_then_tokens(dtype):
    from oxionnx_amd import decoder
    from oxionnx_amd.device import HipContext, torch_dtype
    ctx = HipContext(0)
    try:
        heads, kv, dim, hidden, ffn, page, lengths, more = 4, 2, 64, 160, 224, 16, [37, 1, 20], 3
        cache = ctx.kv_cache(20, page, kv, dim, 32)
        recorded = []
        weight_q4 = ctx.weight_q4
        ctx.weight_q4 = lambda codes, scales, **kw: recorded.append((codes, scales, kw["k"])) or weight_q4(codes, scales, **kw)
        layer = decoder.random_layer(ctx, cache, heads, hidden, ffn, 64, dtype=dtype, group=32, seed=3)
        tdt = torch_dtype(dtype)
        dense = [R.q4_weight(torch.from_numpy(c), torch.from_numpy(s).to(tdt), None, k)[0] for c, s, k in recorded]
        pages = decoder.Pages(cache, len(lengths), 5)
        x = torch.randn((sum(lengths), hidden), generator=torch.Generator().manual_seed(1)).to(tdt)
        cu = torch.tensor(np.concatenate(([0], np.cumsum(lengths))), dtype=torch.int32).cuda()
        y = layer.prefill(x.cuda(), cu, *pages.extend(lengths))
        tokens = [torch.randn((3, hidden), generator=torch.Generator().manual_seed(5 + i)).to(tdt) for i in range(more)]
        steps = []
        for t in tokens:
            slots, positions = pages.extend([1] * 3)
            steps.append(layer.decode(t.cuda(), pages.table, pages.lens, slots, positions))
        codes = R.read_cache(cache)
        values = R.values(codes[0], codes[2]), R.values(codes[1], codes[3])
        # About a dozen tensors are rounded to the type on the way: their errors add up to less than 16 roundings
        most = 16 * R.UNIT[tdt]
        for b, n in enumerate(lengths):
            ids = pages.table[b].cpu().long()
            held = [v[ids].transpose(0, 1).flatten(1, 2) for v in values]
            a = int(cu[b])
            want = _layer64(layer, dense, R.f64(x[a:a + n]), list(range(1, n + 1)), held)
            got = R.f64(y[a:a + n])
            assert (got - want).norm() <= most * want.norm()
            for i in range(more):
                want = _layer64(layer, dense, R.f64(tokens[i][b:b + 1]), [n + i + 1], held)
                assert (R.f64(steps[i][b:b + 1]) - want).norm() <= most * want.norm()
    finally:
        ctx.close()


@pytest.mark.gpu
def test_example_runs(capsys, monkeypatch):
    """The example: prompts, then tokens replayed from a captured graph."""
    import sys

    from oxionnx_amd import decoder
    monkeypatch.setattr(sys, "argv", ["decoder", "--batch", "3", "--prompt", "70", "--tokens", "4"])
    decoder.main()
    assert "us a layer and step" in capsys.readouterr().out
