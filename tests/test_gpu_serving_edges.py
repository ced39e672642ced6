"""The serving operators where their ranges end: infinities, numbers near the largest, groups of infinities, windows
without a limit, captured calls that share the context's buffers."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oxionnx_amd import _lib as L  # noqa: E402
from tests import _serving_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu
CODES = {torch.float32: L.F32, torch.float16: L.F16, torch.bfloat16: L.BF16}
HALF = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ctx():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    from oxionnx_amd.device import HipContext
    c = HipContext(0)
    yield c
    c.close()


def normal(seed, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def ints(seed, lo, hi, shape):
    return torch.randint(lo, hi, shape, generator=torch.Generator().manual_seed(seed))


# ------------------------------------------------------------------ 4-bit products
@pytest.mark.parametrize("dtype", [torch.float32] + HALF, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("m", [1, 2, 5, 16, 20, 40, 64, 70])
@pytest.mark.parametrize("k,group,zp", [(512, 32, True), (300, 64, False), (1160, 128, True)])
def test_q4_infinite_and_huge_activations(ctx, dtype, m, k, group, zp):
    """An infinity gives the infinity of its weight's sign (NaN where that is 0 or infinities meet); products that f32
    holds are numbers, however near its largest they are."""
    n, blocks = 40, -(-k // group)
    codes = ints(k + m, 0, 256, (n, blocks, group // 2)).to(torch.uint8)
    scales = ((0.5 + torch.rand((n, blocks), generator=torch.Generator().manual_seed(m))) / 32).to(dtype)
    zeros = ints(m, 0, 256, (n, (blocks + 1) // 2)).to(torch.uint8) if zp else None
    a = normal(m + 1, (m, k), dtype)
    huge = 6e4 if dtype == torch.float16 else 1e37
    for row in range(m):
        kind, at = row % 5 if m > 1 else k % 5, (37 * row + 11) % k
        if kind < 3:
            a[row, at] = (huge, float("inf"), -float("inf"))[kind]
        if kind == 1 and row % 2:
            a[row, (at + 5) % k] = -float("inf")
        if kind == 3:
            a[row, at] = -huge
    w = ctx.weight_q4(codes.numpy(), scales.float().numpy(), zero_points=None if zeros is None else zeros.numpy(), k=k,
                      dtype=CODES[dtype])
    got = R.f64(ctx.gemm_q4(a.cuda(), w))
    weight, _ = R.q4_weight(codes, scales, zeros, k)
    if m > 64:
        weight = R.f64(weight.to(dtype))   # rounded to the type first
    want = R.f64(a) @ weight
    limit = torch.finfo(dtype).max
    want = torch.where(want.abs() > limit * (1 + R.UNIT[dtype]), want.sign() * torch.inf, want)
    finite = want.isfinite()
    np.testing.assert_array_equal(got[~finite].numpy(), want[~finite].numpy())
    # of bf16 rows that are small, the sums pass through (2 * 143 + 15) times the activations
    size = torch.where(R.f64(a).isfinite(), R.f64(a), 0.0).abs() @ (weight.abs() + 301 * R.f64(scales).max())
    bound = (2 * k + 64) * R.U32 * size
    bound = bound + R.UNIT[dtype] * (want.abs() + bound) + R.TINY[dtype]
    near = finite & (want.abs() + bound < limit)   # (the others may round to infinity)
    assert ((got - want).abs() <= bound)[near].all()
    assert near.any() or m == 1


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", HALF, ids=["f16", "bf16"])
@pytest.mark.parametrize("dim,group", [(64, 32), (128, 64), (128, 128)])
def test_append_groups_of_infinities(ctx, dtype, dim, group):
    """A group of one infinity alone is held as f16's largest number of its sign, one of both from end to end; only a NaN
    makes a group NaN."""
    inf = float("inf")
    cache = ctx.kv_cache(1, 16, 1, dim, group)
    v = torch.zeros((5, 1, dim), dtype=dtype)
    v[0], v[1] = inf, -inf
    v[2], v[2, 0, 1::2] = inf, -inf
    v[3], v[3, 0, 1::2] = inf, float("nan")
    v[4, 0, :group], v[4, 0, group:] = -inf, 1.0
    k, got = ctx.kv_append(cache, v.cuda(), v.cuda(), torch.arange(5, dtype=torch.int32).cuda())[1:]
    kc, vc, kp, vp = R.read_cache(cache)
    for codes, p, out in ((kc, kp, k), (vc, vp, got)):
        low, high = 65504.0, 15 * 65504.0 - 65504.0   # f16's largest; lowest and largest step from minus it
        held = R.values(codes, p)[0, 0]
        assert (held[0] == low).all() and (held[1] == -low).all()
        assert (held[2, ::2] == high).all() and (held[2, 1::2] == -low).all()
        assert held[3].isnan().all()
        assert (held[4, :group] == -low).all() and (held[4, group:] == 1).all()
        for i in range(5):
            np.testing.assert_array_equal(R.f64(out)[i, 0].numpy(), R.f64(held[i].float().to(dtype)).numpy())


# ------------------------------------------------------------------ prompt attention
def offsets(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32)


@pytest.mark.parametrize("dtype", HALF, ids=["f16", "bf16"])
@pytest.mark.parametrize("nq,nk,causal", [([10], [100], False), ([140, 33], [130, 33], True), ([300], [300], True),
                                          ([70], [5], False), ([200, 1], [90, 400], True)])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 200, 700])
def test_prefill_windows_of_everything(ctx, dtype, nq, nk, causal, window):
    """Windows larger than any sequence, up to the type's largest, are none."""
    kv, g, dim = 1, 2, 64
    cu_q, cu_k = offsets(nq), offsets(nk)
    q = normal(51, (int(cu_q[-1]), kv * g, dim), dtype)
    k, v = (normal(52 + i, (int(cu_k[-1]), kv, dim), dtype) for i in range(2))
    got = ctx.attn_prefill(q.cuda(), k.cuda(), v.cuda(), cu_q.cuda(), cu_k.cuda(), causal=causal, window=window)
    R.close(got, R.prefill(q, k, v, cu_q, cu_k, dim ** -0.5, causal, window))
    none = ctx.attn_prefill(q.cuda(), k.cuda(), v.cuda(), cu_q.cuda(), cu_k.cuda(), causal=causal)
    assert torch.equal(got, none)


# ------------------------------------------------------------------ the layer
def test_second_prompt_of_a_sequence_is_refused():
    """Its first tokens are in the cache, which prompt attention does not read; other sequences' prompts go on."""
    from oxionnx_amd import decoder
    from oxionnx_amd.device import HipContext
    ctx = HipContext(0)
    try:
        cache = ctx.kv_cache(20, 16, 2, 64, 32)
        layer = decoder.random_layer(ctx, cache, 4, 160, 224, 64, group=32)
        pages = decoder.Pages(cache, 3, 5)
        x = normal(70, (30, 160), torch.float16).cuda()
        for counts, held in (([7, 0, 12], False), ([0, 9, 0], False), ([4, 0, 0], True), ([0, 1, 3], True)):
            cu = offsets(counts).cuda()
            args = (x[:sum(counts)].contiguous(), cu, *pages.extend(counts))
            if held:
                with pytest.raises(L.OhipError):
                    layer.prefill(*args)
            else:
                assert layer.prefill(*args).isfinite().all()
    finally:
        ctx.close()
