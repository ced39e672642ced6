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
