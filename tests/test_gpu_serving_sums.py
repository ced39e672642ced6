"""Attention over the cache and 4-bit products against 64 bits on bounds that mistakes do not meet
(tests/test_serving_norms.py): the shapes that dispatch tells apart, whole and in pieces."""
import pytest

torch = pytest.importorskip("torch")

from oxionnx_amd import _lib as L  # noqa: E402
from tests import _serving_norms as N  # noqa: E402

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


# ------------------------------------------------------------------ attention over the cache
def full_cache(ctx, seed, pages, page, kv, dim, group):
    from oxionnx_amd.device import KvCache
    cache = ctx.kv_cache(pages, page, kv, dim, group)
    codes = [ints(seed + i, 0, 256, t.shape).to(torch.uint8).cuda() for i, t in enumerate(cache.tensors[:2])]
    params = []
    for i, t in enumerate(cache.tensors[2:]):
        scale = 0.05 + 0.3 * torch.rand(t.shape[:-1], generator=torch.Generator().manual_seed(seed + 5 + i))
        params.append(torch.stack((scale, -7.5 * scale + 0.2), -1).half().cuda())
    return KvCache(*codes, *params)


def tables(seed, lens, page, pages, width=None):
    need = [-(-n // page) for n in lens]
    width = max(need) if width is None else width
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int()
    table, at = torch.full((len(lens), width), -7, dtype=torch.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    return table


def attend(ctx, q, cache, table, lens, **kw):
    return ctx.attn_decode(q.cuda(), cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), **kw)


@pytest.mark.parametrize("dtype", HALF, ids=["f16", "bf16"])
@pytest.mark.parametrize("lens,kv,g,dim,group,page,window", [
    ([1], 1, 1, 64, 32, 16, 0), ([0, 1, 2, 15, 16, 17], 2, 4, 128, 64, 16, 0), ([31, 32, 33, 0], 1, 8, 128, 128, 32, 0),
    ([129, 300, 5], 2, 7, 64, 64, 48, 0), ([1000, 77], 1, 16, 128, 32, 64, 0), ([260, 513], 2, 20, 128, 64, 128, 0),
    ([700, 40, 64], 1, 3, 64, 32, 16, 50), ([64, 65], 3, 33, 64, 64, 64, 0), ([200, 31], 2, 9, 128, 128, 16, 33)])
def test_cache_whole(ctx, dtype, lens, kv, g, dim, group, page, window):
    """Sequences of up to 1024 tokens: a block each."""
    cache = full_cache(ctx, len(lens) + dim, sum(-(-n // page) for n in lens) + 2, page, kv, dim, group)
    table = tables(3, lens, page, cache.pages)
    q = normal(7, (len(lens), kv * g, dim), dtype, 1.5)
    got = attend(ctx, q, cache, table, lens, window=window)
    N.close_rows(got, N.decode(q, cache, table, lens, dim ** -0.5, window))


@pytest.mark.parametrize("dtype", HALF, ids=["f16", "bf16"])
@pytest.mark.parametrize("lens,kv,g,dim,group,page,window", [
    ([2049], 3, 1, 128, 128, 64, 1), ([4100, 3], 1, 4, 128, 64, 64, 1000), ([1025, 1, 0, 33], 2, 20, 128, 64, 128, 0),
    ([3000, 1500], 1, 16, 128, 32, 64, 0), ([2500, 40, 1111], 2, 8, 128, 128, 32, 0), ([1700, 900], 2, 33, 64, 32, 48, 0),
    ([5000, 6000, 10], 1, 7, 128, 32, 16, 4097), ([9000, 1, 12345], 2, 4, 64, 64, 64, 0), ([20000], 2, 4, 64, 32, 64, 0),
    ([40000, 100], 1, 2, 128, 64, 128, 0)])
def test_cache_in_pieces(ctx, dtype, lens, kv, g, dim, group, page, window):
    cache = full_cache(ctx, len(lens) + dim + g, sum(-(-n // page) for n in lens) + 2, page, kv, dim, group)
    table = tables(5, lens, page, cache.pages)
    q = normal(8, (len(lens), kv * g, dim), dtype, 1.5)
    got = attend(ctx, q, cache, table, lens, window=window)
    N.close_rows(got, N.decode(q, cache, table, lens, dim ** -0.5, window))
    for _ in range(2):   # the same sums in the same order
        assert torch.equal(attend(ctx, q, cache, table, lens, window=window), got)


@pytest.mark.parametrize("kv,g,dim", [(1, 2, 64), (2, 9, 64), (1, 4, 128)])
def test_cache_many_unequal(ctx, kv, g, dim):
    lens = [(37 * i * i) % 1500 if i % 7 else 0 for i in range(150)]
    lens[3], lens[140] = 2100, 1
    cache = full_cache(ctx, 6, sum(-(-n // 16) for n in lens) + 1, 16, kv, dim, 32)
    table = tables(11, lens, 16, cache.pages)
    q = normal(12, (len(lens), kv * g, dim), torch.bfloat16)
    N.close_rows(attend(ctx, q, cache, table, lens), N.decode(q, cache, table, lens, dim ** -0.5))


@pytest.mark.parametrize("dtype", HALF, ids=["f16", "bf16"])
@pytest.mark.parametrize("n", [600, 3000])
def test_cache_peaked_and_scaled(ctx, dtype, n):
    """One key far above the rest, and values whose scales go from 1e-5 to 1e4."""
    cache = full_cache(ctx, 2, 50, 64, 1, 128, 64)
    vp = cache.tensors[3]
    vp[..., 0] *= torch.logspace(-5, 4, vp[..., 0].numel()).view(vp.shape[:-1]).cuda().half()
    table = tables(5, [n], 64, 50)
    q = normal(9, (1, 4, 128), dtype, 8.0)
    N.close_rows(attend(ctx, q, cache, table, [n], scale=0.5), N.decode(q, cache, table, [n], 0.5))


@pytest.mark.parametrize("lens,width", [([37, 70], 6), ([1037, 2070], 140)])
def test_cache_garbage_outside(ctx, lens, width):
    """NaN in tokens past the end, before the window, and in pages that no table names; entries that name no page; lengths
    beyond the table."""
    page, window = 16, 20
    pages = sum(-(-n // page) for n in lens) + 1
    cache = full_cache(ctx, 3, pages, page, 2, 64, 32)
    table = tables(6, lens, page, pages, width=width)
    q = normal(10, (2, 4, 64), torch.float16)
    want = N.decode(q, cache, table, lens, 0.125, window)
    for t in cache.tensors[2:]:
        seen = torch.zeros((pages, page), dtype=torch.bool)
        for i, n in enumerate(lens):
            for place in range(n - window, n):
                seen[table[i, place // page], place % page] = True
        t.transpose(1, 2)[~seen.cuda()] = float("nan")
    N.close_rows(attend(ctx, q, cache, table, lens, window=window), want)
    table[0, 1], table[1, 3] = 1 << 30, -1
    again = full_cache(ctx, 3, pages, page, 2, 64, 32)
    N.close_rows(attend(ctx, q, again, table, lens), N.decode(q, again, table, lens, 0.125))
    short = table[:, :width // 2].contiguous()
    held = [width // 2 * page, 0]
    N.close_rows(attend(ctx, q, again, short, [10 ** 6, -4]), N.decode(q, again, short, held, 0.125))


def test_cache_large_scales_of_keys(ctx):
    """Keys of large scales whose minima take them back: scores are small differences of large sums."""
    lens, dim = [500, 1800], 128
    for dtype in HALF:
        cache = full_cache(ctx, 21, 80, 32, 2, dim, 64)
        kp = cache.tensors[2]
        kp[..., 0] *= 8.0
        kp[..., 1] = (-7.5 * kp[..., 0].float()).half()
        table = tables(22, lens, 32, 80)
        q = normal(23, (2, 8, dim), dtype)
        N.close_rows(attend(ctx, q, cache, table, lens, scale=0.02), N.decode(q, cache, table, lens, 0.02))


# ------------------------------------------------------------------ 4-bit products
@pytest.mark.parametrize("dtype", [torch.float32] + HALF, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("zp", [False, True])
@pytest.mark.parametrize("m,k,n,group", [
    (1, 32, 16, 32), (1, 1, 1, 32), (1, 512, 1024, 32), (2, 777, 33, 64), (3, 4096, 50, 128), (7, 129, 17, 128),
    (16, 1000, 31, 256), (33, 257, 95, 32), (5, 12345, 21, 64), (58, 160, 320, 32), (30, 4104, 8200, 128),
    (3, 2600, 8192, 64), (64, 11008, 48, 256), (17, 2200, 8208, 32), (1, 1100, 8192, 256)])
def test_products(ctx, dtype, zp, m, k, n, group):
    blocks = -(-k // group)
    codes = ints(k, 0, 256, (n, blocks, group // 2)).to(torch.uint8)
    zeros = ints(k + 1, 0, 256, (n, (blocks + 1) // 2)).to(torch.uint8) if zp else None
    scales = ((0.5 + torch.rand((n, blocks), generator=torch.Generator().manual_seed(k + 2))) / k ** 0.5).to(dtype)
    a, bias = normal(k + 3, (m, k), dtype), normal(k + 4, (n,), dtype)
    w = ctx.weight_q4(codes.numpy(), scales.float().numpy(), zero_points=None if zeros is None else zeros.numpy(), k=k,
                      dtype=CODES[dtype])
    value, bound = N.gemm_q4(a, codes, scales, zeros, bias)
    got = ctx.gemm_q4(a.cuda(), w, bias.cuda()).cpu().double()
    off = ((got - value).abs() / bound).max()
    assert off <= 1.0, float(off)


def test_prompts_repeat_themselves(ctx):
    """Prompt attention has one order of its sums."""
    for dtype in HALF:
        q, k, v = (normal(60 + i, (700, h, 128), dtype).cuda() for i, h in enumerate((8, 2, 2)))
        cu = torch.tensor([0, 130, 131, 700], dtype=torch.int32).cuda()
        first = ctx.attn_prefill(q, k, v, cu)
        for _ in range(3):
            assert torch.equal(ctx.attn_prefill(q, k, v, cu), first)
