"""The bounds of tests/_serving_norms.py on the host: results with a mistake planted do not meet them."""
import pytest

torch = pytest.importorskip("torch")

from oxionnx_amd import device as D  # noqa: E402
from tests import _serving_norms as N  # noqa: E402
from tests import _serving_ref as R  # noqa: E402


def normal(seed, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def host_cache(seed, pages, page, kv, dim, group):
    g = torch.Generator().manual_seed(seed)
    shapes = (pages, kv, page, 4, dim // 32, 4), (pages, kv, page // 16, 16, 16, dim // 32)
    codes = [torch.randint(0, 256, s, generator=g, dtype=torch.int32).to(torch.uint8) for s in shapes]
    params = []
    for _ in range(2):
        scale = 0.05 + 0.3 * torch.rand((pages, kv, page, dim // group), generator=g)
        params.append(torch.stack((scale, -7.5 * scale + 0.2), -1).half())
    return D.KvCache(*codes, *params)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("lens,kv,g,dim,group,page,window", [
    ([40, 2, 700], 2, 4, 128, 64, 16, 0), ([300, 129], 2, 7, 64, 32, 48, 50), ([1000, 77], 2, 16, 128, 32, 64, 0),
    ([2100, 5], 2, 1, 128, 32, 64, 1000), ([5000], 2, 8, 64, 32, 64, 0)])
def test_mistakes_over_the_cache_show(dtype, lens, kv, g, dim, group, page, window):
    need = [-(-n // page) for n in lens]
    cache = host_cache(len(lens) + dim, sum(need), page, kv, dim, group)
    ids = torch.randperm(sum(need), generator=torch.Generator().manual_seed(1)).int()
    table, at = torch.zeros((len(lens), max(need)), dtype=torch.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    q = normal(7, (len(lens), kv * g, dim), dtype, 1.5)
    scale = dim ** -0.5
    value, limit = N.decode(q, cache, table, lens, scale, window)

    def shows(wrong, rows=slice(None)):
        ratio = N.rows_off(wrong[rows], (value[rows], limit[rows]))
        return bool((ratio > 1).any(1).all())   # in every sequence

    def swapped(i):
        t = list(cache.tensors)
        t[i] = t[i].flip(3)
        return D.KvCache(*t)

    N.close_rows(value.to(dtype), (value, limit))
    # rounded to the type once more than it has to be, and some more of it
    assert not shows(value.to(dtype) * (1 + R.UNIT[dtype] / 4))
    assert N.rows_off(torch.zeros_like(value), (value, limit)).min() > 5       # zeros, in every row
    assert shows(N.decode(q, cache, table, [n - 1 for n in lens], scale, window)[0])             # a token too few
    if window:
        longer = [i for i, n in enumerate(lens) if n > window]
        assert shows(N.decode(q, cache, table, lens, scale, 0)[0], longer)                       # no window
        # (one token of a thousand is as much as a rounding to bf16)
        assert window > 100 or shows(N.decode(q, cache, table, lens, scale, window + 1)[0], longer)
    assert shows(N.decode(q.roll(1, 1), cache, table, lens, scale, window)[0])                   # another head's query
    assert shows(value.unflatten(1, (kv, g)).roll(1, 1).flatten(1, 2))                            # another key head
    assert shows(N.decode(q, swapped(2), table, lens, scale, window)[0])                         # parameters of another group
    assert shows(N.decode(q, swapped(3), table, lens, scale, window)[0])
    long = [i for i, n in enumerate(lens) if n > 16]
    assert shows(N.decode(q, cache, table, lens, scale * 1.05, window)[0], long)                 # a wrong scale


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,k,n,group", [(5, 12345, 21, 64), (16, 11008, 20, 256), (3, 4096, 50, 128), (16, 1000, 31, 32)])
def test_mistakes_of_products_show(dtype, m, k, n, group):
    blocks = -(-k // group)
    g = torch.Generator().manual_seed(k)
    codes = torch.randint(0, 256, (n, blocks, group // 2), generator=g, dtype=torch.int32).to(torch.uint8)
    zeros = torch.randint(0, 256, (n, (blocks + 1) // 2), generator=g, dtype=torch.int32).to(torch.uint8)
    scales = ((0.5 + torch.rand((n, blocks), generator=g)) / k ** 0.5).to(dtype)
    a = normal(k + 1, (m, k), dtype)
    value, bound = N.gemm_q4(a, codes, scales, zeros)
    want = R.q4_weight(codes, scales, zeros, k)[0]
    torch.testing.assert_close(value, R.f64(a) @ want, rtol=1e-12, atol=1e-12)

    def missed(wrong, share=0.5):
        return float(((wrong - value).abs() > bound).double().mean()) >= share

    assert not missed(R.f64(value.to(dtype)), 1e-9)
    assert missed(torch.zeros_like(value), 0.85)
    near = scales.roll(1, 1)
    assert missed(N.gemm_q4(a, codes, near, zeros)[0])                                  # another group's scale
    assert missed(N.gemm_q4(a, codes, scales, zeros ^ 0x11)[0])                         # zero points one off
    assert missed(N.gemm_q4(a.roll(1, 1), codes, scales, zeros)[0])
    assert missed(N.gemm_q4(a, codes ^ 1, scales, zeros)[0])                            # a bit of every other code
    if dtype == torch.float32:
        assert missed(R.f64(value.bfloat16()))                                          # a product done in bf16
        assert missed(N.gemm_q4(a.bfloat16().float(), codes, scales, zeros)[0])
