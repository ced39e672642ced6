"""The serving operators on the GPU against 64-bit results (tests/_serving_ref.py): 4-bit products, appending to the
paged 4-bit cache, attention over prompts and over the cache, their refusals, and a captured step."""
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
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype)


def ints(seed, lo, hi, shape):
    return torch.randint(lo, hi, shape, generator=torch.Generator().manual_seed(seed))


# ------------------------------------------------------------------ 4-bit products
def q4_case(seed, m, k, n, group, zp, dtype):
    blocks = -(-k // group)
    codes = ints(seed, 0, 256, (n, blocks, group // 2)).to(torch.uint8)
    scales = ((0.5 + torch.rand((n, blocks), generator=torch.Generator().manual_seed(seed + 1))) / k ** 0.5).to(dtype)
    zeros = ints(seed + 2, 0, 256, (n, (blocks + 1) // 2)).to(torch.uint8) if zp else None
    return normal(seed + 3, (m, k), dtype), codes, scales, zeros, normal(seed + 4, (n,), dtype)


def q4_weight(ctx, codes, scales, zeros, k):
    return ctx.weight_q4(codes.numpy(), scales.float().numpy(), zero_points=None if zeros is None else zeros.numpy(),
                         k=k, dtype=CODES[scales.dtype])


@pytest.mark.parametrize("dtype", [torch.float32] + HALF, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,k,n,group,zp", [
    (1, 32, 16, 32, False), (1, 1, 1, 32, True), (1, 512, 1024, 32, True), (2, 777, 33, 64, True),
    (3, 4096, 50, 128, False), (7, 129, 17, 128, True), (16, 1000, 31, 256, True), (17, 640, 48, 64, False),
    (33, 257, 95, 32, True), (64, 1408, 40, 128, True), (5, 12345, 21, 64, True)])
def test_q4(ctx, dtype, m, k, n, group, zp):
    a, codes, scales, zeros, bias = q4_case(m + k + n, m, k, n, group, zp, dtype)
    got = ctx.gemm_q4(a.cuda(), q4_weight(ctx, codes, scales, zeros, k), bias.cuda())
    R.close(got, R.gemm_q4(a, codes, scales, zeros, bias))


@pytest.mark.parametrize("dtype", [torch.float32] + HALF, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,k,n,group", [(65, 333, 70, 64), (200, 1024, 256, 128), (130, 100, 19, 32)])
def test_q4_many_rows(ctx, dtype, m, k, n, group):
    a, codes, scales, zeros, bias = q4_case(m, m, k, n, group, True, dtype)
    got = ctx.gemm_q4(a.cuda(), q4_weight(ctx, codes, scales, zeros, k), bias.cuda())
    R.close(got, R.gemm_q4(a, codes, scales, zeros, bias, rounded_weights=True))


@pytest.mark.parametrize("dtype", [torch.float32] + HALF, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("m", [1, 5, 70])
def test_q4_strides_and_activation(ctx, dtype, m):
    k, n = 200, 37
    a, codes, scales, zeros, _ = q4_case(9, m, k, n, 64, True, dtype)
    wide = normal(1, (m, k + 13), dtype).cuda()
    wide[:, 5:5 + k] = a.cuda()                                    # rows at odd addresses
    out = torch.full((m, n + 3), 7.0, dtype=dtype, device="cuda")
    w = q4_weight(ctx, codes, scales, zeros, k)
    ctx.gemm_q4(wide[:, 5:5 + k], w, act=L.ACT_RELU, out=out[:, 1:1 + n])
    value, bound = R.gemm_q4(a, codes, scales, zeros, rounded_weights=m > 64)
    R.close(out[:, 1:1 + n], (value.clamp_min(0.0), bound))
    assert (out[:, 0] == 7).all() and (out[:, 1 + n:] == 7).all()


@pytest.mark.parametrize("dtype", [torch.float32] + HALF, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("zp", [False, True])
@pytest.mark.parametrize("m,k,n,group", [(58, 160, 320, 32), (16, 224, 160, 32), (30, 4104, 8200, 128), (3, 2600, 8192, 64),
                                         (64, 11008, 48, 256), (20, 136, 33, 64)])
def test_q4_aligned_rows(ctx, dtype, zp, m, k, n, group):
    """Rows of whole 16-byte chunks, a last tile of any length, two weights in turn."""
    cases = [q4_case(m + i, m, k, n, group, zp, dtype) for i in range(2)]
    ws = [q4_weight(ctx, codes, scales, zeros, k) for _, codes, scales, zeros, _ in cases]
    dev = [c[0].cuda() for c in cases]
    outs = [ctx.gemm_q4(dev[i % 2], ws[i % 2]) for i in range(4)]
    assert (outs[0] == outs[2]).all() and (outs[1] == outs[3]).all()
    for (a, codes, scales, zeros, _), got in zip(cases, outs):
        R.close(got, R.gemm_q4(a, codes, scales, zeros))


def test_q4_infinite_row_stays_in_its_row(ctx):
    a, codes, scales, zeros, bias = q4_case(4, 4, 256, 32, 32, True, torch.float16)
    a[2, 7] = float("nan")
    got = ctx.gemm_q4(a.cuda(), q4_weight(ctx, codes, scales, zeros, 256), bias.cuda()).cpu()
    assert got[2].isnan().all()
    keep = [0, 1, 3]
    value, bound = R.gemm_q4(a[keep], codes, scales, zeros, bias)
    R.close(got[keep], (value, bound))


def test_q4_named_weight_is_kept(ctx):
    a, codes, scales, zeros, bias = q4_case(5, 2, 64, 16, 32, True, torch.float16)
    before = ctx.counters()
    w1, w2 = (ctx.weight_q4(codes.numpy(), scales.numpy(), zeros.numpy(), name="w.q4") for _ in range(2))
    after = ctx.counters()
    assert after["weight_hits"] == before["weight_hits"] + 1 and w1.handle.value == w2.handle.value
    assert w1.nbytes == 16 * 128 // 2 + 16 * 2 * 2 + 16 * 2
    R.close(ctx.gemm_q4(a.cuda(), w2, bias.cuda()), R.gemm_q4(a, codes, scales, zeros, bias))


def test_q4_refusals(ctx):
    a, codes, scales, zeros, bias = q4_case(6, 2, 64, 16, 32, True, torch.float16)
    w = q4_weight(ctx, codes, scales, zeros, 64)
    ca = a.cuda()
    for args, kw in [((ca[:, :63], w), {}), ((ca.bfloat16(), w), {}), ((a, w), {}), ((ca, w, bias), {}),
                     ((ca, w, bias.cuda()[:8]), {}), ((ca, w), {"out": torch.empty((2, 15), dtype=torch.float16, device="cuda")}),
                     ((ca, w), {"act": 9}), ((torch.empty((64, 2), dtype=torch.float16, device="cuda").t(), w), {})]:
        with pytest.raises(L.OhipError):
            ctx.gemm_q4(*args, **kw)
    with pytest.raises(L.OhipError):
        ctx.weight_q4(codes.numpy(), scales.numpy()[:, :1])
    with pytest.raises(L.OhipError):
        ctx.weight_q4(codes.numpy(), scales.numpy(), k=20)
    with pytest.raises(L.OhipError):
        ctx.weight_q4(codes.numpy(), scales.numpy(), zero_points=zeros.numpy()[:1])
    with pytest.raises(L.OhipDeclined):
        ctx.weight_q4(np.zeros((4, 2, 10), np.uint8), np.ones((4, 2), np.float32))
    assert ctx.gemm_q4(ca[:0], w).shape == (0, 16)


# ------------------------------------------------------------------ append
def angles(rows, rot):
    a = torch.arange(rows)[:, None] * torch.exp(torch.arange(0, rot, 2) * (-9.2 / rot))
    return a.cos().float(), a.sin().float()


def check_held(cache, codes, params, slots, x, bound):
    """The codes and parameters at `slots` stand for x [tokens, kv, dim] (known to `bound`)."""
    page, at = slots // cache.page, slots % cache.page
    c, p = codes[page, :, at], params[page, :, at]
    x, bound = (t.unflatten(-1, (-1, cache.group)) for t in (x, bound))
    low, high, off = x.amin(-1), x.amax(-1), bound.amax(-1)
    half = 2.0 ** -11
    assert ((p[..., 1] - low).abs() <= off + half * (low.abs() + off) + 2.0 ** -25).all()
    step = (high - low) / 15
    soff = (2 * off + 4 * R.U32 * (high - low)) / 15
    assert ((p[..., 0] - step).abs() <= soff + half * (step + soff) + 2.0 ** -25).all()
    s, m = p[..., :1], p[..., 1:]
    c = c.unflatten(-1, (-1, cache.group))
    want = torch.where(s > 0, (x - m) / s.clamp_min(1e-30), 0.0).clamp(0, 15)
    slack = torch.where(s > 0, (bound + 2 * R.U32 * x.abs()) / s.clamp_min(1e-30), 0.0) + 1e-5
    assert ((c - want).abs() <= 0.5 + slack).all()


@pytest.mark.parametrize("dtype", HALF, ids=["f16", "bf16"])
@pytest.mark.parametrize("tokens,kv,g,dim,group,page,rot,interleaved", [
    (1, 1, 1, 64, 32, 16, 64, False), (1, 8, 4, 128, 64, 64, 128, False), (5, 2, 3, 128, 32, 48, 64, True),
    (37, 3, 1, 64, 64, 16, 32, False), (70, 1, 7, 128, 128, 32, 128, True), (19, 2, 0, 128, 64, 16, 16, False),
    (33, 2, 2, 64, 32, 128, 0, False)])
def test_append(ctx, dtype, tokens, kv, g, dim, group, page, rot, interleaved):
    heads, pages = kv * g, -(-tokens // page) + 2
    x = normal(tokens, (tokens, heads + 2 * kv, dim), dtype)
    cache = ctx.kv_cache(pages, page, kv, dim, group)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(1))[:tokens].int()
    positions = ints(2, 0, 500, (tokens,)).int()
    cos, sin = angles(500, rot) if rot else (None, None)
    dx = x.cuda()
    q, k, v = ctx.kv_append(cache, dx[:, heads:heads + kv], dx[:, heads + kv:], slots.cuda(), q=dx[:, :heads] if g else None,
                            positions=positions.cuda(), cos=None if cos is None else cos.cuda(),
                            sin=None if sin is None else sin.cuda(), interleaved=interleaved)
    turn = (lambda t: R.rotate(t, cos[positions.long()], sin[positions.long()], interleaved)) if rot else \
        (lambda t: (R.f64(t), torch.zeros_like(R.f64(t))))
    if g:
        R.close(q, R.rounded(*turn(x[:, :heads]), dtype))
    else:
        assert q is None
    kc, vc, kp, vp = R.read_cache(cache)
    check_held(cache, kc, kp, slots.long(), *turn(x[:, heads:heads + kv]))
    check_held(cache, vc, vp, slots.long(), R.f64(x[:, heads + kv:]), torch.zeros((tokens, kv, dim), dtype=torch.float64))
    at, off = slots.long() // page, slots.long() % page
    for got, c, p in ((k, kc, kp), (v, vc, vp)):
        held = R.values(c, p)[at, :, off].float()      # exact product, one rounding in f32, one to the type
        assert torch.equal(got.cpu(), held.to(dtype))
    touched = torch.zeros(pages * page, dtype=torch.bool)
    touched[slots.long()] = True
    for t in (kc, vc, kp.flatten(-2), vp.flatten(-2)):
        assert (t.transpose(1, 2).flatten(0, 1)[~touched] == 0).all()


def test_append_skips_and_clamps(ctx):
    """Slots outside the cache are not written, positions outside the table are its nearest rows."""
    kv, dim, page = 2, 128, 16
    cache = ctx.kv_cache(2, page, kv, dim)
    x = normal(3, (5, kv, dim), torch.float16).cuda()
    cos, sin = (t.cuda() for t in angles(10, dim))
    slots = torch.tensor([-1, 32, 31, 2 ** 31 - 1, 0], dtype=torch.int32).cuda()
    positions = torch.tensor([-5, 3, 10, 4, 2 ** 31 - 1], dtype=torch.int32)
    _, k, v = ctx.kv_append(cache, x, x, slots, positions=positions.cuda(), cos=cos, sin=sin, out_held=False)
    near = positions.long().clamp(0, 9)
    R.close(k, R.rounded(*R.rotate(x, cos.cpu()[near], sin.cpu()[near], False), torch.float16))
    assert torch.equal(v, x)
    kc, _, kp, vp = R.read_cache(cache)
    written = (vp[..., 0] != 0).any(-1).any(1).flatten().nonzero().flatten().tolist()
    assert written == [0, 31]


def test_append_extremes(ctx):
    """A constant group, a zero group, infinities, NaN, and values that f16 cannot hold."""
    cache = ctx.kv_cache(1, 16, 1, 128, 32)
    v = torch.zeros((4, 1, 128), dtype=torch.bfloat16)
    v[0] = 3.0
    v[1, 0, 0], v[1, 0, 33], v[1, 0, 64] = float("inf"), float("nan"), float("-inf")
    v[2, 0, 5], v[2, 0, 40] = 1e30, -1e30
    v[3] = torch.linspace(-1e-30, 1e-30, 128)
    _, _, got = ctx.kv_append(cache, v.cuda(), v.cuda(), torch.arange(4, dtype=torch.int32).cuda())
    got = got.float().cpu()[:, 0]
    assert (got[0] == 3).all()
    assert got[1, :32].isfinite().all() and got[1, 0] > 6e4 and (got[1, 1:32].abs() < 1e4).all()
    assert got[1, 32:64].isnan().all() and got[1, 64:].isfinite().all() and (got[1, 96:] == 0).all()
    assert got[2].isfinite().all() and got[2, 5] > 6e4 and got[2, 40] < -6e4
    assert (got[3] == 0).all()


def test_append_refusals(ctx):
    cache = ctx.kv_cache(2, 16, 2, 64, 32)
    k = normal(1, (3, 2, 64), torch.float16).cuda()
    slots = torch.arange(3, dtype=torch.int32).cuda()
    cos, sin = (t.cuda() for t in angles(8, 64))
    pos = slots
    for args, kw in [((k, k[:2], slots), {}), ((k, k, slots.long()), {}), ((k, k, slots[:2]), {}), ((k.float(), k, slots), {}),
                     ((k.cpu(), k, slots), {}), ((k[:, :1], k[:, :1], slots), {}), ((k, k, slots), {"q": k[:2]}),
                     ((k, k, slots), {"cos": cos, "sin": sin[:4], "positions": pos}),
                     ((k, k, slots), {"cos": cos.half(), "sin": sin, "positions": pos}),
                     ((k, k, slots), {"k_out": k[:2].clone()}),
                     ((k.transpose(1, 2).contiguous().transpose(1, 2), k, slots), {})]:
        with pytest.raises(L.OhipError):
            ctx.kv_append(cache, *args, **kw)
    for args, kw in [((k.float(), k.float(), slots), {}),
                     ((k, k, slots), {"cos": cos[:, :5].contiguous(), "sin": sin[:, :5].contiguous(), "positions": pos}),
                     ((torch.zeros(3 * 128 + 1, dtype=torch.float16, device="cuda")[1:].view(3, 2, 64), k, slots), {})]:
        with pytest.raises(L.OhipDeclined):
            ctx.kv_append(cache, *args, **kw)
    assert all((t == 0).all() for t in cache.tensors)
    ctx.kv_append(cache, k[:0], k[:0], slots[:0])


# ------------------------------------------------------------------ decode
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


@pytest.mark.parametrize("dtype", HALF, ids=["f16", "bf16"])
@pytest.mark.parametrize("lens,kv,g,dim,group,page,window", [
    ([1], 1, 1, 64, 32, 16, 0), ([0, 1, 2, 15, 16, 17], 2, 4, 128, 64, 16, 0), ([31, 32, 33, 0], 1, 8, 128, 128, 32, 0),
    ([129, 300, 5], 2, 7, 64, 64, 48, 0), ([1000, 77], 1, 16, 128, 32, 64, 0), ([260, 513], 2, 20, 128, 64, 128, 0),
    ([700, 40, 64], 1, 3, 64, 32, 16, 50), ([2049], 3, 1, 128, 128, 64, 1), ([4100, 3], 1, 4, 128, 64, 64, 1000)])
def test_decode(ctx, dtype, lens, kv, g, dim, group, page, window):
    pages = sum(-(-n // page) for n in lens) + 2
    cache = full_cache(ctx, len(lens) + dim, pages, page, kv, dim, group)
    table = tables(3, lens, page, pages)
    q = normal(7, (len(lens), kv * g, dim), dtype, 1.5)
    got = ctx.attn_decode(q.cuda(), cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), window=window)
    R.close(got, R.decode(q, cache, table, lens, dim ** -0.5, window))
    for i, n in enumerate(lens):
        if n == 0:
            assert (got[i] == 0).all()


@pytest.mark.parametrize("lens", [[20000], [9000, 1, 12345]], ids=["one", "three"])
def test_decode_long(ctx, lens):
    """Long contexts, split over blocks."""
    cache = full_cache(ctx, 1, sum(-(-n // 64) for n in lens), 64, 2, 64, 64)
    table = tables(4, lens, 64, cache.pages)
    q = normal(8, (len(lens), 8, 64), torch.float16, 2.0)
    dlens = torch.tensor(lens, dtype=torch.int32).cuda()
    got = ctx.attn_decode(q.cuda(), cache, table.cuda(), dlens)
    R.close(got, R.decode(q, cache, table, lens, 64 ** -0.5))
    for _ in range(3):   # the same sums in the same order
        assert torch.equal(ctx.attn_decode(q.cuda(), cache, table.cuda(), dlens), got)


@pytest.mark.parametrize("kv,g", [(1, 2), (2, 9)])
def test_decode_many_unequal(ctx, kv, g):
    """More sequences than a wave has lanes, of unequal lengths, some empty: pieces begin and end anywhere."""
    lens = [(37 * i * i) % 1500 if i % 7 else 0 for i in range(150)]
    lens[3], lens[140] = 2100, 1
    cache = full_cache(ctx, 6, sum(-(-n // 16) for n in lens) + 1, 16, kv, 64, 32)
    table = tables(11, lens, 16, cache.pages)
    q = normal(12, (len(lens), kv * g, 64), torch.bfloat16)
    got = ctx.attn_decode(q.cuda(), cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    R.close(got, R.decode(q, cache, table, lens, 0.125))


def test_decode_peaked_and_scaled(ctx):
    """One key far above the rest (late, early), and values whose scales span the f16 range."""
    lens = [600]
    cache = full_cache(ctx, 2, 10, 64, 1, 128, 64)
    kp, vp = cache.tensors[2], cache.tensors[3]
    vp[..., 0] *= torch.logspace(-5, 4, vp[..., 0].numel()).view(vp.shape[:-1]).cuda().half()
    table = tables(5, lens, 64, 10)
    q = normal(9, (1, 4, 128), torch.bfloat16, 8.0)
    got = ctx.attn_decode(q.cuda(), cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), scale=0.5)
    R.close(got, R.decode(q, cache, table, lens, 0.5))
    assert kp.isfinite().all()


def test_decode_garbage_outside(ctx):
    """NaN in tokens past the end, before the window, and in pages that no table names; entries that name no page."""
    page, lens, window = 16, [37, 70], 20
    cache = full_cache(ctx, 3, 9, page, 2, 64, 32)
    table = tables(6, lens, page, 9, width=6)
    q = normal(10, (2, 4, 64), torch.float16)
    lens_d = torch.tensor(lens, dtype=torch.int32).cuda()
    want = R.decode(q, cache, table, lens, 0.125, window)
    for t in cache.tensors[2:]:
        seen = torch.zeros((9, page), dtype=torch.bool)
        for i, n in enumerate(lens):
            for place in range(n - window, n):
                seen[table[i, place // page], place % page] = True
        t.transpose(1, 2)[~seen.cuda()] = float("nan")
    got = ctx.attn_decode(q.cuda(), cache, table.cuda(), lens_d, window=window)
    R.close(got, want)
    # a page id outside the cache: its tokens are not seen
    table[0, 1] = 1 << 30
    table[1, 3] = -1
    cache2 = full_cache(ctx, 3, 9, page, 2, 64, 32)
    got = ctx.attn_decode(q.cuda(), cache2, table.cuda(), lens_d)
    R.close(got, R.decode(q, cache2, table, lens, 0.125))
    # a length beyond the table
    got = ctx.attn_decode(q.cuda(), cache2, table[:, :2].contiguous().cuda(), torch.tensor([1000, -4], dtype=torch.int32).cuda())
    R.close(got, R.decode(q, cache2, table[:, :2], [32, 0], 0.125))


def test_decode_refusals(ctx):
    cache = full_cache(ctx, 4, 4, 16, 2, 64, 32)
    q = normal(1, (2, 4, 64), torch.float16).cuda()
    table, lens = torch.zeros((2, 2), dtype=torch.int32).cuda(), torch.ones(2, dtype=torch.int32).cuda()
    for args, kw in [((q[:, :3].contiguous(), cache, table, lens), {}), ((q.cpu(), cache, table, lens), {}),
                     ((q, cache, table.long(), lens), {}), ((q, cache, table[:1], lens), {}), ((q, cache, table, lens[:1]), {}),
                     ((q, cache, table, lens), {"scale": 0.0}), ((q, cache, table, lens), {"scale": float("nan")}),
                     ((q, cache, table, lens), {"window": -1}), ((q[..., :32], cache, table, lens), {}),
                     ((q, cache, table, lens), {"out": q[:1].clone()})]:
        with pytest.raises(L.OhipError):
            ctx.attn_decode(*args, **kw)
    with pytest.raises(L.OhipDeclined):
        ctx.attn_decode(q.float(), cache, table, lens)
    assert ctx.attn_decode(q[:0], cache, table[:0], lens[:0]).shape == (0, 4, 64)


# ------------------------------------------------------------------ prefill
def offsets(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32)


@pytest.mark.parametrize("dtype", HALF, ids=["f16", "bf16"])
@pytest.mark.parametrize("nq,nk,kv,g,dim,causal,window", [
    ([1], None, 1, 1, 64, True, 0), ([1, 0, 2, 31, 33], None, 2, 2, 128, True, 0), ([64, 65, 127, 129], None, 1, 4, 64, True, 0),
    ([200], None, 2, 1, 80, True, 0), ([300, 7], None, 1, 3, 128, True, 40), ([130], None, 1, 2, 8, False, 0),
    ([50, 3, 0, 20], [300, 3, 9, 64], 2, 2, 128, True, 0), ([100, 140], [40, 0], 1, 2, 64, True, 0),
    ([40], [700], 2, 2, 128, True, 100), ([257, 64], None, 1, 1, 96, False, 33), ([10, 150], [0, 20], 1, 1, 104, False, 0),
    ([513], None, 1, 2, 128, True, 1)])
def test_prefill(ctx, dtype, nq, nk, kv, g, dim, causal, window):
    cu_q, cu_k = offsets(nq), offsets(nq if nk is None else nk)
    q = normal(11, (int(cu_q[-1]), kv * g, dim), dtype, 1.5)
    k, v = (normal(12 + i, (int(cu_k[-1]), kv, dim), dtype) for i in range(2))
    got = ctx.attn_prefill(q.cuda(), k.cuda(), v.cuda(), cu_q.cuda(), None if nk is None else cu_k.cuda(), causal=causal,
                           window=window)
    R.close(got, R.prefill(q, k, v, cu_q, cu_k, dim ** -0.5, causal, window))


@pytest.mark.parametrize("dtype", HALF, ids=["f16", "bf16"])
def test_prefill_longer(ctx, dtype):
    """Several tiles of keys, running maxima that grow late, views of a joint projection."""
    lens, kv, g, dim = [700, 1, 430], 2, 2, 64
    x = normal(14, (1131, kv * g + 2 * kv, dim), dtype)
    x[650:700, kv * g:kv * g + kv] *= 6.0
    cu = offsets(lens)
    dx = x.cuda()
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    out = torch.full((1131, 5, dim), 7.0, dtype=dtype, device="cuda")
    ctx.attn_prefill(dx[:, :4], dx[:, 4:6], dx[:, 6:], cu.cuda(), scale=0.3, out=out[:, :4])
    R.close(out[:, :4], R.prefill(q, k, v, cu, cu, 0.3))
    assert (out[:, 4] == 7).all()


def test_prefill_sequences_do_not_meet(ctx):
    """NaN and infinities of one sequence reach no other, nor rows outside the offsets."""
    lens, dim = [40, 30, 50], 64
    q, k, v = (normal(15 + i, (130, 2, dim), torch.float16) for i in range(3))
    cu = offsets(lens)
    want = R.prefill(q[:120], k[:120], v[:120], cu, cu, 0.125)
    for t, bad in ((k, float("nan")), (v, float("inf"))):
        t[40:70] = bad
        t[120:] = bad
    out = torch.full((130, 2, dim), 5.0, dtype=torch.float16, device="cuda")
    ctx.attn_prefill(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), out=out)
    for part in (slice(0, 40), slice(70, 120)):
        R.close(out[part], (want[0][part], want[1][part]))
    assert out[40:70].isnan().all() and (out[120:] == 5).all()


@pytest.mark.parametrize("dtype", HALF, ids=["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("window", [0, 20])
def test_prefill_unseen_values(ctx, dtype, dim, window):
    """Infinities and NaN of keys that a query does not see leave its row as it is; those that it sees reach the
    channels they stand in."""
    lens, ks, kv = [150, 30, 70], [150, 45, 50], 2   # the last sequence's first queries see no key
    cu_q, cu_k = offsets(lens), offsets(ks)
    q = normal(41, (250, kv, dim), dtype)
    k, v = (normal(42 + i, (245, kv, dim), dtype) for i in range(2))
    bad = [(70, 0, 3, float("nan")), (75, 0, 3, float("inf")), (100, 1, 40, float("inf")), (101, 1, 40, float("-inf")),
           (160, 0, 11, float("-inf")), (200, 0, dim - 1, float("inf")), (200, 1, 0, float("nan"))]
    clean = v.clone()
    for row, head, ch, x in bad:
        v[row, head, ch], clean[row, head, ch] = x, 0.0
    k[145, 1, 5] = float("nan")
    got = ctx.attn_prefill(q.cuda(), k.cuda(), v.cuda(), cu_q.cuda(), cu_k.cuda(), window=window).cpu().double()
    k[145, 1, 5] = 0.0
    value, bound = R.prefill(q, k, clean, cu_q, cu_k, dim ** -0.5, True, window)
    for i in range(3):
        for a in range(lens[i]):
            last, row = a + ks[i] - lens[i], int(cu_q[i]) + a
            seen = range(max(0, last - window + 1 if window else 0) + int(cu_k[i]), last + 1 + int(cu_k[i]))
            for head in range(kv):
                if 145 in seen and head == 1 and i == 0:
                    assert got[row, head].isnan().all()
                    continue
                want = value[row, head].clone()
                for at, h, ch, x in bad:
                    if h == head and at in seen:
                        want[ch] += x if abs(want[ch]) != float("inf") or x != x or x == want[ch] else float("nan")
                plain = want.isfinite()
                assert ((got[row, head] - want).abs() <= bound[row, head])[plain].all()
                np.testing.assert_array_equal(got[row, head][~plain].numpy(), want[~plain].numpy())


def test_prefill_offsets_outside(ctx):
    """Offsets beyond the tokens (and falling ones) read and write nothing outside."""
    dim = 64
    q, k, v = (normal(18 + i, (50, 1, dim), torch.float16).cuda() for i in range(3))
    cu = torch.tensor([0, 20, 1000, 10], dtype=torch.int32)
    room = torch.full((60, 1, dim), 5.0, dtype=torch.float16, device="cuda")
    ctx.attn_prefill(q, k, v, cu.cuda(), out=room[5:55])
    assert (room[:5] == 5).all() and (room[55:] == 5).all()
    good = offsets([20, 30])
    R.close(room[5:55], R.prefill(q.cpu(), k.cpu(), v.cpu(), good, good, 0.125))


def test_prefill_refusals(ctx):
    q, k = normal(1, (6, 4, 64), torch.float16).cuda(), normal(2, (6, 2, 64), torch.float16).cuda()
    cu = offsets([6]).cuda()
    for args, kw in [((q, k, k[:5], cu), {}), ((q, k, k, cu.long()), {}), ((q[:, :3].contiguous(), k, k, cu), {}),
                     ((q, k.bfloat16(), k, cu), {}), ((q, k, k, cu, cu[:1]), {}), ((q, k, k, cu), {"scale": -1.0}),
                     ((q, k, k, cu), {"window": -2}), ((q.cpu(), k, k, cu), {}), ((q, k, k, cu), {"out": q[:3].clone()}),
                     ((q, k[..., :32], k[..., :32], cu), {})]:
        with pytest.raises(L.OhipError):
            ctx.attn_prefill(*args, **kw)
    wide = torch.zeros((6, 2, 136), dtype=torch.float16, device="cuda")
    odd = torch.zeros((6, 2, 60), dtype=torch.float16, device="cuda")
    for t in (wide, odd, q.float()):
        with pytest.raises(L.OhipDeclined):
            ctx.attn_prefill(t, t, t, cu)
    assert ctx.attn_prefill(q[:0], k[:0], k[:0], offsets([0]).cuda()).shape == (0, 4, 64)


# ------------------------------------------------------------------ captured
def test_captured_step(ctx):
    """A decode step (product, append, attention) recorded once serves new lengths, slots and activations."""
    import ctypes
    kv, g, dim, page, batch, hidden = 2, 2, 64, 16, 3, 96
    heads = kv * g
    side = torch.cuda.Stream()
    L.check(L.lib().ohip_ctx_set_stream(ctx.h, ctypes.c_void_p(side.cuda_stream)))
    try:
        _, codes, scales, zeros, _ = q4_case(20, 1, hidden, (heads + 2 * kv) * dim, 32, True, torch.float16)
        w = q4_weight(ctx, codes, scales, zeros, hidden)
        cache = full_cache(ctx, 5, 40, page, kv, dim, 32)
        start = [t.clone() for t in cache.tensors]
        cos, sin = (t.cuda() for t in angles(300, dim))
        x = torch.zeros((batch, hidden), dtype=torch.float16, device="cuda")
        table = tables(7, [170] * batch, page, 40).cuda()
        lens, slots, pos = (torch.zeros(batch, dtype=torch.int32, device="cuda") for _ in range(3))
        qkv = torch.empty((batch, heads + 2 * kv, dim), dtype=torch.float16, device="cuda")
        outs = [torch.empty(s, dtype=torch.float16, device="cuda") for s in
                ((batch, heads, dim), (batch, kv, dim), (batch, kv, dim), (batch, heads, dim))]

        def step(cache, outs):
            ctx.gemm_q4(x, w, out=qkv.view(batch, -1))
            ctx.kv_append(cache, qkv[:, heads:heads + kv], qkv[:, heads + kv:], slots, q=qkv[:, :heads], positions=pos,
                          cos=cos, sin=sin, q_out=outs[0], k_out=outs[1], v_out=outs[2])
            ctx.attn_decode(outs[0], cache, table, lens, out=outs[3])

        from oxionnx_amd.device import KvCache
        eager_cache = KvCache(*(t.clone() for t in cache.tensors))
        torch.cuda.synchronize()
        step(cache, outs)
        ctx.sync()
        graph = ctypes.c_void_p()
        L.check(L.lib().ohip_graph_begin(ctx.h))
        step(cache, outs)
        L.check(L.lib().ohip_graph_end(ctx.h, ctypes.byref(graph)))
        for t, s in zip(cache.tensors, start):
            t.copy_(s)
        for i in range(4):
            n = torch.tensor([170 - 40 * i, 1 + i, 3 * i], dtype=torch.int32)
            x.copy_(normal(30 + i, (batch, hidden), torch.float16))
            lens.copy_(n)
            at = (n.long() - 1).clamp_min(0)
            slots.copy_(torch.where(n > 0, table.cpu()[torch.arange(batch), at // page].long() * page + at % page, -1).int())
            pos.copy_(at.int())
            torch.cuda.synchronize()
            L.check(L.lib().ohip_graph_launch(graph))
            ctx.sync()
            got = [t.clone() for t in outs]
            torch.cuda.synchronize()
            eager = [torch.empty_like(t) for t in outs]
            step(eager_cache, eager)
            ctx.sync()
            for a, b in zip(got + list(cache.tensors), eager + list(eager_cache.tensors)):
                assert torch.equal(a, b)
        L.lib().ohip_graph_destroy(graph)
    finally:
        L.check(L.lib().ohip_ctx_set_stream(ctx.h, None))
