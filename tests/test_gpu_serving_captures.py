"""Captured serving calls that hold buffers of the context: attention over the cache in pieces (its partial sums lie in
the scratch) and products of many rows (the unpacked weight lies in a pool buffer), recorded by the context and by
torch, replayed between eager calls that need more scratch and other buffers."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from oxionnx_amd import _lib as L  # noqa: E402
from tests import _serving_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu


def normal(seed, shape, dtype=torch.float16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


class Recorded:
    """A step recorded by the context (ohip_graph_begin) or by torch."""

    def __init__(self, ctx, stream, by, step):
        self.by = by
        if by == "torch":
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph, stream=stream):
                step()
        else:
            self.graph = ctypes.c_void_p()
            L.check(L.lib().ohip_graph_begin(ctx.h))
            step()
            L.check(L.lib().ohip_graph_end(ctx.h, ctypes.byref(self.graph)))

    def replay(self):
        if self.by == "torch":
            self.graph.replay()
        else:
            L.check(L.lib().ohip_graph_launch(self.graph))

    def close(self):
        if self.by == "torch":
            self.graph.reset()
        else:
            L.lib().ohip_graph_destroy(self.graph)


@pytest.fixture
def run():
    """A context on a stream of its own, and that stream."""
    from oxionnx_amd.device import HipContext
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = HipContext(0)
        yield ctx, stream
        torch.cuda.synchronize()
        ctx.close()


def full_cache(ctx, seed, pages, page, kv, dim, group):
    cache = ctx.kv_cache(pages, page, kv, dim, group)
    g = torch.Generator().manual_seed(seed)
    for t in cache.tensors[:2]:
        t.copy_(torch.randint(0, 256, t.shape, generator=g, dtype=torch.int32).to(torch.uint8))
    for t in cache.tensors[2:]:
        scale = 0.05 + 0.3 * torch.rand(t.shape[:-1], generator=g)
        t.copy_(torch.stack((scale, -7.5 * scale + 0.2), -1).half())
    return cache


class Decode:
    """Attention of three sequences over a cache of 2048 tokens each, cut into pieces."""

    def __init__(self, ctx, seed, dim):
        page, entries, kv, g = 64, 32, 2, 4
        self.ctx, self.cache = ctx, full_cache(ctx, seed, 3 * entries, page, kv, dim, 32)
        ids = torch.randperm(3 * entries, generator=torch.Generator().manual_seed(seed)).int()
        self.table = ids.view(3, entries).cuda()
        self.lens = torch.ones(3, dtype=torch.int32).cuda()
        self.q = torch.zeros((3, kv * g, dim), dtype=torch.float16).cuda()
        self.out = torch.empty_like(self.q)

    def set(self, i):
        self.lens.copy_(torch.tensor([2048 - 300 * i, 1 + 500 * i, 0 if i % 2 else 1100], dtype=torch.int32))
        self.q.copy_(normal(90 + i, self.q.shape))

    def step(self, out=None):
        return self.ctx.attn_decode(self.q, self.cache, self.table, self.lens, out=self.out if out is None else out)


@pytest.mark.parametrize("by", ["context", "torch"])
def test_pieces_replayed_after_the_scratch_has_grown(run, by):
    ctx, stream = run
    d, larger = Decode(ctx, 1, 64), Decode(ctx, 2, 128)
    d.set(0)
    d.step()           # warm: the scratch is there
    ctx.sync()
    recorded = Recorded(ctx, stream, by, d.step)
    before = ctx.counters()["device_allocs"]
    filled = []
    for i in range(4):
        larger.set(i)
        larger.step()   # the first one grows the scratch
        ctx.sync()
        filled.append(torch.full((8 << 20,), 7.0, device="cuda"))   # what a freed scratch would lie in
        d.set(i)
        recorded.replay()
        ctx.sync()
        got = d.out.clone()
        eager = d.step(torch.empty_like(d.out))
        ctx.sync()
        assert torch.equal(got, eager)
        R.close(got, R.decode(d.q, d.cache, d.table, d.lens.cpu(), 0.125))
        assert all((t == 7).all() for t in filled)
    assert ctx.counters()["device_allocs"] == before + 1
    recorded.close()


@pytest.mark.parametrize("by", ["context", "torch"])
def test_pieces_recorded_without_scratch_run_whole(run, by):
    """A first call under capture cannot get scratch: it runs a block for each sequence and key head."""
    ctx, stream = run
    d = Decode(ctx, 3, 64)
    d.set(0)
    recorded = Recorded(ctx, stream, by, d.step)
    before = ctx.counters()["device_allocs"]
    for i in range(3):
        d.set(i)
        d.out.fill_(7.0)
        recorded.replay()
        ctx.sync()
        got = R.f64(d.out)
        eager = R.f64(d.step(torch.empty_like(d.out)))   # in pieces, once the scratch is there
        ctx.sync()
        # both are rounded once, from f32 sums of the same products in another order
        assert (got - eager).norm() <= 2.5 * R.UNIT[torch.float16] * eager.norm()
    assert ctx.counters()["device_allocs"] == before + 1
    recorded.close()


@pytest.mark.parametrize("dtype", [L.F16, L.BF16, L.F32], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("by", ["context", "torch"])
def test_products_of_many_rows_replayed_between_others(run, by, dtype):
    """Two products that unpack weights of different sizes, the second of the first one's result."""
    import numpy as np

    from oxionnx_amd.device import torch_dtype
    ctx, stream = run
    tdt, m, rng = torch_dtype(dtype), 70, np.random.default_rng(4)
    sizes = [(256, 640), (640, 192), (256, 640), (192, 4096)]
    ws = [ctx.weight_q4(rng.integers(0, 256, (n, k // 64, 32), dtype=np.uint8),
                        rng.uniform(0.5, 1.5, (n, k // 64)).astype(np.float32) / (4.6 * k ** 0.5), dtype=dtype) for k, n in sizes]
    x = torch.zeros((m, 256), dtype=tdt, device="cuda")
    outs = [torch.empty((m, n), dtype=tdt, device="cuda") for _, n in sizes[:2]]

    def step(outs=outs):
        ctx.gemm_q4(ctx.gemm_q4(x, ws[0], out=outs[0]), ws[1], out=outs[1])

    step()
    if by == "context":   # its captures take a buffer for each product: a dry run leaves them in the pool
        L.check(L.lib().ohip_pool_parking(ctx.h, 1))
        step()
        L.check(L.lib().ohip_pool_parking(ctx.h, 0))
    ctx.sync()
    recorded = Recorded(ctx, stream, by, step)
    held = []
    for i in range(4):
        x.copy_(normal(70 + i, x.shape, tdt))
        ctx.gemm_q4(x, ws[2])   # buffers of the same size, and a larger one
        ctx.gemm_q4(outs[1], ws[3])
        p = ctypes.c_void_p()   # a buffer of the pool that the recorded products must not touch
        L.check(L.lib().ohip_malloc(ctx.h, 256 * 640 * L.ELEM_BYTES[dtype], ctypes.byref(p)))
        mine = np.full(256 * 640 * L.ELEM_BYTES[dtype], 5 + i, np.uint8)
        L.check(L.lib().ohip_memcpy_h2d(ctx.h, p, mine.ctypes.data_as(ctypes.c_void_p), mine.nbytes))
        ctx.sync()
        held.append((p, mine))
        recorded.replay()
        ctx.sync()
        got = [t.clone() for t in outs]
        eager = [torch.empty_like(t) for t in outs]
        step(eager)
        ctx.sync()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
        for q, want in held:
            back = np.empty_like(want)
            L.check(L.lib().ohip_memcpy_d2h(ctx.h, back.ctypes.data_as(ctypes.c_void_p), q, back.nbytes))
            ctx.sync()
            assert (back == want).all()
    for q, _ in held:
        L.check(L.lib().ohip_free(ctx.h, q))
    recorded.close()
