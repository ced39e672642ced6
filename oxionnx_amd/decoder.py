"""One decoder layer of a language model on the serving operators, as a serving program runs it.

`Pages` hands the pages of a `KvCache` to a batch of sequences; `DecoderLayer` runs prompts (`prefill`) and single
tokens (`decode`) through 4-bit projections, the rotating append and attention.  Norms, the gate and the residual
sums are elementwise torch operations on the same stream.

    python -m oxionnx_amd.decoder            # a random layer: a batch of prompts, then tokens from a captured graph
"""
import argparse
import time

import numpy as np

from . import _lib as L
from .device import HipContext


class Pages:
    """Which pages of a cache the sequences of a batch have: bookkeeping on the host, tables on the device."""

    def __init__(self, cache, batch, width):
        import torch
        self.cache, self.free = cache, list(range(cache.pages - 1, -1, -1))
        self.held = [[] for _ in range(batch)]
        at = torch.device("cuda", cache.device)
        self.host_table, self.host_lens = np.zeros((batch, width), np.int32), np.zeros(batch, np.int32)
        self.table = torch.zeros((batch, width), dtype=torch.int32, device=at)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=at)

    def extend(self, counts):
        """Room for counts[b] more tokens of each sequence: their slots and positions (int32, packed by sequence);
        the tables then describe the longer sequences."""
        import torch
        page = self.cache.page
        need = [-(-(int(n) + c) // page) - len(h) for n, c, h in zip(self.host_lens, counts, self.held)]
        if any(len(h) + n > self.host_table.shape[1] for h, n in zip(self.held, need)):
            raise MemoryError("a sequence needs more pages than its table has entries")
        if sum(need) > len(self.free):
            raise MemoryError(f"{sum(need)} pages are needed, {len(self.free)} are free")
        slots, positions = [], []
        for b, (n, c) in enumerate(zip(need, counts)):
            for _ in range(n):
                self.host_table[b, len(self.held[b])] = self.free[-1]
                self.held[b].append(self.free.pop())
            at = np.arange(self.host_lens[b], self.host_lens[b] + c)
            slots.append(np.asarray(self.held[b], np.int64)[at // page] * page + at % page if c else at)
            positions.append(at)
            self.host_lens[b] += c
        self.table.copy_(torch.from_numpy(self.host_table))
        self.lens.copy_(torch.from_numpy(self.host_lens))
        return tuple(torch.from_numpy(np.concatenate(x).astype(np.int32)).to(self.table.device) for x in (slots, positions))

    def release(self, b):
        """Sequence b ends: its pages are free again."""
        self.free.extend(reversed(self.held[b]))
        self.held[b], self.host_lens[b] = [], 0
        self.lens[b] = 0


def angles(positions, rot, base=10000.0, device=0):
    """cos and sin [positions, rot / 2] of the usual frequencies base^(-2 i / rot)."""
    import torch
    at = torch.device("cuda", device)
    a = torch.arange(positions, device=at, dtype=torch.float64)[:, None] * base ** (
        -torch.arange(0, rot, 2, device=at, dtype=torch.float64) / rot)
    return a.cos().float(), a.sin().float()


class DecoderLayer:
    """Weights of `HipContext.weight_q4`: qkv [hidden, (heads + 2 kv_heads) dim], out [heads dim, hidden], gate_up
    [hidden, 2 ffn], down [ffn, hidden]; norm1 / norm2 [hidden] scales of the root-mean-square norms."""

    def __init__(self, ctx, cache, heads, qkv, out, gate_up, down, norm1, norm2, cos, sin, eps=1e-5):
        self.ctx, self.cache, self.heads = ctx, cache, heads
        self.qkv, self.out, self.gate_up, self.down = qkv, out, gate_up, down
        self.norm1, self.norm2, self.cos, self.sin, self.eps = norm1, norm2, cos, sin, eps

    def _norm(self, x, scale):
        f = x.float()
        return (f * (f.square().mean(-1, keepdim=True) + self.eps).rsqrt() * scale.float()).to(x.dtype)

    def _append(self, x, slots, positions):
        kv, h = self.cache.kv_heads, self.heads
        qkv = self.ctx.gemm_q4(self._norm(x, self.norm1), self.qkv).view(x.shape[0], h + 2 * kv, self.cache.dim)
        # prompts attend to the keys and values as the cache holds them, which is what later tokens will see
        return self.ctx.kv_append(self.cache, qkv[:, h:h + kv], qkv[:, h + kv:], slots, q=qkv[:, :h], positions=positions,
                                  cos=self.cos, sin=self.sin)

    def _rest(self, x, y):
        import torch
        x = x + self.ctx.gemm_q4(y.view(x.shape[0], -1), self.out)
        gate, up = self.ctx.gemm_q4(self._norm(x, self.norm2), self.gate_up).chunk(2, -1)
        return x + self.ctx.gemm_q4((torch.nn.functional.silu(gate.float()) * up.float()).to(x.dtype), self.down)

    def prefill(self, x, cu, slots, positions):
        """Whole prompts, packed: x [tokens, hidden], offsets cu [sequences + 1].  They begin at position 0: attention
        over prompts does not read the cache, so a sequence that holds tokens already is refused (a capture cannot look
        at the positions: there the caller sees to it)."""
        import torch
        ends = None
        if x.shape[0] and not (positions.is_cuda and torch.cuda.is_current_stream_capturing()):
            ends = torch.stack((cu[:-1], cu[1:], positions[cu[:-1].clamp(max=x.shape[0] - 1)]))
            if ends.is_cuda:   # looked at when the layer is under way: the host does not wait for the stream here
                ends = torch.empty(ends.shape, dtype=ends.dtype, pin_memory=True).copy_(ends, non_blocking=True)
                there = torch.cuda.Event()
                there.record()
            else:
                self._begin_at_0(ends)
        q, k, v = self._append(x, slots, positions)
        y = self._rest(x, self.ctx.attn_prefill(q, k, v, cu))
        if ends is not None and positions.is_cuda:
            there.synchronize()
            self._begin_at_0(ends)
        return y

    @staticmethod
    def _begin_at_0(ends):
        if any(first and a < b for a, b, first in zip(*ends.tolist())):
            raise L.OhipError(L.E_INVALID, "prefill: a sequence holds tokens already")

    def decode(self, x, table, lens, slots, positions):
        """One token a sequence: x [sequences, hidden]; lens count it."""
        q, _, _ = self._append(x, slots, positions)
        return self._rest(x, self.ctx.attn_decode(q, self.cache, table, lens))


def random_layer(ctx, cache, heads, hidden, ffn, positions, dtype=L.F16, group=64, seed=0):
    """A layer of random weights, scaled so that activations keep their size."""
    import torch
    from .device import torch_dtype
    rng = np.random.default_rng(seed)

    def weight(k, n):
        blocks = -(-k // group)
        codes = rng.integers(0, 256, (n, blocks, group // 2), dtype=np.uint8)
        return ctx.weight_q4(codes, rng.uniform(0.5, 1.5, (n, blocks)).astype(np.float32) / (4.6 * k ** 0.5), k=k, dtype=dtype)

    width = (heads + 2 * cache.kv_heads) * cache.dim
    ones = torch.ones(hidden, dtype=torch_dtype(dtype), device=torch.device("cuda", ctx.device))
    cos, sin = angles(positions, cache.dim, device=ctx.device)
    return DecoderLayer(ctx, cache, heads, weight(hidden, width), weight(heads * cache.dim, hidden),
                        weight(hidden, 2 * ffn), weight(ffn, hidden), ones, ones, cos, sin)


def main():
    import torch
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--batch", type=int, default=8)
    p.add_argument("--prompt", type=int, default=500, help="tokens of the longest prompt")
    p.add_argument("--tokens", type=int, default=64)
    a = p.parse_args()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = HipContext(0)   # adopts the stream, so torch's work and the context's are captured together
        heads, kv, dim, page, hidden, ffn = 32, 8, 128, 64, 4096, 11008
        width = -(-(a.prompt + a.tokens + 2) // page)
        cache = ctx.kv_cache(a.batch * width, page, kv, dim)
        layer, pages = random_layer(ctx, cache, heads, hidden, ffn, a.prompt + a.tokens + 2), Pages(cache, a.batch, width)
        lengths = [max(1, a.prompt - i * a.prompt // (2 * a.batch)) for i in range(a.batch)]
        cu = torch.tensor(np.concatenate(([0], np.cumsum(lengths))), dtype=torch.int32, device="cuda")
        x = torch.randn((sum(lengths), hidden), device="cuda").half()
        slots, positions = pages.extend(lengths)
        y = layer.prefill(x, cu, slots, positions)
        ctx.sync()
        t = time.perf_counter()
        y = layer.prefill(x, cu, slots, positions)
        ctx.sync()
        t = time.perf_counter() - t
        print(f"prompts of {sum(lengths)} tokens: {t * 1e3:.2f} ms a layer")
        token, slots, positions = y[(cu[1:] - 1).long()].contiguous(), *pages.extend([1] * a.batch)
        step = [slots.clone(), positions.clone()]
        layer.decode(token, pages.table, pages.lens, *step)   # warm: scratch and torch's buffers
        ctx.sync()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = layer.decode(token, pages.table, pages.lens, *step)
        ctx.sync()
        t = time.perf_counter()
        for _ in range(a.tokens):
            graph.replay()
            token.copy_(out)
            slots, positions = pages.extend([1] * a.batch)
            step[0].copy_(slots)
            step[1].copy_(positions)
        ctx.sync()
        t = time.perf_counter() - t
        print(f"{a.tokens} steps of {a.batch} tokens: {t / a.tokens * 1e6:.0f} us a layer and step")
        del graph
        ctx.close()


if __name__ == "__main__":
    main()
