"""The serving operators in 64 bits, and bounds of what f32 sums and 16-bit roundings may add.

Each function returns (value, bound) arrays: a kernel that forms its products and sums in f32 and rounds once (or
where the comment says twice) stays within the bound, whatever the order of its sums.
"""
import numpy as np
import torch

U32 = 2.0 ** -24                                                   # unit roundoffs
UNIT = {torch.float32: U32, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}   # half of the least step


def f64(t):
    return t.detach().cpu().double()


def nibbles(b):
    b = b.long()
    return torch.stack((b & 15, b >> 4), -1).flatten(-2).double()


# ------------------------------------------------------------------ 4-bit products
def q4_weight(codes, scales, zero_points, k):
    """[K, N] values, and the magnitudes that the sums may pass through: codes of bf16 activations are multiplied
    with a bias of 128 that a second product takes off."""
    n, blocks, _ = codes.shape
    z = torch.full((n, blocks), 8.0, dtype=torch.float64) if zero_points is None else nibbles(zero_points)[:, :blocks]
    c = nibbles(codes)
    w = ((c - z[..., None]) * f64(scales)[..., None]).reshape(n, -1)[:, :k]
    big = ((c + 256 + z[..., None]) * f64(scales).abs()[..., None]).reshape(n, -1)[:, :k]
    return w.t(), big.t()


def gemm_q4(a, codes, scales, zero_points, bias=None, rounded_weights=False):
    dt, k = a.dtype, a.shape[1]
    a = f64(a)
    w, big = q4_weight(codes, scales, zero_points, k)
    y, size = a @ w, a.abs() @ (big if dt == torch.bfloat16 else w.abs())
    bound = (k + 64) * U32 * size
    if rounded_weights:   # the weights rounded to the type before the product
        bound = bound + UNIT[dt] * (a.abs() @ w.abs()) + TINY[dt] * a.abs().sum(1, keepdim=True)
    if bias is not None:
        y = y + f64(bias)
        bound = bound + 2 * U32 * (y.abs() + f64(bias).abs())
    return y, bound + UNIT[dt] * (y.abs() + bound) + TINY[dt]


# ------------------------------------------------------------------ the cache
def read_cache(cache):
    """Codes [pages, kv, page, dim] and parameters [pages, kv, page, groups, 2] of keys and of values."""
    kc, vc, kp, vp = (t.cpu() for t in cache.tensors)
    k = nibbles(kc.transpose(3, 4).flatten(3))                               # 32 s + 8 q + 2 b
    v = nibbles(vc.transpose(3, 4).flatten(2, 3)).transpose(3, 4).flatten(3)   # [page, column, code] -> code, column
    return k, v, f64(kp), f64(vp)


def values(codes, params):
    x = codes.unflatten(-1, (params.shape[-2], -1))
    return (x * params[..., :1] + params[..., 1:]).flatten(-2)


def rotate(x, cos, sin, interleaved):
    """(value, bound) of [tokens, heads, dim] turned by the angles of [tokens, rot / 2], products rounded in f32."""
    x, c, s = f64(x), f64(cos)[:, None], f64(sin)[:, None]
    rot = 2 * c.shape[-1]
    i = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
    j = i + (1 if interleaved else rot // 2)
    y, bound = x.clone(), torch.zeros_like(x)
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    size = (x[..., i] * c).abs() + (x[..., j] * s).abs(), (x[..., j] * c).abs() + (x[..., i] * s).abs()
    bound[..., i], bound[..., j] = 3 * U32 * size[0], 3 * U32 * size[1]
    return y, bound


# ------------------------------------------------------------------ attention
def attend(q, k, v, sees, scale, size_k=None, size_v=None, weight=0.0, tiny=0.0):
    """One head: q [a, dim], k and v [b, dim], sees [a, b].  size_k / size_v: the magnitudes that products pass through
    (the values' own by default); weight / tiny: relative and least rounding of the weights (their largest is 1)."""
    size_k, size_v = k.abs() if size_k is None else size_k, v.abs() if size_v is None else size_v
    x = torch.where(sees, q @ k.t() * scale, -torch.inf)
    some = sees.any(1, keepdim=True)
    x = x - torch.where(some, x.amax(1, keepdim=True), 0.0)
    p = torch.exp(x)
    total = torch.where(some, p.sum(1, keepdim=True), 1.0)
    y = torch.where(some, p @ torch.where(sees.any(0)[:, None], v, 0.0) / total, 0.0)
    # a score's f32 error, twice (its own and the maximum's), and that of the exponential's argument
    n = k.shape[0]
    score = (2 * (q.shape[1] + 8) * U32 * scale * (q.abs() @ size_k.t())).amax(1, keepdim=True) if n else 0.0
    arg = 4 * U32 * (1 + torch.where(torch.isfinite(x), x.abs(), 0.0)) if n else 0.0
    seen_v = torch.where(sees.any(0)[:, None], size_v, 0.0)
    rel = score + weight + (2 * n + 64) * U32
    bound = (p * (rel + arg) + torch.where(sees, tiny, 0.0)) @ seen_v / total
    own = (p * (rel + arg) + torch.where(sees, tiny, 0.0)).sum(1, keepdim=True) / total * y.abs()   # of the sum of weights
    return y, torch.where(some, bound + own, 0.0)


def rounded(value, bound, dtype):
    return value, bound + UNIT[dtype] * (value.abs() + bound) + TINY[dtype]


def decode(q, cache, table, lens, scale, window=0):
    kc, vc, kp, vp = read_cache(cache)
    dt, heads = q.dtype, q.shape[1]
    q, table, g = f64(q), table.cpu().long(), heads // cache.kv_heads
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    bias = 1024.0 if dt == torch.float16 else 128.0
    for b in range(q.shape[0]):
        n = max(0, min(int(lens[b]), table.shape[1] * cache.page))
        if not n:
            continue
        ids = table[b, :(n + cache.page - 1) // cache.page]
        known = (ids >= 0) & (ids < cache.pages)
        ids = torch.where(known, ids, 0)
        place = torch.arange(n)
        sees = known[place // cache.page] & (place >= (n - window if window else 0))
        for h in range(cache.kv_heads):
            def rows(x):
                return x[ids, h].flatten(0, 1)[:n]
            k, v = values(rows(kc), rows(kp)), values(rows(vc), rows(vp))
            grp = cache.group
            sk, sv = (((rows(c).unflatten(-1, (-1, grp)) + 2 * by) * rows(p)[..., :1].abs() + rows(p)[..., 1:].abs()).flatten(-2)
                      for c, p, by in ((kc, kp, bias), (vc, vp, 128.0)))
            k, v, sk, sv = (torch.where(sees[:, None], t, 0.0) for t in (k, v, sk, sv))
            hs = slice(h * g, (h + 1) * g)
            # the weights meet the codes in two bf16 parts: 2^-17 of a weight at most
            y, e = attend(q[b, hs], k, v, sees.expand(g, n), scale, sk, sv, weight=0.0)
            w = attend(q[b, hs], k, v, sees.expand(g, n), scale, sk, v.abs() + sv * 0, weight=2.0 ** -16)[1]
            out[b, hs], bound[b, hs] = y, e + w
    return rounded(out, bound, dt)


def prefill(q, k, v, cu_q, cu_k, scale, causal=True, window=0):
    dt, heads, kv = q.dtype, q.shape[1], k.shape[1]
    q, k, v, g = f64(q), f64(k), f64(v), heads // kv
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for i in range(len(cu_q) - 1):
        a, b = slice(int(cu_q[i]), int(cu_q[i + 1])), slice(int(cu_k[i]), int(cu_k[i + 1]))
        nq, nk = a.stop - a.start, b.stop - b.start
        at, key = torch.arange(nq)[:, None] + nk - nq, torch.arange(nk)[None]
        sees = torch.ones((nq, nk), dtype=torch.bool)
        if causal:
            sees &= key <= at
        if window:
            sees &= key > at - window
        if not nq or not nk:
            continue
        for h in range(heads):
            # the weights are rounded to the type (the largest is 1)
            y, e = attend(q[a, h], k[b, h // g], v[b, h // g], sees, scale, weight=UNIT[dt], tiny=TINY[dt])
            out[a, h], bound[a, h] = y, e
    return rounded(out, bound, dt)


def close(got, want):
    value, bound = want
    got = f64(got)
    assert got.shape == value.shape
    off = (got - value).abs()
    assert torch.isfinite(got).all()
    worst = float((off / bound).max()) if off.numel() else 0.0
    assert worst <= 1.0, (worst, float(off.max()), np.unravel_index(int((off / bound).argmax()), off.shape))
