"""Bounds that a wrong result cannot meet: 4-bit products element by element, attention over the cache by the norm of a
head's row.

Every rounding of an f32 sum is at most U32 of the partial sum that it rounds, and a partial sum of terms of either sign
is about as large as their norm.  n such errors, of independent signs, count as eight times sqrt(n) of one at its largest
(eight standard deviations and more): added up as they are they exceed the values themselves over long sums.
"""
import torch

from tests._serving_ref import TINY, U32, UNIT, f64, nibbles, read_cache, values

SIGMAS = 8.0


# ------------------------------------------------------------------ 4-bit products
def gemm_q4(a, codes, scales, zero_points, bias=None):
    """(value, bound) of products whose codes are multiplied as they are.  A group's sum has a term for each k (of bf16
    two, with 128 + c and -(128 + z)), and each addition rounds."""
    dt, k = a.dtype, a.shape[1]
    n, blocks, half = codes.shape
    group = 2 * half
    z = torch.full((n, blocks), 8.0, dtype=torch.float64) if zero_points is None else nibbles(zero_points)[:, :blocks]
    s = f64(scales)
    w = ((nibbles(codes) - z[..., None]) * s[..., None]).reshape(n, -1)
    a = torch.nn.functional.pad(f64(a), (0, blocks * group - k))
    w[:, k:] = 0.0
    y = a @ w.t()
    norms = a.unflatten(1, (blocks, group)).norm(dim=-1)                    # [m, blocks]
    terms, most = (2, 143.0) if dt == torch.bfloat16 else (1, 15.0)
    total = (terms * group + 4) * most ** 2 * (norms.square() @ s.square().t())
    groups = a.unflatten(1, (blocks, group)).transpose(0, 1).contiguous() @ w.t().unflatten(0, (blocks, group)).contiguous()
    total = total + (blocks + 16) * groups.square().sum(0)                  # sums of groups, and of waves
    bound = SIGMAS * U32 * total.sqrt()
    if bias is not None:
        y = y + f64(bias)
        bound = bound + 2 * U32 * (y.abs() + f64(bias).abs())
    return y, bound + UNIT[dt] * (y.abs() + bound) + TINY[dt]


# ------------------------------------------------------------------ attention over the cache
def decode(q, cache, table, lens, scale, window=0):
    """(rows, limits): rows [batch, heads, dim] and what the norm of a row's error may be at most."""
    kc, vc, kp, vp = read_cache(cache)
    dt, heads, dim, grp = q.dtype, q.shape[1], q.shape[2], cache.group
    q, table, g, groups = f64(q), table.cpu().long(), heads // cache.kv_heads, cache.dim // cache.group
    out, limit = torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64)
    # the codes' bias: of f16 channels 1024 and 64, two of each in turn (their root mean square), of bf16 128
    bias = ((1024.0 ** 2 + 64.0 ** 2) / 2) ** 0.5 if dt == torch.float16 else 128.0
    for b in range(q.shape[0]):
        n = max(0, min(int(lens[b]), table.shape[1] * cache.page))
        if not n:
            continue
        ids = table[b, :(n + cache.page - 1) // cache.page]
        known = (ids >= 0) & (ids < cache.pages)
        ids, place = torch.where(known, ids, 0), torch.arange(n)
        sees = known[place // cache.page] & (place >= (n - window if window else 0))
        if not sees.any():
            continue
        step = (place // 32)[sees]
        for h in range(cache.kv_heads):
            def rows(x):
                return x[ids, h].flatten(0, 1)[:n][sees]
            ks, km, vs, vm = rows(kp)[..., 0], rows(kp)[..., 1], rows(vp)[..., 0], rows(vp)[..., 1]   # [tokens, groups]
            k, v = values(rows(kc), rows(kp)), values(rows(vc), rows(vp))
            qh = q[b, h * g:(h + 1) * g]
            x = qh @ k.t() * scale                                                                    # [g, tokens]
            x = x - x.amax(1, keepdim=True)
            p = torch.exp(x)
            p = p / p.sum(1, keepdim=True)
            o = p @ v
            out[b, h * g:(h + 1) * g] = o
            # scores: partial sums of a group are about the norm of its terms, 3 * group of them are rounded
            qg = qh.unflatten(1, (groups, grp))
            part = qg.norm(dim=-1) * (bias + 15.0) * (3 * grp) ** 0.5                                 # [g, groups]
            low = qg.norm(dim=-1) * grp * 3 ** 0.5
            err = (U32 * scale) ** 2 * (part.square() @ ks.square().t() + low.square() @ km.square().t())
            err = err + (4 * U32 * (1 + x.abs())) ** 2                                                # the exponentials
            away = (v.square().sum(1)[None] - 2 * o @ v.t() + o.square().sum(1, keepdim=True)).clamp_min(0.0)
            total = (p.square() * err * away).sum(1)
            # weights in two bf16 parts: 2^-16 of a weight, times codes of at most 8 from the middle
            total = total + (p.square() @ (2.0 ** -16 * 8 * vs).square().sum(1, keepdim=True))[:, 0] * grp
            # a step's products pass through 136 times its weights; the minima's sums
            weights = torch.zeros((g, int(step.max()) + 1, groups), dtype=torch.float64)
            weights.index_add_(1, step, p[..., None] * vs.abs()[None])
            total = total + ((136 * U32 * 128 ** 0.5 * weights).square().sum((1, 2))) * grp
            middle = (p @ (vm + 8 * vs).abs()).square().sum(1) * grp
            total = total + n * U32 ** 2 * (middle + o.square().sum(1))
            rest = SIGMAS * total.sqrt()
            limit[b, h * g:(h + 1) * g] = rest + UNIT[dt] * (o.norm(dim=1) + rest) + TINY[dt] * dim ** 0.5
    return out, limit


def rows_off(got, want):
    """The norm of each row's error over what it may be."""
    value, limit = want
    off = (f64(got) - value).norm(dim=-1)
    return torch.where(limit > 0, off / limit.clamp_min(1e-300), torch.where(off > 0, torch.inf, 0.0))


def close_rows(got, want):
    ratio = rows_off(got, want)
    assert not ratio.isnan().any()
    assert ratio.numel() == 0 or float(ratio.max()) <= 1.0, (float(ratio.max()), [int(i) for i in (ratio == ratio.max()).nonzero()[0]])
