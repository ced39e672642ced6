"""Performance cases of the serving operators of a language model: 4-bit products, the paged 4-bit cache of keys and
values, and attention over prompts and over that cache.

`run` computes an operator in its plain form (elementary torch operations in 32 bits, rounded once), or, where `own`
is true, through the public calls of `oxionnx_amd.device.HipContext`.  `listed` names twelve cases, `draw` gives more
from the same ranges.

The cache: pages of `page` tokens.  Of every token and key/value head, groups of `group` channels share a scale and a
minimum (f16 each, `params[page, head, token, group, (scale, minimum)]`); a channel stands for scale * code + minimum.
Codes are 4 bits, the lower channel of a pair in the low bits of its byte.  Keys lie as
`k_codes[page, head, token, q, s, byte]` with channel 32 s + 8 q + 2 byte (+ 1), values as
`v_codes[page, head, token / 16, column, token % 16, byte]` with channel column + 16 (2 byte (+ 1)).
"""
import functools
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # The smallest product: a style projection of one row (512 -> 1024) with 4-bit weights, f32 activations.
        {"name": "q4_small_f32", "kind": "q4", "dtype": "f32", "m": 1, "k": 512, "n": 1024, "group": 32, "zp": True},
        # One token of one user through a 4096 -> 11008 MLP projection.
        {"name": "q4_row_f16", "kind": "q4", "dtype": "f16", "m": 1, "k": 4096, "n": 11008, "group": 128, "zp": False},
        # A decode batch of sixteen users through the way back, 11008 -> 4096, with zero points.
        {"name": "q4_batch_bf16", "kind": "q4", "dtype": "bf16", "m": 16, "k": 11008, "n": 4096, "group": 64, "zp": True},
        # A decode step of eight users: one new token each, all of the work is latency.
        {"name": "append_step_f16", "kind": "append", "dtype": "f16", "tokens": 8, "kv": 8, "g": 4, "dim": 128,
         "group": 64, "page": 64, "rot": 128, "interleaved": False},
        # Prompts of 8191 tokens in all enter the cache at once.
        {"name": "append_prompt_bf16", "kind": "append", "dtype": "bf16", "tokens": 8191, "kv": 8, "g": 4, "dim": 128,
         "group": 64, "page": 64, "rot": 128, "interleaved": False},
        # One user, a short context, as many key heads as query heads.
        {"name": "decode_one_f16", "kind": "decode", "dtype": "f16", "batch": 1, "len": 389, "kv": 12, "g": 1,
         "dim": 64, "group": 32, "page": 16},
        # A serving batch of 64 users with contexts of 512 to 4096 tokens.
        {"name": "decode_batch_bf16", "kind": "decode", "dtype": "bf16", "batch": 64, "len": 4096, "kv": 8, "g": 4,
         "dim": 128, "group": 64, "page": 64},
        # Two users with whole books in the cache.
        {"name": "decode_long_f16", "kind": "decode", "dtype": "f16", "batch": 2, "len": 131071, "kv": 8, "g": 8,
         "dim": 128, "group": 128, "page": 128},
        # A prompt of 197 tokens through twelve heads of 64.
        {"name": "prefill_short_f16", "kind": "prefill", "dtype": "f16", "seqs": 1, "tokens": 197, "kv": 12, "g": 1,
         "dim": 64, "window": 0, "past": 0},
        # Seven prompts of unequal lengths packed into one batch of 8191 tokens, grouped heads.
        {"name": "prefill_packed_bf16", "kind": "prefill", "dtype": "bf16", "seqs": 7, "tokens": 8191, "kv": 8, "g": 4,
         "dim": 128, "window": 0, "past": 0},
        # The last 1000 tokens of a prompt whose first 3000 are already there, within a sliding window.
        {"name": "prefill_chunk_f16", "kind": "prefill", "dtype": "f16", "seqs": 1, "tokens": 1000, "kv": 8, "g": 4,
         "dim": 128, "window": 2048, "past": 3000},
        # One prompt of 8192 tokens: the most work.
        {"name": "prefill_long_bf16", "kind": "prefill", "dtype": "bf16", "seqs": 1, "tokens": 8192, "kv": 8, "g": 4,
         "dim": 128, "window": 0, "past": 0},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["q4", "append", "decode", "prefill"])
    if kind == "q4":
        group = rng.choice([32, 64, 128])
        while True:
            m, k, n = _log_int(rng, 1, 64), _log_int(rng, 64, 11008), _log_int(rng, 32, 11008)
            if rng.random() < 0.5:
                k, n = (k + group - 1) // group * group, (n + 15) // 16 * 16
            if k * n <= 4096 * 11008:
                return {"kind": kind, "dtype": rng.choice(["f32", "f16", "bf16"]), "m": m, "k": k, "n": n,
                        "group": group, "zp": rng.random() < 0.5}
    dtype, kv, g, dim = rng.choice(["f16", "bf16"]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 7, 8]), rng.choice([64, 128])
    if kind == "prefill":
        dim = rng.choice([64, 80, 128])
        while True:
            seqs, past, window = rng.randint(1, 12), rng.choice([0, 0, _log_int(rng, 1, 4096)]), rng.choice([0, 0, _log_int(rng, 8, 2048)])
            tokens = _log_int(rng, seqs, 8192)
            if kv * g * tokens * (tokens + seqs * past) <= 32 * 8192 * 8192:
                return {"kind": kind, "dtype": dtype, "seqs": seqs, "tokens": tokens, "kv": kv, "g": g, "dim": dim,
                        "window": window, "past": past}
    group, page = rng.choice([32, 64, dim]), rng.choice([16, 32, 64, 128])
    if kind == "append":
        return {"kind": kind, "dtype": dtype, "tokens": _log_int(rng, 1, 8191), "kv": kv, "g": min(g, 4), "dim": dim,
                "group": group, "page": page, "rot": rng.choice([dim, dim, dim // 2]), "interleaved": rng.random() < 0.3}
    while True:
        batch, length = _log_int(rng, 1, 128), _log_int(rng, 1, 131071)
        if batch * length * kv * dim <= 2 * 131071 * 8 * 128:
            return {"kind": kind, "dtype": dtype, "batch": batch, "len": length, "kv": kv, "g": g, "dim": dim,
                    "group": group, "page": page}


# ------------------------------------------------------------------ lengths
def _cut(tokens, seqs):
    """`tokens` in `seqs` unequal parts of at least one."""
    weights = [1 + 5 * i % 7 for i in range(seqs)]
    rest, total = tokens - seqs, sum(weights)
    parts = [1 + rest * w // total for w in weights]
    parts[0] += tokens - sum(parts)
    return parts


def _contexts(case):
    """The context lengths of a decode batch, from the longest to an eighth of it."""
    b, n = case["batch"], case["len"]
    return [max(1, n - n * 7 * i // (8 * b)) for i in range(b)]


# ------------------------------------------------------------------ state
# One context per process, as a program has: it holds the stream and the scratch.
@functools.lru_cache(None)
def _ctx():
    from oxionnx_amd.device import HipContext
    return HipContext(0)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _bytes(g, shape):
    return torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _offsets(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def _pools(case, pages, g=None):
    """Codes and parameters of a cache: of an empty one, or (with a generator) of one full of values."""
    kv, dim, page, groups = case["kv"], case["dim"], case["page"], case["dim"] // case["group"]
    shapes = (pages, kv, page, 4, dim // 32, 4), (pages, kv, page // 16, 16, 16, dim // 32)
    p = {}
    for name, shape in zip(("k", "v"), shapes):
        if g is None:
            p[name + "_codes"] = torch.zeros(shape, dtype=torch.uint8, device="cuda")
            p[name + "_params"] = torch.zeros((pages, kv, page, groups, 2), dtype=torch.float16, device="cuda")
        else:
            p[name + "_codes"] = _bytes(g, shape)
            scale = 0.15 + 0.2 * torch.rand((pages, kv, page, groups), generator=g, device="cuda")
            low = -7.5 * scale + 0.3 * torch.randn(scale.shape, generator=g, device="cuda")
            p[name + "_params"] = torch.stack((scale, low), -1).half()
    return p


def _cache(p):
    from oxionnx_amd.device import KvCache
    return KvCache(p["k_codes"], p["v_codes"], p["k_params"], p["v_params"])


def _inputs(case, seed):
    g, kind, dt = _gen(seed), case["kind"], DTYPES[case["dtype"]]
    order = random.Random(seed)
    if kind == "q4":
        m, k, n, group = case["m"], case["k"], case["n"], case["group"]
        blocks = (k + group - 1) // group
        t = {"a": _normal(g, (m, k), dt), "codes": _bytes(g, (n, blocks, group // 2)),
             "scales": ((0.5 + torch.rand((n, blocks), generator=g, device="cuda")) / (4 * math.sqrt(k))).to(dt),
             "zero_points": _bytes(g, (n, (blocks + 1) // 2)) if case["zp"] else None,
             "bias": _normal(g, (n,), dt)}
        return t
    kv, heads, dim = case["kv"], case["kv"] * case["g"], case["dim"]
    if kind == "append":
        # Rows of a joint projection (queries, keys, values); each token has a slot of its own in some page.
        tokens, page = case["tokens"], case["page"]
        pages = (tokens + page - 1) // page + 3
        x = _normal(g, (tokens, heads + 2 * kv, dim), dt)
        start = order.randrange(1, 1024)
        angle = torch.arange(start + tokens, device="cuda")[:, None] * torch.exp(
            torch.arange(0, case["rot"], 2, device="cuda") * (-math.log(10000.0) / case["rot"]))
        shuffled = torch.randperm(pages, generator=g, device="cuda")
        token = torch.arange(tokens, device="cuda")
        slots = shuffled[token // page] * page + token % page
        return {"q": x[:, :heads], "k": x[:, heads:heads + kv], "v": x[:, heads + kv:], "cos": angle.cos().float(),
                "sin": angle.sin().float(), "positions": (token + start).int(), "slots": slots.int(), **_pools(case, pages)}
    if kind == "decode":
        lengths = _contexts(case)
        order.shuffle(lengths)
        page, width = case["page"], (case["len"] + case["page"] - 1) // case["page"]
        need = [(n + page - 1) // page for n in lengths]
        pages = sum(need) + 3
        ids = torch.randperm(pages, generator=g, device="cuda").int()
        table, at = torch.zeros((len(lengths), width), dtype=torch.int32, device="cuda"), 0
        for i, n in enumerate(need):
            table[i, :n] = ids[at:at + n]
            at += n
        return {"q": _normal(g, (len(lengths), heads, dim), dt), "table": table,
                "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"), **_pools(case, pages, g)}
    lengths = _cut(case["tokens"], case["seqs"])
    order.shuffle(lengths)
    cu_q, cu_k = _offsets(lengths), _offsets([n + case["past"] for n in lengths])
    tokens, keys = case["tokens"], case["tokens"] + case["seqs"] * case["past"]
    if case["past"] == 0:   # views of a joint projection's rows
        x = _normal(g, (tokens, heads + 2 * kv, dim), dt)
        q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    else:
        q, k, v = _normal(g, (tokens, heads, dim), dt), _normal(g, (keys, kv, dim), dt), _normal(g, (keys, kv, dim), dt)
    return {"q": q, "k": k, "v": v, "cu_q": cu_q, "cu_k": cu_k}


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if not own:
        return s
    # What a serving program keeps: the context, packed weights, the cache's handle and output buffers.
    s["ctx"], kind = _ctx(), case["kind"]
    if kind == "q4":
        host = [None if t is None else t.cpu().numpy() if t.dtype != torch.bfloat16 else t.view(torch.int16).cpu().numpy()
                for t in (s["codes"], s["scales"], s["zero_points"])]
        s["w"] = s["ctx"].weight_q4(host[0], host[1], zero_points=host[2], k=case["k"], dtype=case["dtype"])
        s["y"] = torch.empty((case["m"], case["n"]), dtype=s["a"].dtype, device="cuda")
    elif kind == "prefill":
        s["y"] = torch.empty(s["q"].shape, dtype=s["q"].dtype, device="cuda")
    else:
        s["cache"] = _cache(s)
        s["y"] = [torch.empty(s[n].shape, dtype=s[n].dtype, device="cuda") for n in ("q", "k", "v") if n in s]
    return s


# ------------------------------------------------------------------ the plain forms
def _nibbles(b):
    """[..., n] bytes -> [..., 2 n] codes in f32."""
    return torch.stack((b & 15, b >> 4), -1).flatten(-2).float()


def _q4(s):
    c = s["case"]
    blocks = s["codes"].shape[1]
    w = _nibbles(s["codes"])
    z = 8.0 if s["zero_points"] is None else _nibbles(s["zero_points"])[:, :blocks, None]
    w = ((w - z) * s["scales"].float()[..., None]).flatten(1)[:, :c["k"]]
    return (s["a"].float() @ w.t() + s["bias"].float()).to(s["a"].dtype)


def _rotate(x, cos, sin, rot, interleaved):
    """The first `rot` channels of [tokens, heads, dim] turned by the angles of [tokens, 1, rot / 2]."""
    head, tail = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = head[..., :rot // 2], head[..., rot // 2:]
        head = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((head, tail), -1)


def _quantise(x, group):
    """Codes [..., groups, group] and parameters [..., groups, 2] of [..., dim] in f32."""
    x = x.unflatten(-1, (-1, group))
    low = x.amin(-1, keepdim=True)
    scale = ((x.amax(-1, keepdim=True) - low) * (1 / 15)).half().float()
    low = low.half().float()
    codes = torch.where(scale > 0, torch.round((x - low) / scale), 0.0).clamp(0.0, 15.0)
    return codes, torch.cat((scale, low), -1).half(), (codes * scale + low).flatten(-2)


def _append(s):
    c = s["case"]
    dim, page = c["dim"], c["page"]
    cos, sin = (s[n][s["positions"].long()][:, None, :] for n in ("cos", "sin"))
    q = _rotate(s["q"].float(), cos, sin, c["rot"], c["interleaved"])
    k = _rotate(s["k"].float(), cos, sin, c["rot"], c["interleaved"])
    at, off = s["slots"].long() // page, s["slots"].long() % page
    kc, kp, held_k = _quantise(k, c["group"])
    vc, vp, held_v = _quantise(s["v"].float(), c["group"])
    kc, vc = (x.flatten(-2).to(torch.uint8) for x in (kc, vc))
    kc, vc = kc.unflatten(-1, (-1, 2)), vc.unflatten(-1, (-1, 2, 16)).transpose(-1, -2)
    kc, vc = kc[..., 0] | (kc[..., 1] << 4), vc[..., 0] | (vc[..., 1] << 4)
    s["k_codes"][at, :, off] = kc.unflatten(-1, (dim // 32, 4, 4)).transpose(2, 3)
    s["v_codes"][at, :, off // 16, :, off % 16] = vc.transpose(2, 3)
    s["k_params"][at, :, off] = kp
    s["v_params"][at, :, off] = vp
    return [x.to(s["q"].dtype) for x in (q, held_k, held_v)]


def _read(codes, params, group):
    """[sequences, tokens, kv, dim] in f32 of codes [sequences, pages, kv, page, dim]."""
    x = codes.unflatten(-1, (-1, group))
    x = (x * params[..., 0:1].float() + params[..., 1:2].float()).flatten(-2)
    return x.transpose(2, 3).flatten(1, 2)


def _decode(s):
    c = s["case"]
    t = s["table"].long()
    k = _nibbles(s["k_codes"][t].transpose(4, 5).flatten(4))
    v = _nibbles(s["v_codes"][t].transpose(4, 5).flatten(3, 4)).transpose(4, 5).flatten(4)
    k, v = _read(k, s["k_params"][t], c["group"]), _read(v, s["v_params"][t], c["group"])
    q = s["q"].float().unflatten(1, (c["kv"], c["g"]))
    x = q @ k.permute(0, 2, 3, 1) * c["dim"] ** -0.5
    inside = torch.arange(x.shape[-1], device=x.device) < s["lengths"][:, None, None, None]
    x = torch.where(inside, x, -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    return (e @ v.transpose(1, 2) / e.sum(-1, keepdim=True)).flatten(1, 2).to(s["q"].dtype)


def _places(cu, tokens):
    """Sequence and place within it of each of `tokens` packed rows."""
    i = torch.arange(tokens, device=cu.device)
    seq = (i[:, None] >= cu[None, 1:]).sum(1)
    return seq, i - cu[seq]


def _prefill(s):
    c = s["case"]
    q, k, v = (s[n].float() for n in ("q", "k", "v"))
    (sq, iq), (sk, ik) = _places(s["cu_q"], q.shape[0]), _places(s["cu_k"], k.shape[0])
    iq = iq + c["past"]
    sees = (sq[:, None] == sk) & (ik <= iq[:, None])
    if c["window"]:
        sees &= ik > iq[:, None] - c["window"]
    q = q.unflatten(1, (c["kv"], c["g"])).permute(1, 2, 0, 3).flatten(1, 2)
    x = (q @ k.permute(1, 2, 0) * c["dim"] ** -0.5).unflatten(1, (c["g"], -1))
    x = torch.where(sees, x, -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    y = e.flatten(1, 2) @ v.transpose(0, 1) / e.sum(-1, keepdim=True).flatten(1, 2)
    return y.unflatten(1, (c["g"], -1)).permute(2, 0, 1, 3).flatten(1, 2).to(s["q"].dtype)


def run(s):
    c = s["case"]
    kind = c["kind"]
    if own:
        ctx = s["ctx"]
        if kind == "q4":
            return ctx.gemm_q4(s["a"], s["w"], s["bias"], out=s["y"])
        if kind == "decode":
            return ctx.attn_decode(s["q"], s["cache"], s["table"], s["lengths"], out=s["y"][0])
        if kind == "prefill":
            return ctx.attn_prefill(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], window=c["window"], out=s["y"])
        y = ctx.kv_append(s["cache"], s["k"], s["v"], s["slots"], q=s["q"], positions=s["positions"], cos=s["cos"],
                          sin=s["sin"], interleaved=c["interleaved"], q_out=s["y"][0], k_out=s["y"][1], v_out=s["y"][2])
    elif kind != "append":
        return {"q4": _q4, "decode": _decode, "prefill": _prefill}[kind](s)
    else:
        y = _append(s)
    # The keys and values are those that the cache now stands for; the cache itself is the state's own.
    return {"q": y[0], "k": y[1], "v": y[2], **{n: s[n] for n in ("k_codes", "v_codes", "k_params", "v_params")}}


# ------------------------------------------------------------------ work
def _pairs(case):
    """Query-key pairs of a prompt's attention that are computed."""
    n, w, past = 0, case["window"] or 1 << 60, case["past"]
    for length in _cut(case["tokens"], case["seqs"]):
        first, last = past + 1, past + length          # keys that the first and last query see without a window
        full = max(0, min(last, w) - first + 1)
        n += (first + min(last, w)) * full // 2 + (length - full) * min(w, last)
    return n


def work(case):
    kind, eb = case["kind"], BYTES[case["dtype"]]
    if kind == "q4":
        m, k, n = case["m"], case["k"], case["n"]
        blocks = (k + case["group"] - 1) // case["group"]
        weights = n * k / 2 + n * blocks * (eb + (0.5 if case["zp"] else 0))
        return {"bytes": weights + eb * (m * k + m * n + n), "flops": 2.0 * m * k * n}
    kv, heads, dim = case["kv"], case["kv"] * case["g"], case["dim"]
    if kind == "prefill":
        keys = case["tokens"] + case["seqs"] * case["past"]
        return {"bytes": 2 * dim * (2 * case["tokens"] * heads + 2 * keys * kv), "flops": 4.0 * dim * heads * _pairs(case)}
    held = 2 * kv * (dim // 2 + 4 * (dim // case["group"]))   # bytes of a token's keys and values in the cache
    if kind == "append":
        t = case["tokens"]
        return {"bytes": t * (2 * 2 * dim * (heads + 2 * kv) + 4 * case["rot"] + 8 + held), "flops": 3.0 * t * case["rot"] * (heads + kv)}
    n = sum(_contexts(case))
    return {"bytes": n * held + 2 * 2 * case["batch"] * heads * dim, "flops": 4.0 * n * heads * dim}


# ------------------------------------------------------------------ 64 bits
def _split_bytes(b):
    x = b.long()
    out = torch.empty(x.shape[:-1] + (2 * x.shape[-1],), dtype=torch.float64, device=x.device)
    out[..., 0::2], out[..., 1::2] = (x % 16).double(), (x // 16).double()
    return out


def _attend(q, k, v, first, window):
    """One head group in 64 bits: q [g, a, dim], k and v [b, dim]; query i stands at place first + i."""
    x = torch.matmul(q, k.t()) / math.sqrt(k.shape[-1])
    i = first + torch.arange(q.shape[1], device=q.device)[:, None]
    j = torch.arange(k.shape[0], device=q.device)[None, :]
    hidden = j > i
    if window:
        hidden |= i - j >= window
    return torch.matmul(torch.softmax(x.masked_fill(hidden, -math.inf), -1), v)


def exact(case, seed):
    t, kind = _inputs(case, seed), case["kind"]
    if kind == "q4":
        n, blocks, _ = t["codes"].shape
        z = torch.full((n, blocks), 8.0, dtype=torch.float64, device="cuda")
        if t["zero_points"] is not None:
            z = _split_bytes(t["zero_points"])[:, :blocks]
        w = (_split_bytes(t["codes"]) - z.unsqueeze(-1)) * t["scales"].double().unsqueeze(-1)
        return torch.addmm(t["bias"].double(), t["a"].double(), w.reshape(n, -1)[:, :case["k"]].t().contiguous())
    kv, g, dim, group = case["kv"], case["g"], case["dim"], case.get("group")
    if kind == "prefill":
        out = torch.empty(t["q"].shape, dtype=torch.float64, device="cuda")
        a, b = t["cu_q"].tolist(), t["cu_k"].tolist()
        for i in range(case["seqs"]):
            for h in range(kv):
                q = t["q"][a[i]:a[i + 1], h * g:(h + 1) * g].double().transpose(0, 1)
                k, v = (t[n][b[i]:b[i + 1], h].double() for n in ("k", "v"))
                out[a[i]:a[i + 1], h * g:(h + 1) * g] = _attend(q, k, v, case["past"], case["window"]).transpose(0, 1)
        return out
    if kind == "append":
        angle = [t[n][t["positions"].long()].double().unsqueeze(1) for n in ("cos", "sin")]
        half = case["rot"] // 2
        even = torch.arange(0, case["rot"], 2, device="cuda") if case["interleaved"] else torch.arange(half, device="cuda")
        odd = even + (1 if case["interleaved"] else half)
        out = []
        for name in ("q", "k", "v"):
            x = t[name].double()
            if name != "v":
                y = x.clone()
                y[..., even] = x[..., even] * angle[0] - x[..., odd] * angle[1]
                y[..., odd] = x[..., odd] * angle[0] + x[..., even] * angle[1]
                x = y
            if name != "q":
                x = x.reshape(x.shape[0], kv, -1, group)
                low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
                step, low = ((high - low) / 15).half().double(), low.half().double()
                x = (torch.clamp(torch.round((x - low) / step.clamp_min(1e-30)), 0, 15) * step + low).reshape(-1, kv, dim)
            out.append(x)
        return {"q": out[0], "k": out[1], "v": out[2], "k_codes": None, "v_codes": None, "k_params": None, "v_params": None}
    out = torch.empty(t["q"].shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(t["lengths"].tolist()):
        ids = t["table"][i, :(n + case["page"] - 1) // case["page"]].long()
        for h in range(kv):
            kc = _split_bytes(t["k_codes"][ids, h].permute(0, 1, 3, 2, 4).reshape(-1, dim // 2))
            vc = _split_bytes(t["v_codes"][ids, h].permute(0, 1, 3, 2, 4).reshape(-1, 16, dim // 32)).transpose(1, 2)
            rows = []
            for codes, params in ((kc, t["k_params"]), (vc, t["v_params"])):
                p = params[ids, h].reshape(-1, dim // group, 2).double()
                x = codes.reshape(-1, dim // group, group)
                rows.append((x * p[..., :1] + p[..., 1:]).reshape(-1, dim)[:n])
            q = t["q"][i, h * g:(h + 1) * g].double().unsqueeze(1)
            out[i, h * g:(h + 1) * g] = _attend(q, rows[0], rows[1], n - 1, 0).squeeze(1)
    return out
