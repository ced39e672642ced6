"""Arguments of the serving calls on the host: what reaches the library, and what is refused before it does."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oxionnx_amd import _lib as L  # noqa: E402
from oxionnx_amd import device as D  # noqa: E402


class _Recorder:
    """Stands for a HipContext and its library: records the operands of ohip_weight_q4."""
    h, device = None, -1

    def __init__(self, monkeypatch):
        self._weights, self.calls = set(), []
        monkeypatch.setattr(L, "lib", lambda: self)

    def ohip_weight_q4(self, h, key, codes, k, n, group, dtype, scales, zero_points, out):
        size = n * (-(-k // group)) * L.ELEM_BYTES[dtype]
        self.calls.append((k, n, group, dtype, ctypes.string_at(scales, size), zero_points))
        return L.OK

    def ohip_weight_release(self, h):
        pass


@pytest.mark.parametrize("name, code, tdt", [("f32", L.F32, torch.float32), ("f16", L.F16, torch.float16),
                                             ("bf16", L.BF16, torch.bfloat16)])
def test_weight_types_by_name_and_scales_as_bits(monkeypatch, name, code, tdt):
    """A type's name stands for its code, and bfloat16 scales may come as their bits (numpy has no such type)."""
    rec = _Recorder(monkeypatch)
    codes = np.zeros((5, 3, 16), np.uint8)
    scales = (torch.rand((5, 3), generator=torch.Generator().manual_seed(1)) + 0.5).to(torch.bfloat16)
    want = scales.to(tdt).view(torch.uint8).numpy().tobytes()
    bits = scales.view(torch.int16).numpy()
    for given in (bits, bits.view(np.uint16), np.asfortranarray(bits), scales.float().numpy()):
        for dtype in (name, code):
            D.HipContext.weight_q4(rec, codes, given, k=90, dtype=dtype)
    assert rec.calls == [(90, 5, 32, code, want, None)] * 8


def test_weight_type_by_default(monkeypatch):
    rec = _Recorder(monkeypatch)
    codes = np.zeros((2, 1, 16), np.uint8)
    for scales, code in ((np.ones((2, 1), np.float32), L.F32), (np.ones((2, 1), np.float16), L.F16),
                         (np.full((2, 1), 0x3f80, np.uint16), L.BF16)):
        D.HipContext.weight_q4(rec, codes, scales)
        assert rec.calls[-1][3] == code
    with pytest.raises(L.OhipError):
        D.HipContext.weight_q4(rec, codes, np.ones((2, 1), np.float32), dtype="f64")


class _Context:
    """A HipContext of tensors on the host; its library must not be reached."""
    h, device = None, -1
    gemm_q4, kv_append = D.HipContext.gemm_q4, D.HipContext.kv_append
    attn_decode, attn_prefill = D.HipContext.attn_decode, D.HipContext.attn_prefill


@pytest.fixture
def host_ctx(monkeypatch):
    def raw(name):
        raise AssertionError(f"{name} was reached")
    monkeypatch.setattr(L, "raw", raw)
    return _Context()


def _ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _cache():
    params = (3, 2, 16, 2, 2)
    return D.KvCache(torch.zeros((3, 2, 16, 4, 2, 4), dtype=torch.uint8), torch.zeros((3, 2, 1, 16, 16, 2), dtype=torch.uint8),
                     torch.zeros(params, dtype=torch.float16), torch.zeros(params, dtype=torch.float16))


def _rows(tokens, heads, shared):
    """[tokens, heads, 64] of which (shared) all tokens are one, or neighbours overlap."""
    if shared == "expanded":
        return torch.zeros((1, heads, 64), dtype=torch.float16).expand(tokens, heads, 64)
    if shared == "overlapping":
        return torch.zeros(tokens * 64 * heads, dtype=torch.float16).as_strided((tokens, heads, 64), (8, 64, 1))
    return torch.zeros((tokens, heads, 64), dtype=torch.float16)


@pytest.mark.parametrize("shared", ["expanded", "overlapping"])
@pytest.mark.parametrize("at", ["a", "out"])
def test_product_refuses_rows_that_share_memory(host_ctx, shared, at):
    class _Weight:
        shape, handle = (64, 64), None
    t = {"a": _rows(8, 1, None)[:, 0], "out": _rows(8, 1, None)[:, 0], at: _rows(8, 1, shared)[:, 0]}
    with pytest.raises(L.OhipError):
        host_ctx.gemm_q4(t["a"], _Weight(), out=t["out"])


@pytest.mark.parametrize("shared", ["expanded", "overlapping"])
@pytest.mark.parametrize("at", ["q", "k", "v", "q_out", "k_out", "v_out"])
def test_append_refuses_tokens_that_share_memory(host_ctx, shared, at):
    t = {n: _rows(8, 4 if n[0] == "q" else 2, shared if n == at else None) for n in ("q", "k", "v", "q_out", "k_out", "v_out")}
    with pytest.raises(L.OhipError):
        host_ctx.kv_append(_cache(), t.pop("k"), t.pop("v"), _ints(8), **t)


@pytest.mark.parametrize("shared", ["expanded", "overlapping"])
@pytest.mark.parametrize("at", ["q", "k", "v", "out"])
def test_attention_refuses_tokens_that_share_memory(host_ctx, shared, at):
    t = {n: _rows(8, 2 if n in "kv" else 4, shared if n == at else None) for n in ("q", "k", "v", "out")}
    with pytest.raises(L.OhipError):
        host_ctx.attn_prefill(t["q"], t["k"], t["v"], _ints(2), out=t["out"])
    if at in ("q", "out"):
        with pytest.raises(L.OhipError):
            host_ctx.attn_decode(t["q"], _cache(), _ints(8, 1), _ints(8), out=t["out"])


def test_tokens_of_one_row_may_have_any_stride():
    assert D._heads(torch.zeros((1, 4, 64), dtype=torch.float16).expand(1, 4, 64), "q", torch.float16, -1) == 256
    assert D._heads(torch.zeros((5, 300), dtype=torch.float16)[:, :256].view(5, 4, 64), "q", torch.float16, -1) == 300


def test_append_refuses_half_of_a_rotation_and_of_queries(host_ctx):
    k, angles, at = _rows(8, 2, None), torch.zeros((4, 32)), _ints(8)
    for kw in ({"cos": angles, "sin": angles}, {"cos": angles, "positions": at}, {"sin": angles, "positions": at},
               {"sin": angles}, {"q_out": _rows(8, 4, None)}):
        with pytest.raises(L.OhipError):
            host_ctx.kv_append(_cache(), k, k, _ints(8), **kw)


@pytest.mark.parametrize("window", [2 ** 31, 2 ** 32 + 5, -2 ** 31 - 1, 2 ** 63])
def test_windows_beyond_the_descriptor_are_refused(host_ctx, window):
    """(their low bits would be another window)"""
    q = _rows(8, 4, None)
    with pytest.raises(L.OhipError):
        host_ctx.attn_prefill(q, q, q, _ints(2), window=window)
    with pytest.raises(L.OhipError):
        host_ctx.attn_decode(q, _cache(), _ints(8, 1), _ints(8), window=window)


def test_integers_beyond_a_descriptor_are_refused():
    for packer in (D._GEMM, D._CONV, D._CONVT, D._MATMUL, D._GEMM_Q4, D._KV_CACHE, D._KV_APPEND, D._ATTN_DECODE, D._ATTN_PREFILL):
        fields = packer._desc._fields_
        for i, (_, t) in enumerate(fields):
            if t in (ctypes.c_int, ctypes.c_int64):
                bits = 8 * ctypes.sizeof(t)
                for v in (2 ** (bits - 1), -2 ** (bits - 1) - 1, 2 ** bits + 1):
                    with pytest.raises(L.OhipError):
                        packer(*(v if j == i else 1 for j in range(len(fields))))
