"""The serving operators on the host: packed descriptors, the cache's argument checks, and the references that the GPU
tests compare with."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oxionnx_amd import _lib as L  # noqa: E402
from oxionnx_amd import device as D  # noqa: E402
from tests import _serving_ref as R  # noqa: E402


@pytest.mark.parametrize("packer", [D._GEMM_Q4, D._KV_CACHE, D._KV_APPEND, D._ATTN_DECODE, D._ATTN_PREFILL],
                         ids=lambda p: p._desc.__name__)
def test_packed_bytes_are_the_structure(packer):
    desc, rng = packer._desc, np.random.default_rng(5)
    values = [float(np.float32(rng.normal())) if t is ctypes.c_float else int(rng.integers(1, 1000)) + i
              for i, (_, t) in enumerate(desc._fields_)]
    got, want = desc.from_buffer_copy(packer(*values)), desc(*values)
    for name, _ in desc._fields_:
        assert getattr(got, name) == getattr(want, name), name


def _cache(pages=3, page=32, kv=2, dim=64, group=32):
    params = (pages, kv, page, dim // group, 2)
    return [torch.zeros((pages, kv, page, 4, dim // 32, 4), dtype=torch.uint8),
            torch.zeros((pages, kv, page // 16, 16, 16, dim // 32), dtype=torch.uint8),
            torch.zeros(params, dtype=torch.float16), torch.zeros(params, dtype=torch.float16)]


def test_cache_of_tensors():
    c = D.KvCache(*_cache())
    assert (c.pages, c.page, c.kv_heads, c.dim, c.group) == (3, 32, 2, 64, 32)
    assert c.nbytes == 3 * 2 * 32 * (2 * 32 + 2 * 2 * 2 * 2)
    d = L.KvCacheDesc.from_buffer_copy(c.desc)
    assert (d.pages, d.page, d.kv_heads, d.head_dim, d.group) == (3, 32, 2, 64, 32)
    assert [d.k_codes, d.v_codes, d.k_params, d.v_params] == [t.data_ptr() for t in c.tensors]


@pytest.mark.parametrize("i, change", [
    (0, lambda t: t[:, :, :, :3].contiguous()), (0, lambda t: t.flatten(4)), (0, lambda t: t.to(torch.int8)),
    (0, lambda t: t.transpose(1, 2)), (1, lambda t: t[:2]), (1, lambda t: t[:, :, :1]), (2, lambda t: t.float()),
    (2, lambda t: t[..., :1]), (2, lambda t: t[:, :, :, :0]), (3, lambda t: t[:, :1]), (3, lambda t: t.flatten(3))])
def test_cache_refuses(i, change):
    tensors = _cache()
    tensors[i] = change(tensors[i])
    with pytest.raises(L.OhipError):
        D.KvCache(*tensors)


@pytest.mark.parametrize("args", [(0, 16, 1, 64, 64), (2, 24, 1, 64, 64), (2, 16, 0, 64, 64), (2, 16, 1, 80, 80),
                                  (2, 16, 1, 64, 0), (2, 16, 1, 64, 48), (2, 16, 1, 64, 128)])
def test_empty_cache_refuses(args):
    with pytest.raises(L.OhipError):
        D.KvCache.empty(*args)


def test_cache_layout_of_the_reference():
    """Channel and token of every code, from the layout's description."""
    c = D.KvCache(*_cache(pages=2, page=32, kv=1, dim=64))
    rng = np.random.default_rng(1)
    for t in c.tensors[:2]:
        t.copy_(torch.from_numpy(rng.integers(0, 256, t.shape, dtype=np.uint8)))
    k, v, _, _ = R.read_cache(c)
    kc, vc = (t.numpy() for t in c.tensors[:2])
    for token in (0, 5, 16, 31):
        for ch in range(64):
            byte = kc[1, 0, token, ch % 32 // 8, ch // 32, ch % 8 // 2]
            assert k[1, 0, token, ch] == (byte >> 4 if ch % 2 else byte & 15)
            byte = vc[1, 0, token // 16, ch % 16, token % 16, ch // 32]
            assert v[1, 0, token, ch] == (byte >> 4 if ch % 32 >= 16 else byte & 15)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_of_the_reference(interleaved):
    x = torch.randn(5, 2, 64, dtype=torch.float64)
    a = torch.rand(5, 16, dtype=torch.float64) * 6
    got, _ = R.rotate(x, a.cos(), a.sin(), interleaved)
    pairs = x[..., :32].unflatten(-1, (16, 2)) if interleaved else torch.stack((x[..., :16], x[..., 16:32]), -1)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(a), a)[:, None])
    want = turned.flatten(-2) if interleaved else torch.cat((turned[..., 0], turned[..., 1]), -1)
    torch.testing.assert_close(got, torch.cat((want, x[..., 32:]), -1), rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("causal, window", [(True, 0), (False, 0), (True, 7)])
def test_attention_of_the_reference(causal, window):
    nq, nk = 20, 26
    q, k, v = torch.randn(nq, 4, 16).half(), torch.randn(nk, 2, 16).half(), torch.randn(nk, 2, 16).half()
    got, _ = R.prefill(q, k, v, torch.tensor([0, nq]), torch.tensor([0, nk]), 0.25, causal, window)
    i, j = torch.arange(nq)[:, None] + nk - nq, torch.arange(nk)
    sees = torch.ones(nq, nk, dtype=torch.bool)
    if causal:
        sees &= j <= i
    if window:
        sees &= j > i - window
    for h in range(4):
        s = (q[:, h].double() @ k[:, h // 2].double().t() * 0.25).masked_fill(~sees, -torch.inf)
        torch.testing.assert_close(got[:, h], torch.softmax(s, 1) @ v[:, h // 2].double(), rtol=1e-12, atol=1e-12)


def test_weight_arguments_are_checked_first():
    """Refusals of shapes that no context is needed for."""
    w = D.HipContext.weight_q4
    codes, scales = np.zeros((4, 2, 16), np.uint8), np.ones((4, 2), np.float16)
    for args, kw in [((codes[0], scales), {}), ((codes.astype(np.int8), scales), {}), ((codes, scales[:, :1]), {}),
                     ((codes, scales), {"k": 32}), ((codes, scales), {"k": 65}), ((codes, scales), {"dtype": L.I8}),
                     ((codes, scales, np.zeros((4, 2), np.uint8)), {}), ((codes, scales, np.zeros((4, 1), np.int8)), {})]:
        with pytest.raises(L.OhipError):
            w(None, *args, **kw)
