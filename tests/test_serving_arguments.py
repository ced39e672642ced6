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
