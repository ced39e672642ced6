"""Device-level Python handle over the C ABI, with torch tensors as device memory.

PyTorch only provides allocation and the stream here; every contraction runs
in libohip.so.  The context adopts torch's current stream so library work and
torch work are ordered without extra synchronisation.
"""
import ctypes
import math
import struct

import numpy as np

from . import _lib as L

# torch.dtype -> element code, and back; filled with the first use of torch
_OHIP_DT = {}
_TORCH_DT = {}


def _torch():
    import torch
    if not _OHIP_DT:
        _TORCH_DT.update({L.F32: torch.float32, L.F16: torch.float16, L.BF16: torch.bfloat16, L.U8: torch.uint8,
                          L.I8: torch.int8, L.I32: torch.int32})
        _OHIP_DT.update({t: d for d, t in _TORCH_DT.items()})
    return torch


def torch_dtype(dt):
    _torch()
    return _TORCH_DT[dt]


def ohip_dtype(tdt):
    if not _OHIP_DT:
        _torch()
    return _OHIP_DT[tdt]


class _Packer:
    """Packs a descriptor of the single-operator calls in C's native layout (its
    ctypes structure and the pointer objects cost a call more than the launch).
    Values that only the structure takes (a float beyond f32) go through it."""

    def __init__(self, fmt, desc):
        self._pack, self._desc = struct.Struct(fmt).pack, desc
        assert struct.calcsize(fmt) == ctypes.sizeof(desc), "descriptor layout"

    def __call__(self, *values):
        try:
            return self._pack(*values)
        except (struct.error, OverflowError):
            types = [t for _, t in self._desc._fields_]
            d = self._desc(*(ctypes.cast(v, t) if issubclass(t, ctypes._Pointer) else v
                             for v, t in zip(values, types)))
            for (name, t), v in zip(self._desc._fields_, values):   # ctypes would take an integer's low bits
                if t in (ctypes.c_int, ctypes.c_int64) and getattr(d, name) != v:
                    raise L.OhipError(L.E_INVALID, f"{name} = {v} is out of range")
            return bytes(d)


_GEMM = _Packer("@3q2i2f2i2f2q", L.GemmDesc)
_CONV = _Packer("@16q4i2fi0q", L.ConvDesc)
_CONVT = _Packer("@18qi0q", L.ConvTDesc)
_MATMUL = _Packer("@6qi0q", L.MatMulDesc)
_QGEMM = _Packer("@3qiP2i2f3i2q", L.QGemmDesc)
_GEMM_Q4 = _Packer("@3q2i2f2q", L.GemmQ4Desc)
_KV_CACHE = _Packer("@q4i4P", L.KvCacheDesc)
_KV_APPEND = _Packer("@q5i7q", L.KvAppendDesc)
_ATTN_DECODE = _Packer("@q4if2q", L.AttnDecodeDesc)
_ATTN_PREFILL = _Packer("@3q6if4q", L.AttnPrefillDesc)
# the zero points that one byte can hold, for calls with a single one
_ZERO_POINTS = np.arange(-128, 256, dtype=np.int32)
_ZERO_POINTS_AT = _ZERO_POINTS.ctypes.data
_TYPE_NAMES = {"f32": L.F32, "f16": L.F16, "bf16": L.BF16}


def _out_dim(size, pad_begin, pad_end, k, dil, stride):
    """ohip_conv_out_dim."""
    if stride <= 0 or k <= 0 or dil <= 0 or size < 0 or pad_begin < 0 or pad_end < 0:
        return -1
    room = size + pad_begin + pad_end - (k - 1) * dil - 1
    return -1 if room < 0 else room // stride + 1


def _np_ohip_dtype(a):
    return {np.dtype(np.float32): L.F32, np.dtype(np.float16): L.F16, np.dtype(np.uint8): L.U8,
            np.dtype(np.int8): L.I8}[a.dtype]


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _key(name, label):
    if name is None:
        return None
    return ctypes.byref(L.WeightKey(name.encode(), (label or "").encode()))


def _invalid(msg):
    return L.OhipError(L.E_INVALID, msg)


def _heads(t, name, dtype, device):
    """Checks [tokens, heads, channels] of a 16-bit `dtype` on GPU `device`, heads next to each other;
    the elements between tokens."""
    strides = t.stride()
    if t.dtype != dtype or t.get_device() != device or len(strides) != 3:
        raise _invalid(f"{name}: [tokens, heads, channels] of {dtype} on GPU {device} is expected")
    tokens, heads, dim = t.shape
    if (strides[2] != 1 and dim > 1) or (strides[1] != dim and heads > 1):
        raise _invalid(f"{name}: a token's heads are not next to each other")
    if tokens > 1 and strides[0] < heads * dim:   # (a stride of 0, an expanded tensor's, is the library's "packed")
        raise _invalid(f"{name}: tokens share memory")
    return strides[0] if tokens > 1 else heads * dim


def _table(t, name, dtype, device, shape):
    if t.dtype != dtype or t.get_device() != device or t.shape != shape or not t.is_contiguous():
        raise _invalid(f"{name}: a contiguous {dtype} array of {tuple(shape)} on GPU {device} is expected")
    return t.data_ptr()


class KvCache:
    """A paged cache of keys and values in 4 bits (the layout is ohip_kv_cache's, include/ohip.h), in
    caller-owned tensors: codes uint8 [pages, kv_heads, page, 4, head_dim / 32, 4] of the keys and
    [pages, kv_heads, page / 16, 16, 16, head_dim / 32] of the values, and float16
    [pages, kv_heads, page, head_dim / group, 2] scales and minima of each."""

    def __init__(self, k_codes, v_codes, k_params, v_params):
        torch = _torch()
        if k_codes.dim() != 6 or k_params.dim() != 5 or 0 in k_params.shape:
            raise _invalid("KvCache: codes or parameters of another rank, or empty")
        pages, kv, page, _, words, _ = k_codes.shape
        self.device, self.dim, groups = k_codes.get_device(), 32 * words, k_params.shape[3]
        self.pages, self.page, self.kv_heads, self.group = pages, page, kv, self.dim // groups
        want = (((pages, kv, page, 4, words, 4), torch.uint8), ((pages, kv, page // 16, 16, 16, words), torch.uint8),
                ((pages, kv, page, groups, 2), torch.float16), ((pages, kv, page, groups, 2), torch.float16))
        self.tensors = (k_codes, v_codes, k_params, v_params)
        for t, (shape, dtype) in zip(self.tensors, want):
            if tuple(t.shape) != shape or t.dtype != dtype or not t.is_contiguous() or t.get_device() != self.device:
                raise _invalid(f"KvCache: a contiguous {dtype} tensor of {shape} on one device is expected")
        if page % 16 or self.group * groups != self.dim:
            raise _invalid("KvCache: pages are a multiple of 16 tokens, groups divide the head")
        self.desc = _KV_CACHE(pages, page, kv, self.dim, self.group, *(t.data_ptr() for t in self.tensors))

    @staticmethod
    def empty(pages, page, kv_heads, head_dim, group=64, device=0):
        """A cache of zeros."""
        if min(pages, page, kv_heads, head_dim, group) <= 0 or page % 16 or head_dim % 32 or head_dim % group:
            raise _invalid("KvCache: pages are a multiple of 16 tokens, heads of 32 channels, groups divide the head")
        torch = _torch()
        at = torch.device("cuda", device)
        params = (pages, kv_heads, page, head_dim // group, 2)
        return KvCache(torch.zeros((pages, kv_heads, page, 4, head_dim // 32, 4), dtype=torch.uint8, device=at),
                       torch.zeros((pages, kv_heads, page // 16, 16, 16, head_dim // 32), dtype=torch.uint8, device=at),
                       torch.zeros(params, dtype=torch.float16, device=at),
                       torch.zeros(params, dtype=torch.float16, device=at))

    @property
    def nbytes(self):
        return sum(t.nbytes for t in self.tensors)


class Weight:
    """A packed, device-resident operand (cached in the context when keyed)."""

    def __init__(self, ctx, handle, kind, dtype, shape, cached):
        self.ctx, self.handle, self.kind, self.dtype, self.shape, self.cached = ctx, handle, kind, dtype, shape, cached
        ctx._weights.add(self)

    @property
    def nbytes(self):
        return L.lib().ohip_weight_bytes(self.handle)

    def release(self):
        if self.handle is not None and not self.cached:
            L.lib().ohip_weight_release(self.handle)
        self.handle = None

    def __del__(self):
        try:
            self.release()
        except Exception:
            pass


class HipContext:
    """Owns one ohip_ctx on one GPU (oxionnx-cuda's CudaContext counterpart)."""

    def __init__(self, device=0, adopt_torch_stream=True):
        import weakref
        torch = _torch()
        self.device = device
        self._weights = weakref.WeakSet()
        self._dtensors = weakref.WeakSet()
        h = ctypes.c_void_p()
        L.check(L.lib().ohip_ctx_create(device, ctypes.byref(h)))
        self.h = h
        if adopt_torch_stream:
            # torch's default stream is the legacy null stream (handle 0); the
            # context's own stream is a blocking stream, which the null stream
            # already orders against, so only a non-default torch stream is
            # adopted explicitly.
            with torch.cuda.device(device):
                s = torch.cuda.current_stream(device).cuda_stream
            if s:
                L.check(L.lib().ohip_ctx_set_stream(self.h, ctypes.c_void_p(s)))

    def close(self):
        if self.h:
            for w in list(self._weights):
                w.handle = None       # the context frees every weight it owns
            for t in list(self._dtensors):
                t.free()              # device tensors return their buffers to the context's pool
            L.lib().ohip_ctx_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # --------------------------------------------------------------- admin
    def sync(self):
        L.check(L.lib().ohip_sync(self.h))

    def set_tile(self, tile_id):
        """Force the MFMA block tile by id (include/ohip.h); 0 = automatic."""
        L.check(L.lib().ohip_set_tile_override(self.h, tile_id))

    def tuning(self):
        t = L.Tuning()
        L.check(L.lib().ohip_get_tuning(self.h, ctypes.byref(t)))
        return t

    def set_tuning(self, t):
        L.check(L.lib().ohip_set_tuning(self.h, ctypes.byref(t)))

    def counters(self):
        c = L.Counters()
        L.check(L.lib().ohip_get_counters(self.h, ctypes.byref(c)))
        return {f: getattr(c, f) for f, _ in L.Counters._fields_}

    def reset_counters(self):
        L.check(L.lib().ohip_reset_counters(self.h))

    def stream(self):
        return L.lib().ohip_ctx_stream(self.h)

    # --------------------------------------------------------------- weights
    def weight_gemm(self, b, trans_b=False, dtype=L.F32, name=None, label="Gemm.B"):
        b = np.ascontiguousarray(b)
        if b.dtype == np.float64:
            b = b.astype(np.float32)
        k, n = (b.shape[1], b.shape[0]) if trans_b else b.shape
        h = ctypes.c_void_p()
        L.check(L.lib().ohip_weight_gemm(self.h, _key(name, label), _np_ohip_dtype(b),
                                         b.ctypes.data_as(ctypes.c_void_p), k, n, int(trans_b), dtype,
                                         ctypes.byref(h)))
        return Weight(self, h, "gemm", dtype, (k, n), name is not None)

    def weight_conv(self, w, dtype=L.F32, name=None, label="Conv.W"):
        w = np.ascontiguousarray(w)
        if w.dtype == np.float64:
            w = w.astype(np.float32)
        h = ctypes.c_void_p()
        L.check(L.lib().ohip_weight_conv(self.h, _key(name, label), _np_ohip_dtype(w),
                                         w.ctypes.data_as(ctypes.c_void_p), *w.shape, dtype, ctypes.byref(h)))
        return Weight(self, h, "conv", dtype, w.shape, name is not None)

    def weight_conv_transpose(self, w, dtype=L.F32, strides=(1, 1), pads=(0, 0, 0, 0), dilations=(1, 1),
                              group=1, name=None, label="ConvTranspose.W"):
        """ConvTranspose filter [Cin, Cout/group, KH, KW], packed for the node's
        strides / top-left pads / dilations / group."""
        w = np.ascontiguousarray(w)
        if w.dtype == np.float64:
            w = w.astype(np.float32)
        h = ctypes.c_void_p()
        L.check(L.lib().ohip_weight_conv_transpose(self.h, _key(name, label), _np_ohip_dtype(w),
                                                   w.ctypes.data_as(ctypes.c_void_p), *w.shape, strides[0],
                                                   strides[1], pads[0], pads[1], dilations[0], dilations[1],
                                                   group, dtype, ctypes.byref(h)))
        return Weight(self, h, "convt", dtype, w.shape, name is not None)

    def weight_qgemm(self, b, zp=None, scale=None, trans_b=False, name=None, label="QLinearMatMul.B"):
        b = np.ascontiguousarray(b)
        k, n = (b.shape[1], b.shape[0]) if trans_b else b.shape
        zp_a = None if zp is None else np.ascontiguousarray(np.atleast_1d(np.asarray(zp, np.int32)))
        sc = None if scale is None else np.ascontiguousarray(np.atleast_1d(np.asarray(scale, np.float32)))
        h = ctypes.c_void_p()
        L.check(L.lib().ohip_weight_qgemm(
            self.h, _key(name, label), _np_ohip_dtype(b), b.ctypes.data_as(ctypes.c_void_p), k, n, int(trans_b),
            None if zp_a is None else zp_a.ctypes.data_as(ctypes.c_void_p), 0 if zp_a is None else zp_a.size,
            None if sc is None else sc.ctypes.data_as(ctypes.c_void_p), 0 if sc is None else sc.size,
            ctypes.byref(h)))
        return Weight(self, h, "qgemm", L.I8, (k, n), name is not None)

    def weight_qconv(self, w, zp=None, scale=None, name=None, label="QLinearConv.W"):
        w = np.ascontiguousarray(w)
        zp_a = None if zp is None else np.ascontiguousarray(np.atleast_1d(np.asarray(zp, np.int32)))
        sc = None if scale is None else np.ascontiguousarray(np.atleast_1d(np.asarray(scale, np.float32)))
        h = ctypes.c_void_p()
        L.check(L.lib().ohip_weight_qconv(
            self.h, _key(name, label), _np_ohip_dtype(w), w.ctypes.data_as(ctypes.c_void_p), *w.shape,
            None if zp_a is None else zp_a.ctypes.data_as(ctypes.c_void_p), 0 if zp_a is None else zp_a.size,
            None if sc is None else sc.ctypes.data_as(ctypes.c_void_p), 0 if sc is None else sc.size,
            ctypes.byref(h)))
        return Weight(self, h, "qconv", L.I8, w.shape, name is not None)

    def weight_q4(self, codes, scales, zero_points=None, k=None, dtype=None, name=None, label="Gemm.B4"):
        """A weight [K, N] of 4-bit codes (ohip_weight_q4): codes uint8 [N, blocks, group / 2], scales [N, blocks]
        (float32, float16, or bfloat16 as its 16 bits, rounded to `dtype`), zero_points uint8 [N, ceil(blocks / 2)]
        or None (8 everywhere); dtype: the activations' type (L.F32 / F16 / BF16 or "f32" / "f16" / "bf16"), by
        default the scales' own; k if K does not fill the last block."""
        codes, scales = np.ascontiguousarray(codes), np.asarray(scales)
        if codes.ndim != 3 or codes.dtype != np.uint8 or scales.shape != codes.shape[:2]:
            raise _invalid("weight_q4: codes uint8 [N, blocks, group / 2] and scales [N, blocks]")
        n, blocks, half = codes.shape
        k = blocks * 2 * half if k is None else k
        if not blocks or not half or (k + 2 * half - 1) // (2 * half) != blocks:
            raise _invalid("weight_q4: K does not end in the last block")
        bits = scales.dtype in (np.uint16, np.int16)   # numpy has no bfloat16
        if dtype is None:
            dtype = L.BF16 if bits else L.F16 if scales.dtype == np.float16 else L.F32
        dtype = _TYPE_NAMES.get(dtype, dtype)
        if dtype not in (L.F32, L.F16, L.BF16):
            raise _invalid("weight_q4: dtype")
        if bits and dtype != L.BF16:
            scales = (scales.view(np.uint16).astype(np.uint32) << 16).view(np.float32)
        if dtype == L.F32:
            scales = np.ascontiguousarray(scales, np.float32)
        elif dtype == L.F16:
            scales = np.ascontiguousarray(scales, np.float16)
        elif bits:
            scales = np.ascontiguousarray(scales)
        else:
            torch = _torch()
            scales = torch.from_numpy(np.array(scales, np.float32)).to(torch.bfloat16).view(torch.int16).numpy()
        if zero_points is not None:
            zero_points = np.ascontiguousarray(zero_points)
            if zero_points.dtype != np.uint8 or zero_points.shape != (n, (blocks + 1) // 2):
                raise _invalid("weight_q4: zero points uint8 [N, ceil(blocks / 2)]")
        h = ctypes.c_void_p()
        L.check(L.lib().ohip_weight_q4(self.h, _key(name, label), codes.ctypes.data, k, n, 2 * half, dtype,
                                       scales.ctypes.data, None if zero_points is None else zero_points.ctypes.data,
                                       ctypes.byref(h)))
        return Weight(self, h, "q4", dtype, (k, n), name is not None)

    # --------------------------------------------------------------- ops
    def gemm(self, a, w, c=None, alpha=1.0, beta=1.0, trans_a=False, act=L.ACT_NONE, act_lo=0.0, act_hi=0.0,
             out=None):
        dt = ohip_dtype(a.dtype)
        m = a.size(1) if trans_a else a.size(0)
        k, n = w.shape
        if out is None:
            out = _torch().empty((m, n), dtype=a.dtype, device=a.device)
        c_kind = L.C_NONE
        if c is not None:
            c_kind = L.C_SCALAR if c.numel() == 1 else (L.C_ROW if c.dim() == 1 else L.C_FULL)
        d = _GEMM(m, k, n, dt, int(trans_a), alpha, beta, c_kind, act, act_lo, act_hi, a.stride(0), out.stride(0))
        rc = L.raw("ohip_gemm")(self.h, d, a.data_ptr(), w.handle, _ptr(c), out.data_ptr())
        if rc:
            L.check(rc)
        return out

    def conv2d(self, x, w, bias=None, strides=(1, 1), pads=(0, 0, 0, 0), dilations=(1, 1), act=L.ACT_NONE,
               act_lo=0.0, act_hi=0.0, in_layout=L.NCHW, out_layout=L.NCHW, out=None, group=1, noalloc=False):
        """pads = [top, left, bottom, right]; x NCHW (or NHWC channel-padded);
        w holds Cin / group input channels per filter (ONNX Conv's group).
        noalloc=True calls ohip_conv2d_noalloc (static scratch, no device
        allocation; `out` should then be given)."""
        dt = ohip_dtype(x.dtype)
        cout, cin, kh, kw = w.shape
        if in_layout == L.NCHW:
            n, c, h, wd = x.shape
        else:
            n, h, wd = x.shape[:3]
            c = cin * group
        oh = _out_dim(h, pads[0], pads[2], kh, dilations[0], strides[0])
        ow = _out_dim(wd, pads[1], pads[3], kw, dilations[1], strides[1])
        if oh < 0 or ow < 0:
            raise L.OhipError(L.E_SHAPE, "bad conv geometry")
        if out is None:
            torch = _torch()
            if out_layout == L.NCHW:
                out = torch.empty((n, cout, oh, ow), dtype=x.dtype, device=x.device)
            else:
                ce = 16 // L.ELEM_BYTES[dt]
                out = torch.zeros((n, oh, ow, (cout + ce - 1) // ce * ce), dtype=x.dtype, device=x.device)
        d = _CONV(n, c, h, wd, cout, kh, kw, group, strides[0], strides[1], dilations[0], dilations[1],
                       pads[0], pads[1], pads[2], pads[3], dt, in_layout, out_layout, act, act_lo, act_hi, L.PAD_ZEROS)
        rc = L.raw("ohip_conv2d_noalloc" if noalloc else "ohip_conv2d")(self.h, d, x.data_ptr(), w.handle, _ptr(bias),
                                                                       out.data_ptr())
        if rc:
            L.check(rc)
        return out

    def conv2d_instnorm(self, x, w, bias=None, pads=(0, 0, 0, 0), strides=(1, 1), dilations=(1, 1), eps=1e-5,
                        gamma=None, beta=None, scale_offset=0, bias_offset=0, relu=False, out=None,
                        residual=None, nhwc=False):
        """Conv (ungrouped, no activation) followed by instance
        normalisation in one call (ohip_conv2d_instnorm); gamma / beta are
        optional [N, S] device rows of the tensor's dtype (the AdaIN form:
        channel c of sample n reads element n * S + offset + c); residual is
        added last.  nhwc: x, the output and the residual are NHWC (channels
        a whole number of 16-byte chunks), else NCHW."""
        torch = _torch()
        dt = ohip_dtype(x.dtype)
        cout, cin, kh, kw = w.shape
        if nhwc:
            n, h, wd, c = x.shape
        else:
            n, c, h, wd = x.shape
        oh = L.lib().ohip_conv_out_dim(h, pads[0], pads[2], kh, dilations[0], strides[0])
        ow = L.lib().ohip_conv_out_dim(wd, pads[1], pads[3], kw, dilations[1], strides[1])
        if out is None:
            shape = (n, oh, ow, cout) if nhwc else (n, cout, oh, ow)
            out = torch.empty(shape, dtype=x.dtype, device=x.device)
        lay = L.NHWC if nhwc else L.NCHW
        d = L.ConvDesc(n, c, h, wd, cout, kh, kw, 1, strides[0], strides[1], dilations[0], dilations[1],
                       pads[0], pads[1], pads[2], pads[3], dt, lay, lay, L.ACT_NONE, 0.0, 0.0, 0)
        nd = L.NormDesc(eps, None, None, 0, 0, 0, L.ACT_RELU if relu else L.ACT_NONE, 0.0,
                        None if residual is None else residual.data_ptr(), lay)
        if gamma is not None:
            eb = L.ELEM_BYTES[dt]
            nd.scale = gamma.data_ptr() + scale_offset * eb
            nd.bias = beta.data_ptr() + bias_offset * eb
            nd.per_sample, nd.stride, nd.same_type = 1, gamma.shape[1], 1
        L.check(L.lib().ohip_conv2d_instnorm(self.h, ctypes.byref(d), _ptr(x), w.handle, _ptr(bias),
                                             ctypes.byref(nd), _ptr(out)))
        return out

    def matmul(self, a, b, out=None):
        """Batched MatMul of two device tensors, [..., M, K] x [..., K, N], with the
        reference's slice rule (slice s: A slice s % a_batches, B slice s % b_batches)."""
        dt = ohip_dtype(a.dtype)
        sa, sb = tuple(a.shape), tuple(b.shape)
        m, k, n = sa[-2], sa[-1], sb[-1]
        na, nb = math.prod(sa[:-2]), math.prod(sb[:-2])
        batch_shape = sa[:-2] if sa[:-2] == sb[:-2] else np.broadcast_shapes(sa[:-2], sb[:-2])
        if out is None:
            out = _torch().empty(batch_shape + (m, n), dtype=a.dtype, device=a.device)
        d = _MATMUL(m, k, n, math.prod(batch_shape), na, nb, dt)
        a, b = a.contiguous(), b.contiguous()
        rc = L.raw("ohip_matmul")(self.h, d, a.data_ptr(), b.data_ptr(), out.data_ptr())
        if rc:
            L.check(rc)
        return out

    def conv_transpose2d(self, x, w, bias=None, strides=(1, 1), pads=(0, 0, 0, 0), dilations=(1, 1),
                         output_padding=(0, 0), group=1, out=None):
        """ConvTranspose, NCHW; pads = [top, left, bottom, right] (already resolved)."""
        dt = ohip_dtype(x.dtype)
        cin, coutg, kh, kw = w.shape
        n, c, h, wd = x.shape
        oh = L.lib().ohip_conv_transpose_out_dim(h, strides[0], output_padding[0], kh, dilations[0], pads[0], pads[2])
        ow = L.lib().ohip_conv_transpose_out_dim(wd, strides[1], output_padding[1], kw, dilations[1], pads[1], pads[3])
        if oh < 0 or ow < 0:
            raise L.OhipError(L.E_SHAPE, "bad ConvTranspose geometry")
        if out is None:
            out = _torch().empty((n, coutg * group, oh, ow), dtype=x.dtype, device=x.device)
        d = _CONVT(n, c, h, wd, coutg * group, kh, kw, group, strides[0], strides[1], dilations[0],
                        dilations[1], pads[0], pads[1], pads[2], pads[3], output_padding[0], output_padding[1], dt)
        rc = L.raw("ohip_conv_transpose2d")(self.h, d, x.data_ptr(), w.handle, _ptr(bias), out.data_ptr())
        if rc:
            L.check(rc)
        return out

    def qgemm(self, a, w, a_zp=0, out_kind=L.QOUT_U8, a_scale=1.0, y_scale=1.0, y_zp=0, lo=0, hi=255, out=None):
        m, k = a.shape
        n = w.shape[1]
        if type(a_zp) is int and -128 <= a_zp <= 255:
            azp_at, n_azp = _ZERO_POINTS_AT + 4 * (a_zp + 128), 1
        else:
            azp = np.ascontiguousarray(np.atleast_1d(np.asarray(a_zp, np.int32)))
            azp_at, n_azp = azp.ctypes.data, azp.size
        if out is None:
            torch = _torch()
            odt = {L.QOUT_U8: torch.uint8, L.QOUT_I8: torch.int8, L.QOUT_I32: torch.int32,
                   L.QOUT_F32: torch.float32}[out_kind]
            out = torch.empty((m, n), dtype=odt, device=a.device)
        d = _QGEMM(m, k, n, ohip_dtype(a.dtype), azp_at, n_azp, out_kind, a_scale, y_scale, y_zp, lo, hi,
                        a.stride(0), out.stride(0))
        rc = L.raw("ohip_qgemm")(self.h, d, a.data_ptr(), w.handle, out.data_ptr())
        if rc:
            L.check(rc)
        return out

    def qconv2d(self, x, w, bias=None, x_zp=0, out_kind=L.QOUT_U8, x_scale=1.0, y_scale=1.0, y_zp=0, lo=0,
                hi=255, strides=(1, 1), pads=(0, 0, 0, 0), dilations=(1, 1), in_layout=L.NCHW,
                out_layout=L.NCHW, out=None, group=1):
        torch = _torch()
        cout, cin, kh, kw = w.shape
        if in_layout == L.NCHW:
            n, c, h, wd = x.shape
        else:
            n, h, wd = x.shape[:3]
            c = cin * group
        oh = L.lib().ohip_conv_out_dim(h, pads[0], pads[2], kh, dilations[0], strides[0])
        ow = L.lib().ohip_conv_out_dim(wd, pads[1], pads[3], kw, dilations[1], strides[1])
        if oh < 0 or ow < 0:
            raise L.OhipError(L.E_SHAPE, "bad conv geometry")
        odt = {L.QOUT_U8: torch.uint8, L.QOUT_I8: torch.int8, L.QOUT_I32: torch.int32,
                   L.QOUT_F32: torch.float32}[out_kind]
        if out is None:
            if out_layout == L.NCHW:
                out = torch.empty((n, cout, oh, ow), dtype=odt, device=x.device)
            else:
                ld = (cout + 15) // 16 * 16 if out_kind in (L.QOUT_U8, L.QOUT_I8) else (cout + 3) // 4 * 4
                out = torch.zeros((n, oh, ow, ld), dtype=odt, device=x.device)
        d = L.QConvDesc(n, c, h, wd, cout, kh, kw, group, strides[0], strides[1], dilations[0], dilations[1],
                        pads[0], pads[1], pads[2], pads[3], ohip_dtype(x.dtype), int(x_zp), out_kind, x_scale,
                        y_scale, y_zp, lo, hi, in_layout, out_layout)
        L.check(L.lib().ohip_qconv2d(self.h, ctypes.byref(d), _ptr(x), w.handle, _ptr(bias), _ptr(out)))
        return out

    # --------------------------------------------------------------- serving
    def gemm_q4(self, a, w, bias=None, act=L.ACT_NONE, act_lo=0.0, act_hi=0.0, out=None):
        """act(a @ w + bias) of a [M, K] and a weight of weight_q4 (ohip_gemm_q4); bias [N] of a's type."""
        m, k = a.shape
        n = w.shape[1]
        if out is None:
            out = _torch().empty((m, n), dtype=a.dtype, device=a.device)
        at = self.device
        if (a.get_device() != at or out.get_device() != at or out.dtype != a.dtype or out.shape != (m, n)
                or (k > 1 and a.stride(1) != 1) or (n > 1 and out.stride(1) != 1)):
            raise _invalid("gemm_q4: a [M, K] and out [M, N] of one type on the context's GPU, rows contiguous")
        if m > 1 and (a.stride(0) < k or out.stride(0) < n):   # (a stride of 0 is the library's "packed")
            raise _invalid("gemm_q4: rows share memory")
        if bias is not None and (bias.dtype != a.dtype or bias.get_device() != at or not bias.is_contiguous()
                                 or bias.numel() != n):
            raise _invalid("gemm_q4: bias [N] of the activations' type")
        d = _GEMM_Q4(m, k, n, ohip_dtype(a.dtype), act, act_lo, act_hi, a.stride(0) if m > 1 else k,
                     out.stride(0) if m > 1 else n)
        rc = L.raw("ohip_gemm_q4")(self.h, d, a.data_ptr(), w.handle, _ptr(bias), out.data_ptr())
        if rc:
            L.check(rc)
        return out

    def kv_cache(self, pages, page, kv_heads, head_dim, group=64):
        """An empty KvCache on this context's GPU."""
        return KvCache.empty(pages, page, kv_heads, head_dim, group, self.device)

    def kv_append(self, cache, k, v, slots, q=None, positions=None, cos=None, sin=None, interleaved=False,
                  out_held=True, q_out=None, k_out=None, v_out=None):
        """Appends keys and values [tokens, kv_heads, dim] at `slots` (int32, page * page size + place; negative:
        not written), keys and queries rotated by rows `positions` (int32) of cos / sin (float32 [positions,
        rot / 2]); see ohip_kv_append.  Returns (q_out, k_out, v_out): the rotated queries, and keys and values
        as the cache holds them (out_held) or as they went in; k_out / v_out False: not wanted."""
        at, dt = self.device, k.dtype
        shape = k.shape
        if len(shape) != 3 or v.shape != shape or shape[1] != cache.kv_heads or shape[2] != cache.dim or cache.device != at:
            raise _invalid("kv_append: keys and values [tokens, kv_heads, dim] of the cache")
        tokens, kv, dim = shape
        ldk, ldv = _heads(k, "kv_append: k", dt, at), _heads(v, "kv_append: v", dt, at)
        heads = ldq = ldqo = ldko = ldvo = rot = rows = 0
        qp = qop = kop = vop = pos = cs = sn = None
        if q is not None:
            qshape = q.shape
            if len(qshape) != 3 or qshape[0] != tokens or qshape[2] != dim:
                raise _invalid("kv_append: q [tokens, heads, dim]")
            heads, ldq = qshape[1], _heads(q, "kv_append: q", dt, at)
            if q_out is None:
                q_out = _torch().empty(qshape, dtype=dt, device=q.device)
            elif q_out.shape != qshape:
                raise _invalid("kv_append: q_out has another shape than q")
            ldqo, qp, qop = _heads(q_out, "kv_append: q_out", dt, at), q.data_ptr(), q_out.data_ptr()
        elif q_out is not None:
            raise _invalid("kv_append: q_out without q")
        if k_out is None:
            k_out = _torch().empty(shape, dtype=dt, device=k.device)
        if k_out is not False:
            if k_out.shape != shape:
                raise _invalid("kv_append: k_out has another shape than k")
            ldko, kop = _heads(k_out, "kv_append: k_out", dt, at), k_out.data_ptr()
        if v_out is None:
            v_out = _torch().empty(shape, dtype=dt, device=k.device)
        if v_out is not False:
            if v_out.shape != shape:
                raise _invalid("kv_append: v_out has another shape than k")
            ldvo, vop = _heads(v_out, "kv_append: v_out", dt, at), v_out.data_ptr()
        i32 = _TORCH_DT[L.I32]
        if (cos is None) != (sin is None) or (cos is not None and positions is None):
            raise _invalid("kv_append: cos, sin and positions come together")
        if cos is not None:
            f32, angles = _TORCH_DT[L.F32], cos.shape
            if len(angles) != 2:
                raise _invalid("kv_append: cos [positions, rot / 2]")
            rows, rot = angles[0], 2 * angles[1]
            cs, sn = _table(cos, "kv_append: cos", f32, at, angles), _table(sin, "kv_append: sin", f32, at, angles)
            pos = _table(positions, "kv_append: positions", i32, at, (tokens,))
        d = _KV_APPEND(tokens, ohip_dtype(dt), heads, rot, interleaved, out_held, rows, ldq, ldk, ldv, ldqo, ldko, ldvo)
        rc = L.raw("ohip_kv_append")(self.h, d, cache.desc, qp, k.data_ptr(), v.data_ptr(), pos, cs, sn,
                                     _table(slots, "kv_append: slots", i32, at, (tokens,)), qop, kop, vop)
        if rc:
            L.check(rc)
        return q_out, (None if k_out is False else k_out), (None if v_out is False else v_out)

    def attn_decode(self, q, cache, table, lens, scale=None, window=0, out=None):
        """Attention of one query token a sequence [batch, heads, dim] over the first lens[b] (int32) tokens of
        the pages table[b] (int32 [batch, entries]) of `cache`, at most the last `window` of them (0: all);
        scale: 1 / sqrt(dim) by default (ohip_attn_decode)."""
        at, dt = self.device, q.dtype
        ldq = _heads(q, "attn_decode: q", dt, at)
        batch, heads, dim = q.shape
        if dim != cache.dim or cache.device != at:
            raise _invalid("attn_decode: q [batch, heads, dim] of the cache")
        if out is None:
            out = _torch().empty(q.shape, dtype=dt, device=q.device)
        elif out.shape != q.shape:
            raise _invalid("attn_decode: out has another shape than q")
        i32 = _TORCH_DT[L.I32]
        width = table.shape[-1]
        d = _ATTN_DECODE(batch, ohip_dtype(dt), heads, width, window, dim ** -0.5 if scale is None else scale, ldq,
                         _heads(out, "attn_decode: out", dt, at))
        rc = L.raw("ohip_attn_decode")(self.h, d, cache.desc, q.data_ptr(),
                                       _table(table, "attn_decode: table", i32, at, (batch, width)),
                                       _table(lens, "attn_decode: lens", i32, at, (batch,)), out.data_ptr())
        if rc:
            L.check(rc)
        return out

    def attn_prefill(self, q, k, v, cu_q, cu_k=None, scale=None, causal=True, window=0, out=None):
        """Attention over packed sequences: q [tokens, heads, dim], k and v [key tokens, kv_heads, dim], int32
        offsets cu_q (and cu_k, by default the same) of sequences + 1 entries; see ohip_attn_prefill."""
        at, dt = self.device, q.dtype
        ldq, ldk, ldv = (_heads(t, n, dt, at) for t, n in ((q, "attn_prefill: q"), (k, "attn_prefill: k"),
                                                           (v, "attn_prefill: v")))
        (tokens, heads, dim), (keys, kv, kdim) = q.shape, k.shape
        if v.shape != k.shape or kdim != dim:
            raise _invalid("attn_prefill: k and v [key tokens, kv_heads, dim], dim as q")
        if out is None:
            out = _torch().empty(q.shape, dtype=dt, device=q.device)
        elif out.shape != q.shape:
            raise _invalid("attn_prefill: out has another shape than q")
        cu_k = cu_q if cu_k is None else cu_k
        i32, seqs = _TORCH_DT[L.I32], cu_q.shape[0] - 1
        if seqs < 0:
            raise _invalid("attn_prefill: cu_q needs an entry")
        d = _ATTN_PREFILL(tokens, keys, seqs, ohip_dtype(dt), heads, kv, dim, int(causal), window,
                          dim ** -0.5 if scale is None else scale, ldq, ldk, ldv,
                          _heads(out, "attn_prefill: out", dt, at))
        rc = L.raw("ohip_attn_prefill")(self.h, d, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                        _table(cu_q, "attn_prefill: cu_q", i32, at, (seqs + 1,)),
                                        _table(cu_k, "attn_prefill: cu_k", i32, at, (seqs + 1,)), out.data_ptr())
        if rc:
            L.check(rc)
        return out
