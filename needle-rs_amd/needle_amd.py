"""Python mirror of needle-rs's hot-path operator interface over the C ABI
(include/needle_amd.h), for callers that hold torch device tensors.

Names follow the reference: CqWeight.{prepare_input, matvec_rows_prepared,
matmul_rows_prepared, dequantize_row} (crates/needle-core/src/cq.rs),
fake_quant_vec / quantize_rows / V3Cache.write_kv / span
(v3/cache.rs), attend_step / attend (v3/attention.rs).  Every call goes
through libneedle_amd.so; there is no CPU fallback -- a missing library or
GPU raises.  torch supplies device memory and the stream only.
"""
from __future__ import annotations

import ctypes as C
import math
import os
import re

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libneedle_amd.so")
HEADER = os.path.join(os.path.dirname(HERE), "include", "needle_amd.h")

ND_OK = 0
ND_ERR_ARG, ND_ERR_CACT, ND_ERR_V3_GEOMETRY, ND_ERR_V3_LAYOUT = 1, 20, 21, 22
ERRORS = {1: "ND_ERR_ARG", 2: "ND_ERR_HIP", 3: "ND_ERR_NOMEM", 4: "ND_ERR_BUSY", 11: "UnsupportedBits",
          12: "BadGroup", 13: "BadCodebookLen", 14: "ShortBlob", 15: "EmptyShape",
          20: "CactError", 21: "V3GeometryError", 22: "V3LayoutError"}


class NeedleError(RuntimeError):
    def __init__(self, code, msg):
        super().__init__(f"{ERRORS.get(code, code)}: {msg}")
        self.code = code


class KvGeom(C.Structure):
    _fields_ = [("num_heads", C.c_int32), ("num_kv_heads", C.c_int32),
                ("qk_head_dim", C.c_int32), ("v_head_dim", C.c_int32), ("cap", C.c_int32)]


class Rope(C.Structure):
    _fields_ = [("layout", C.c_int32), ("scaling", C.c_int32), ("rot_dim", C.c_int32),
                ("theta", C.c_double), ("factor", C.c_double), ("trained", C.c_double),
                ("turns_lo", C.c_double), ("turns_hi", C.c_double), ("gain", C.c_double)]


class LogitsRules(C.Structure):
    _fields_ = [("hist", C.c_void_p), ("hist_stride", C.c_size_t), ("hist_len", C.c_void_p),
                ("out_from", C.c_void_p), ("repeat", C.c_void_p), ("frequency", C.c_void_p),
                ("presence", C.c_void_p), ("bias_id", C.c_void_p), ("bias", C.c_void_p),
                ("bias_stride", C.c_size_t), ("bias_len", C.c_void_p), ("mask", C.c_void_p),
                ("mask_stride", C.c_size_t), ("mask_rows", C.c_size_t), ("mask_row", C.c_void_p)]


_lib = None
_vp, _sz = C.c_void_p, C.c_size_t

# (name, restype, argtypes) for every entry point of include/needle_amd.h.
_SIGS = [
    ("nd_last_error", C.c_char_p, []),
    ("nd_ctx_create", C.c_int, [C.c_int, C.POINTER(_vp)]),
    ("nd_ctx_create_on_stream", C.c_int, [C.c_int, _vp, C.POINTER(_vp)]),
    ("nd_ctx_destroy", None, [_vp]),
    ("nd_ctx_synchronize", C.c_int, [_vp]),
    ("nd_malloc", C.c_int, [_vp, _sz, C.POINTER(_vp)]),
    ("nd_free", C.c_int, [_vp, _vp]),
    ("nd_memcpy_htod", C.c_int, [_vp, _vp, _vp, _sz]),
    ("nd_memcpy_dtoh", C.c_int, [_vp, _vp, _vp, _sz]),
    ("nd_cb8_gemv", C.c_int, [_vp, _vp, _vp, _vp, _vp, _sz, _sz]),
    ("nd_cb8_gemv_batched", C.c_int, [_vp, _sz, _vp, _sz, _vp, _sz, _vp, _sz, _vp, _sz, _sz, _sz]),
    ("nd_cb8_gemm", C.c_int, [_vp, _vp, _vp, _vp, _vp, _sz, _sz, _sz]),
    ("nd_cb8_gemm_batched", C.c_int, [_vp, _sz, _vp, _sz, _vp, _sz, _vp, _sz, _vp, _sz, _sz, _sz, _sz]),
    ("nd_cq_from_blob", C.c_int, [_vp, _vp, _sz, _sz, _sz, _sz, C.c_uint8, _vp, _sz, C.POINTER(_vp)]),
    ("nd_cq_free", None, [_vp]),
    ("nd_cq_shape", C.c_int, [_vp, C.POINTER(_sz), C.POINTER(_sz), C.POINTER(_sz), C.POINTER(_sz),
                              C.POINTER(C.c_uint8)]),
    ("nd_cq_prepare_input", C.c_int, [_vp, _vp, _vp, _sz, _vp]),
    ("nd_cq_matvec_rows_prepared", C.c_int, [_vp, _vp, _vp, _sz, _sz, _vp]),
    ("nd_cq_matmul_rows_prepared", C.c_int, [_vp, _vp, _vp, _sz, _sz, _sz, _vp]),
    ("nd_cq_matvec_rows_exact", C.c_int, [_vp, _vp, _vp, _sz, _sz, _vp]),
    ("nd_cq_matmul_rows_exact", C.c_int, [_vp, _vp, _vp, _sz, _sz, _sz, _vp]),
    ("nd_cq_dequantize_rows", C.c_int, [_vp, _vp, _vp, _sz, _vp]),
    ("nd_fold_rows", C.c_int, [_vp, _vp, _sz, _sz, _vp]),
    ("nd_fake_quant", C.c_int, [_vp, _vp, _sz, _sz]),
    ("nd_quantize_rows", C.c_int, [_vp, _vp, _sz, _sz, _vp, _vp]),
    ("nd_kv_block_bytes", _sz, [C.POINTER(KvGeom)]),
    ("nd_kv_v_offset", _sz, [C.POINTER(KvGeom)]),
    ("nd_kv_ks_offset", _sz, [C.POINTER(KvGeom)]),
    ("nd_kv_vs_offset", _sz, [C.POINTER(KvGeom)]),
    ("nd_kv_write", C.c_int, [_vp, C.POINTER(KvGeom), _vp, _sz, _sz, _vp, _vp, _vp]),
    ("nd_attend_step_i8", C.c_int, [_vp, C.POINTER(KvGeom), _vp, _sz, _sz, _vp, _vp, _vp,
                                    C.c_float, C.c_int, _vp]),
    ("nd_attend_step_i8_exact", C.c_int, [_vp, C.POINTER(KvGeom), _vp, _sz, _sz, _vp, _vp, _vp,
                                          C.c_float, C.c_int, _vp]),
    ("nd_attend_step_i8_noalloc", C.c_int, [_vp, C.POINTER(KvGeom), _vp, _sz, _sz, _vp, _vp, _vp,
                                            C.c_float, C.c_int, _vp]),
    ("nd_v3_model_create", C.c_int, [_vp, _vp, _vp, _sz, _vp, _sz, C.POINTER(_vp)]),
    ("nd_v3_model_free", None, [_vp]),
    ("nd_v3_logit_rows", _sz, [_vp]),
    ("nd_v3_batch_create", C.c_int, [_vp, _vp, _sz, _sz, _sz, C.POINTER(_vp)]),
    ("nd_v3_batch_free", None, [_vp]),
    ("nd_v3_positions", C.c_int, [_vp, _vp]),
    ("nd_v3_step", C.c_int, [_vp, _vp, _vp, _vp, _vp, _vp]),
    ("nd_argmax_rows", C.c_int, [_vp, _vp, _sz, _sz, _vp]),
    ("nd_v3_batch_create_chunked", C.c_int, [_vp, _vp, _sz, _sz, _sz, _sz, C.POINTER(_vp)]),
    ("nd_v3_prefill", C.c_int, [_vp, _vp, _vp, _vp, _sz, _vp, _vp]),
    ("nd_v3_generate", C.c_int, [_vp, _vp, _vp, _vp, _sz, _vp]),
    ("nd_v3_generate_many", C.c_int, [_vp, _vp, _vp, _sz, _vp, _sz, _vp]),
    ("nd_v3_cact_config", C.c_int, [_vp, _sz, _vp, C.POINTER(_sz)]),
    ("nd_v3_model_from_cact", C.c_int, [_vp, _vp, _sz, C.POINTER(_vp)]),
    ("nd_v3_batch_set_graphs", C.c_int, [_vp, C.c_int]),
    ("nd_v3_kv_bytes", _sz, [_vp, _sz, C.c_int]),
    ("nd_v3_ladder", C.c_int, [_sz, _sz, C.POINTER(C.c_int32)]),
    ("nd_v3_cact_config_at_depth", C.c_int, [_vp, _sz, _sz, _vp, C.POINTER(C.c_int32)]),
    ("nd_v3_model_from_cact_at_depth", C.c_int, [_vp, _vp, _sz, _sz, C.POINTER(_vp)]),
    ("nd_kv_f32_block_bytes", _sz, [C.POINTER(KvGeom)]),
    ("nd_kv_f32_v_offset", _sz, [C.POINTER(KvGeom)]),
    ("nd_kv_write_f32", C.c_int, [_vp, C.POINTER(KvGeom), _vp, _sz, _sz, _vp, _vp, _vp]),
    ("nd_attend_step_f32_exact", C.c_int, [_vp, C.POINTER(KvGeom), _vp, _sz, _sz, _vp, _vp, _vp,
                                           C.c_float, _vp]),
    ("nd_v3_batch_create_ex", C.c_int, [_vp, _vp, _sz, _sz, _sz, _sz, C.c_int, C.POINTER(_vp)]),
    ("nd_libm_map", C.c_int, [_vp, C.c_int, _vp, _sz, _vp]),
    ("nd_rope_freqs", C.c_int, [C.POINTER(Rope), C.POINTER(C.c_double)]),
    ("nd_rope_rows", C.c_int, [_vp, C.POINTER(Rope), _sz, _vp, _sz, _sz, _vp, _sz, _vp, _sz]),
    ("nd_kv_write_rope", C.c_int, [_vp, C.POINTER(KvGeom), C.POINTER(Rope), _vp, _sz, _sz, _sz, _vp,
                                   _vp, _vp, _sz, _vp, _sz, _vp, _sz, _vp, _sz]),
    ("nd_kv_read", C.c_int, [_vp, C.POINTER(KvGeom), _vp, _sz, _sz, _sz, _vp, _vp, _vp]),
    ("nd_attend_tree_i8_work", _sz, [_vp, C.POINTER(KvGeom), _sz, _sz]),
    ("nd_attend_tree_i8", C.c_int, [_vp, C.POINTER(KvGeom), _vp, _sz, _sz, _sz, _vp, _vp, _vp, _vp, _vp,
                                    C.c_float, C.c_int, _vp, _vp, _sz]),
    ("nd_logits_adjust_work", _sz, [_vp, _sz, _sz]),
    ("nd_logits_adjust", C.c_int, [_vp, _vp, _sz, _sz, _sz, C.POINTER(LogitsRules), _vp, _sz, _vp, _vp,
                                   _sz]),
]


def header_symbols():
    """Function names declared in include/needle_amd.h."""
    text = open(HEADER).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(nd_[a-z0-9_]+)\s*\(", text)))


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is not built: run `make -C needle-rs_amd` "
                               "(or __graft_entry__.build()); there is no CPU fallback")
        L = C.CDLL(LIB_PATH)
        for name, res, args in _SIGS:
            f = getattr(L, name)
            f.restype = res
            f.argtypes = args
        _lib = L
    return _lib


def last_error():
    m = lib().nd_last_error()
    return m.decode() if m else None


def _check(rc):
    if rc != ND_OK:
        raise NeedleError(rc, last_error())


def _ptr(t):
    return C.c_void_p(t.data_ptr()) if t is not None else C.c_void_p(0)


def _arg(t, dtype, name, numel=0, rows=False):
    """The device pointer of tensor `t` once it is a device tensor of `dtype`
    holding at least `numel` elements, contiguous (with rows=True: each
    slice t[i] contiguous, for the strided batched calls).  The library
    reads exactly the bytes its sizes imply, so a wrong dtype or layout
    would read past the buffer or in the wrong order: raise instead."""
    if not t.is_cuda:
        raise ValueError(f"{name}: a device tensor is required")
    if t.dtype != dtype:
        raise ValueError(f"{name}: dtype {t.dtype}, expected {dtype}")
    # A contiguous tensor of two slices or more has contiguous slices that do
    # not overlap (one slice: by its stride); a slice itself (1 us to form) is
    # looked at only where that does not settle it.
    if not (t.is_contiguous() and (not rows or t.dim() < 2 or t.size(0) > 1 or
                                   (t.size(0) == 1 and t.stride(0) >= t.numel()))):
        ok = (t.dim() == 0 or all(t[i].is_contiguous() for i in range(min(t.shape[0], 1)))) \
            if rows else t.is_contiguous()
        if rows and t.dim() > 1:
            ok = ok and t.stride(0) >= t[0].numel()
        if not ok:
            raise ValueError(f"{name}: layout {tuple(t.shape)} strides {t.stride()} is not contiguous")
    if numel and t.numel() < numel:
        raise ValueError(f"{name}: {t.numel()} elements, at least {numel} needed")
    return t.data_ptr()


_torch_module = None


def _torch():
    """torch, once it has been seen to have a GPU (0.6 us a call to ask)."""
    global _torch_module
    if _torch_module is None:
        import torch
        if not torch.cuda.is_available():
            raise RuntimeError("no GPU visible: the HIP path has no CPU fallback")
        _torch_module = torch
    return _torch_module


class Ctx:
    """nd_ctx bound to a device and to torch's current stream on it."""

    def __init__(self, device=0, stream=None):
        torch = _torch()
        self.device = device
        if stream is None:
            stream = torch.cuda.current_stream(device)
        self.stream = stream
        h = C.c_void_p()
        _check(lib().nd_ctx_create_on_stream(device, C.c_void_p(stream.cuda_stream), C.byref(h)))
        self.h = h

    def synchronize(self):
        _check(lib().nd_ctx_synchronize(self.h))

    def close(self):
        if getattr(self, "h", None) and _lib is not None:
            _lib.nd_ctx_destroy(self.h)
            self.h = None

    __del__ = close


# ---- Format B ---------------------------------------------------------------

def cb8_gemv(ctx, w, cb, x, y=None):
    torch = _torch()
    out, inn = w.shape
    if y is None:
        y = torch.empty(out, dtype=torch.float32, device=w.device)
    f32 = torch.float32
    _check(lib().nd_cb8_gemv(ctx.h, _arg(w, torch.uint8, "w"),
                             _arg(cb, f32, "cb", (out + 63) // 64 * 256), _arg(x, f32, "x", inn),
                             _arg(y, f32, "y", out), out, inn))
    return y


def cb8_gemv_batched(ctx, w, cb, x, y):
    """w [count, out, in] u8, cb [count, out/64, 256], x [count, in], y [count, out]."""
    torch = _torch()
    count, out, inn = w.shape
    f32 = torch.float32
    _check(lib().nd_cb8_gemv_batched(
        ctx.h, count, _arg(w, torch.uint8, "w", rows=True), w.stride(0),
        _arg(cb, f32, "cb", rows=True), cb.stride(0), _arg(x, f32, "x", rows=True), x.stride(0),
        _arg(y, f32, "y", rows=True), y.stride(0), out, inn))
    return y


def cb8_gemm(ctx, x, w, cb, y=None):
    torch = _torch()
    m, inn = x.shape
    out = w.shape[0]
    if y is None:
        y = torch.empty(m, out, dtype=torch.float32, device=x.device)
    f32 = torch.float32
    _check(lib().nd_cb8_gemm(ctx.h, _arg(x, f32, "x"), _arg(w, torch.uint8, "w", out * inn),
                             _arg(cb, f32, "cb", (out + 63) // 64 * 256), _arg(y, f32, "y", m * out),
                             m, out, inn))
    return y


def cb8_gemm_batched(ctx, x, w, cb, y):
    """x [count][m][in] f32, w [count][out][in] u8, cb [count][out/64][256],
    y [count][m][out]: one launch."""
    torch = _torch()
    count, m, inn = x.shape
    out = w.shape[1]
    f32 = torch.float32
    _check(lib().nd_cb8_gemm_batched(
        ctx.h, count, _arg(x, f32, "x", rows=True), x.stride(0),
        _arg(w, torch.uint8, "w", rows=True), w.stride(0), _arg(cb, f32, "cb", rows=True),
        cb.stride(0), _arg(y, f32, "y", rows=True), y.stride(0), m, out, inn))
    return y


# ---- Format A ---------------------------------------------------------------

class CqWeight:
    """Device CqWeight (cq.rs:117-810) built from a host blob."""

    def __init__(self, ctx, blob, out_feat, in_feat, group, bits, codebook):
        self.ctx = ctx
        blob = np.ascontiguousarray(blob, np.uint8)
        cb = np.ascontiguousarray(codebook, np.float32)
        h = C.c_void_p()
        _check(lib().nd_cq_from_blob(ctx.h, blob.ctypes.data_as(C.c_void_p), blob.size, out_feat,
                                     in_feat, group, bits, cb.ctypes.data_as(C.c_void_p), cb.size,
                                     C.byref(h)))
        self.h = h
        o, i, p, g, b = _sz(), _sz(), _sz(), _sz(), C.c_uint8()
        _check(lib().nd_cq_shape(h, C.byref(o), C.byref(i), C.byref(p), C.byref(g), C.byref(b)))
        self.out_feat, self.in_feat, self.in_padded = o.value, i.value, p.value
        self.group, self.bits = g.value, b.value

    def close(self):
        if getattr(self, "h", None) and _lib is not None:
            _lib.nd_cq_free(self.h)
            self.h = None

    __del__ = close

    def prepare_input(self, x, xh=None):
        torch = _torch()
        x2 = x if x.dim() == 2 and x.size(1) == self.in_feat else x.reshape(-1, self.in_feat)
        if xh is None:
            xh = torch.empty(x2.shape[0], self.in_padded, dtype=torch.float32, device=x.device)
        n = x2.shape[0]
        _check(lib().nd_cq_prepare_input(self.ctx.h, self.h, _arg(x2, torch.float32, "x"), n,
                                         _arg(xh, torch.float32, "xh", n * self.in_padded)))
        return xh

    def matvec_rows_prepared(self, xh, row_start, rows, y=None, exact=False):
        """exact=True: the reference's summation order, bit-identical."""
        torch = _torch()
        if y is None:
            y = torch.empty(rows, dtype=torch.float32, device=xh.device)
        fn = lib().nd_cq_matvec_rows_exact if exact else lib().nd_cq_matvec_rows_prepared
        _check(fn(self.ctx.h, self.h, _arg(xh, torch.float32, "xh", self.in_padded), row_start,
                  rows, _arg(y, torch.float32, "y", rows)))
        return y

    def matvec_prepared(self, xh, y=None):
        return self.matvec_rows_prepared(xh, 0, self.out_feat, y)

    def matvec(self, x):
        return self.matvec_prepared(self.prepare_input(x))

    def matmul_rows_prepared(self, xh, batch, row_start, rows, y=None, exact=False):
        """exact=True: the reference's summation order, bit-identical."""
        torch = _torch()
        if y is None:
            y = torch.empty(batch * rows, dtype=torch.float32, device=xh.device)
        fn = lib().nd_cq_matmul_rows_exact if exact else lib().nd_cq_matmul_rows_prepared
        _check(fn(self.ctx.h, self.h, _arg(xh, torch.float32, "xh", batch * self.in_padded),
                  batch, row_start, rows, _arg(y, torch.float32, "y", batch * rows)))
        return y

    def dequantize_rows(self, rows_i32, out=None):
        torch = _torch()
        n = rows_i32.numel()
        if out is None:
            out = torch.empty(n, self.in_feat, dtype=torch.float32, device=rows_i32.device)
        _check(lib().nd_cq_dequantize_rows(self.ctx.h, self.h, _arg(rows_i32, torch.int32, "rows"),
                                           n, _arg(out, torch.float32, "out", n * self.in_feat)))
        return out


# ---- int8 KV ----------------------------------------------------------------

def fold_rows(ctx, x, y=None):
    """y[r] = the sequential fp32 sum of row r of x ([rows][n], n <= 4096),
    in the reference's order (kernels.rs:22-24, v3/attention.rs:361-365)."""
    torch = _torch()
    rows, n = x.shape
    if y is None:
        y = torch.empty(rows, dtype=torch.float32, device=x.device)
    _check(lib().nd_fold_rows(ctx.h, _arg(x, torch.float32, "x"), rows, n,
                              _arg(y, torch.float32, "y", rows)))
    return y


def argmax_rows(ctx, x, out=None):
    """The greedy token of each row of x ([count][n] fp32): the first maximum
    (needle-infer/src/v3_engine.rs:410-420)."""
    torch = _torch()
    count, n = x.shape
    if out is None:
        out = torch.empty(count, dtype=torch.int32, device=x.device)
    _check(lib().nd_argmax_rows(ctx.h, _arg(x, torch.float32, "x"), count, n,
                                _arg(out, torch.int32, "out", count)))
    return out


LIBM = {"expf": 0, "logf": 1, "sigmoid": 2}


def libm_map(ctx, fn, x, y=None):
    """The device copy of the reference's libm wrapper `fn` ("expf", "logf",
    "sigmoid"; math.rs:3-46) applied to every element of x (fp32)."""
    torch = _torch()
    if y is None:
        y = torch.empty_like(x)
    n = x.numel()
    _check(lib().nd_libm_map(ctx.h, LIBM[fn], _arg(x, torch.float32, "x"), n,
                             _arg(y, torch.float32, "y", n)))
    return y


def fake_quant(ctx, x, dim):
    """fake_quant_vec(x[r], 8) for every row of `dim`, in place."""
    torch = _torch()
    _check(lib().nd_fake_quant(ctx.h, _arg(x, torch.float32, "x"), x.numel() // dim, dim))
    return x


def quantize_rows(ctx, x, head_dim):
    torch = _torch()
    rows = x.numel() // head_dim
    ints = torch.empty(rows * head_dim, dtype=torch.int8, device=x.device)
    scales = torch.empty(rows, dtype=torch.float32, device=x.device)
    _check(lib().nd_quantize_rows(ctx.h, _arg(x, torch.float32, "x"), rows, head_dim, _ptr(ints),
                                  _ptr(scales)))
    return ints, scales


def kv_geom(num_heads, num_kv_heads, qk, vd, cap):
    return KvGeom(num_heads, num_kv_heads, qk, vd, cap)


def kv_block_bytes(g):
    return lib().nd_kv_block_bytes(C.byref(g))


def kv_offsets(g):
    L = lib()
    return dict(v=L.nd_kv_v_offset(C.byref(g)), ks=L.nd_kv_ks_offset(C.byref(g)),
                vs=L.nd_kv_vs_offset(C.byref(g)), total=L.nd_kv_block_bytes(C.byref(g)))


def kv_alloc(g, count=1, device=0):
    """`count` zeroed KV blocks, one after another (stride = block bytes)."""
    torch = _torch()
    nb = kv_block_bytes(g)
    return torch.zeros(count * nb, dtype=torch.uint8, device=device), nb


def kv_write(ctx, g, kv, kv_stride, pos_i32, k, v):
    torch = _torch()
    n = pos_i32.numel()
    blocks = kv_block_bytes(g) + (n - 1) * kv_stride if n else 0
    _check(lib().nd_kv_write(
        ctx.h, C.byref(g), _arg(kv, torch.uint8, "kv", blocks), kv_stride, n,
        _arg(pos_i32, torch.int32, "pos"),
        _arg(k, torch.float32, "k", n * g.num_kv_heads * g.qk_head_dim),
        _arg(v, torch.float32, "v", n * g.num_kv_heads * g.v_head_dim)))


def attend_step_i8(ctx, g, kv, kv_stride, lo_i32, hi_i32, q, scale=None, quant_query=False,
                   out=None, exact=False, noalloc=False):
    """exact=True: nd_attend_step_i8_exact, bit-identical to attend_step.
    noalloc=True: nd_attend_step_i8_noalloc (no device allocation; split-K
    partials in the library's fixed per-GPU array)."""
    torch = _torch()
    count = lo_i32.numel()
    if scale is None:
        scale = float(np.float32(1.0) / np.sqrt(np.float32(g.qk_head_dim)))
    if out is None:
        out = torch.empty(count, g.num_heads * g.v_head_dim, dtype=torch.float32, device=q.device)
    fn = lib().nd_attend_step_i8_exact if exact else lib().nd_attend_step_i8
    if noalloc:
        if exact:
            raise ValueError("the no-allocation entry point is the tolerance-order kernel")
        fn = lib().nd_attend_step_i8_noalloc
    blocks = kv_block_bytes(g) + (count - 1) * kv_stride if count else 0
    i32, f32 = torch.int32, torch.float32
    _check(fn(ctx.h, C.byref(g), _arg(kv, torch.uint8, "kv", blocks), kv_stride, count,
              _arg(lo_i32, i32, "lo"), _arg(hi_i32, i32, "hi", count),
              _arg(q, f32, "q", count * g.num_heads * g.qk_head_dim), scale,
              int(bool(quant_query)), _arg(out, f32, "out", count * g.num_heads * g.v_head_dim)))
    return out


# ---- f32 KV (KvPrecision::F32) ----------------------------------------------

def kv_f32_block_bytes(g):
    return lib().nd_kv_f32_block_bytes(C.byref(g))


def kv_alloc_f32(g, count=1, device=0):
    """`count` zeroed f32 KV blocks, one after another (stride = block bytes)."""
    torch = _torch()
    nb = kv_f32_block_bytes(g)
    return torch.zeros(count * nb, dtype=torch.uint8, device=device), nb


def kv_write_f32(ctx, g, kv, kv_stride, pos_i32, k, v):
    """V3Cache::write_kv with KvPrecision::F32 (cache.rs:359-362)."""
    torch = _torch()
    n = pos_i32.numel()
    blocks = kv_f32_block_bytes(g) + (n - 1) * kv_stride if n else 0
    _check(lib().nd_kv_write_f32(
        ctx.h, C.byref(g), _arg(kv, torch.uint8, "kv", blocks), kv_stride, n,
        _arg(pos_i32, torch.int32, "pos"),
        _arg(k, torch.float32, "k", n * g.num_kv_heads * g.qk_head_dim),
        _arg(v, torch.float32, "v", n * g.num_kv_heads * g.v_head_dim)))


def attend_step_f32(ctx, g, kv, kv_stride, lo_i32, hi_i32, q, scale=None, out=None):
    """attend_step over KvStore::F32 (attention.rs:166-189, 327-377),
    bit-identical (nd_attend_step_f32_exact)."""
    torch = _torch()
    count = lo_i32.numel()
    if scale is None:
        scale = float(np.float32(1.0) / np.sqrt(np.float32(g.qk_head_dim)))
    if out is None:
        out = torch.empty(count, g.num_heads * g.v_head_dim, dtype=torch.float32, device=q.device)
    blocks = kv_f32_block_bytes(g) + (count - 1) * kv_stride if count else 0
    i32, f32 = torch.int32, torch.float32
    _check(lib().nd_attend_step_f32_exact(
        ctx.h, C.byref(g), _arg(kv, torch.uint8, "kv", blocks), kv_stride, count,
        _arg(lo_i32, i32, "lo"), _arg(hi_i32, i32, "hi", count),
        _arg(q, f32, "q", count * g.num_heads * g.qk_head_dim), scale,
        _arg(out, f32, "out", count * g.num_heads * g.v_head_dim)))
    return out


def kv_unpack_f32(g, block_u8):
    """One f32 device block (CPU uint8 numpy array) as the reference's
    slot-major views: k [cap][kvh][qk] f32, v [cap][kvh][vd]."""
    H, cap, qk, vd = g.num_kv_heads, g.cap, g.qk_head_dim, g.v_head_dim
    vo = lib().nd_kv_f32_v_offset(C.byref(g))
    b = np.asarray(block_u8)
    k = b[:4 * H * cap * qk].view(np.float32).reshape(H, cap, qk).transpose(1, 0, 2)
    v = b[vo:vo + 4 * H * cap * vd].view(np.float32).reshape(H, cap, vd).transpose(1, 0, 2)
    return np.ascontiguousarray(k), np.ascontiguousarray(v)


def kv_unpack(g, block_u8):
    """Split one device block (as a CPU uint8 numpy array) into the
    reference's slot-major views: k [cap][kvh][qk] i8, v, ks [cap][kvh], vs."""
    off = kv_offsets(g)
    H, cap, qk, vd = g.num_kv_heads, g.cap, g.qk_head_dim, g.v_head_dim
    b = np.asarray(block_u8)
    k = b[:H * cap * qk].view(np.int8).reshape(H, cap, qk).transpose(1, 0, 2)
    v = b[off["v"]:off["v"] + H * cap * vd].view(np.int8).reshape(H, cap, vd).transpose(1, 0, 2)
    ks = b[off["ks"]:off["ks"] + 4 * H * cap].view(np.float32).reshape(H, cap).T
    vs = b[off["vs"]:off["vs"] + 4 * H * cap].view(np.float32).reshape(H, cap).T
    return (np.ascontiguousarray(k), np.ascontiguousarray(ks), np.ascontiguousarray(v),
            np.ascontiguousarray(vs))


class V3LayerCache:
    """One layer of V3Cache (cache.rs:125-393) with an int8 device block.

    The device block holds `cap` slots from the start; the reference's
    logical ring size (`slots`, grown by doubling, cache.rs:291-309) is kept
    here because span() clamps with it (cache.rs:322-331).  Physical slot
    pos % cap equals the reference's pos % slots at every write and read:
    while slots < cap every live position is below slots.
    """

    def __init__(self, ctx, num_heads, num_kv_heads, qk, vd, hint, window, max_seq_len):
        self.ctx = ctx
        hint = min(max(hint, 1), max_seq_len)
        self.window = window
        self.cap = min(window, max_seq_len) if window else max_seq_len
        self.slots = min(hint, self.cap)
        self.geom = kv_geom(num_heads, num_kv_heads, qk, vd, self.cap)
        self.block, self.block_bytes = kv_alloc(self.geom, 1, ctx.device)

    def _ensure(self, pos):
        if pos < self.slots or self.slots >= self.cap:
            return
        self.slots = min(max(self.slots * 2, pos + 1), self.cap)

    def write_kv(self, pos, k, v):
        torch = _torch()
        self._ensure(pos)
        p = torch.tensor([pos], dtype=torch.int32, device=k.device)
        kv_write(self.ctx, self.geom, self.block, 0, p, k, v)

    def span(self, pos):
        lo = pos + 1 - self.window if (self.window and pos + 1 > self.window) else 0
        lo = max(lo, max(pos + 1 - self.slots, 0))
        return lo, pos

    def attend_step(self, q, lo, hi, quant_query=False):
        torch = _torch()
        lo_t = torch.tensor([lo], dtype=torch.int32, device=q.device)
        hi_t = torch.tensor([hi], dtype=torch.int32, device=q.device)
        return attend_step_i8(self.ctx, self.geom, self.block, 0, lo_t, hi_t, q,
                              quant_query=quant_query)[0]


def attend_i8_prefill(ctx, num_heads, num_kv_heads, qk, vd, q, k, v, window=0, quant_query=False):
    """attend (attention.rs:218-287) with an int8 store: every prompt row t
    attends to max(0, t+1-window)..=t of the prompt's own quantised K/V."""
    torch = _torch()
    seq = q.shape[0]
    g = kv_geom(num_heads, num_kv_heads, qk, vd, max(seq, 1))
    blk, _ = kv_alloc(g, 1, q.device.index or 0)
    if isinstance(window, int) and window >= 0 and seq > 0:
        # both ends of the spans in two operations: 1 - w .. seq - 1 clamped to
        # 0 holds every row's first position, then, w - 1 on, its last (its own)
        w = min(window, seq) if window else seq
        ends = torch.arange(1 - w, seq, dtype=torch.int32, device=q.device).clamp_(min=0)
        lo, hi = ends[:seq], ends[w - 1:]
    else:
        hi = torch.arange(seq, dtype=torch.int32, device=q.device)
        lo = torch.clamp(hi + 1 - window, min=0).to(torch.int32) if window else torch.zeros_like(hi)
    kv_write(ctx, g, blk, 0, hi, k.contiguous(), v.contiguous())
    scale = float(np.float32(1.0) / np.float32(math.sqrt(qk)))
    return attend_step_i8(ctx, g, blk, 0, lo, hi, q.contiguous(), scale, quant_query)


# ---- rotary positions --------------------------------------------------------

_LAYOUTS = {"halves": 0, "pairs": 1}
_SCALINGS = {"plain": 0, "linear": 1, "parts": 2}


def rope(rot_dim, theta=10000.0, layout="halves", scaling="plain", factor=1.0, trained=0,
         turns=(1.0, 32.0), gain=1.0):
    """How positions turn a head vector (nd_rope, include/needle_amd.h): its
    first rot_dim elements in pairs (j, j + rot_dim / 2) or (2j, 2j + 1), by
    theta^(-2j / rot_dim) a position; scaling "linear" divides the frequencies
    by factor, "parts" those that make fewer than turns[0] turns over `trained`
    positions, none of those above turns[1], and in between in part; gain
    multiplies the turned elements."""
    if layout not in _LAYOUTS or scaling not in _SCALINGS:
        raise ValueError(f"layout {layout!r}: halves or pairs; scaling {scaling!r}: plain, linear or parts")
    return Rope(_LAYOUTS[layout], _SCALINGS[scaling], rot_dim, theta, factor, trained, turns[0], turns[1], gain)


def rope_freqs(r):
    """The rot_dim / 2 angles a position (fp64).  Host only."""
    out = np.zeros(max(r.rot_dim // 2, 1), np.float64)
    _check(lib().nd_rope_freqs(C.byref(r), out.ctypes.data_as(C.POINTER(C.c_double))))
    return out


def _near(ctx, t, name):
    """`t` is on the context's device."""
    if t.device.index != ctx.device:
        raise ValueError(f"{name}: on {t.device}, the context is on device {ctx.device}")


def _rows_arg(ctx, t, rows, width, name):
    """(address, row stride) of fp32 rows whose elements lie one after another."""
    f32 = _torch().float32
    if t.shape != (rows, width):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {(rows, width)}")
    if t.dtype != f32 or t.get_device() != ctx.device:
        if t.dtype != f32 or not t.is_cuda:
            raise ValueError(f"{name}: a device tensor of float32 is required, not {t.dtype} on {t.device}")
        _near(ctx, t, name)
    apart, step = t.stride()
    if rows and ((step != 1 and width > 1) or (rows > 1 and apart < width)):
        raise ValueError(f"{name}: strides {t.stride()}: rows must be contiguous and apart")
    return t.data_ptr(), apart


def _dev_arg(ctx, t, dtype, name, numel=0):
    """_arg of a tensor on the context's device, None of None."""
    if t is None:
        return None
    if t.dtype == dtype and t.get_device() == ctx.device and t.numel() >= numel and t.is_contiguous():
        return t.data_ptr()
    p = _arg(t, dtype, name, numel)  # says what is wrong
    _near(ctx, t, name)
    return p


def _empty(ctx, shape, dtype):
    """An output of a call: allocated for the context's stream, and kept until
    torch's current stream is done with it too where that is another one."""
    torch = _torch()
    if torch._C._cuda_getCurrentRawStream(ctx.device) == ctx.stream.cuda_stream:  # (1 us less than current_stream)
        return torch.empty(shape, dtype=dtype, device=ctx.stream.device)
    with torch.cuda.stream(ctx.stream):
        t = torch.empty(shape, dtype=dtype, device=ctx.stream.device)
    t.record_stream(torch.cuda.current_stream(ctx.device))
    return t


def rope_rows(ctx, r, x, pos, heads, out=None):
    """Rows of `heads` head vectors ([rows][heads * dim] fp32, rows may be
    apart) turned by their positions (int32; a row of negative position is not
    written).  out may be x."""
    torch = _torch()
    rows, width = x.shape
    if heads < 1 or width % heads:
        raise ValueError(f"x: {width} elements a row are not {heads} heads")
    xp, xs = _rows_arg(ctx, x, rows, width, "x")
    if out is None:
        out = _empty(ctx, (rows, width), torch.float32)
    yp, ys = _rows_arg(ctx, out, rows, width, "out")
    _check(lib().nd_rope_rows(ctx.h, C.byref(r), rows, _dev_arg(ctx, pos, torch.int32, "pos", rows), heads,
                              width // heads, xp, xs, yp, ys))
    return out


def kv_write_rope(ctx, g, r, kv, kv_stride, pos, k, v, q=None, q_out=None, rot_pos=None, per_block=1):
    """kv_write of keys turned by rot_pos (pos by default), per_block rows a
    block, and the queries turned in the same launch (returned; q_out may be
    q).  q, k and v are [count][heads * dim] fp32 whose rows may be apart, e.g.
    parts of one projection."""
    torch = _torch()
    n, i32 = pos.numel(), torch.int32
    if per_block < 1:
        raise ValueError(f"per_block {per_block} must be positive")
    blocks = kv_block_bytes(g) + (n - 1) // per_block * kv_stride if n else 0
    kp, ks = _rows_arg(ctx, k, n, g.num_kv_heads * g.qk_head_dim, "k")
    vp, vs = _rows_arg(ctx, v, n, g.num_kv_heads * g.v_head_dim, "v")
    qp = op = None
    qs = os_ = 0
    if q is not None:
        width = g.num_heads * g.qk_head_dim
        qp, qs = _rows_arg(ctx, q, n, width, "q")
        if q_out is None:
            q_out = _empty(ctx, (n, width), torch.float32)
        op, os_ = _rows_arg(ctx, q_out, n, width, "q_out")
    elif q_out is not None:
        raise ValueError("q_out without q")
    _check(lib().nd_kv_write_rope(
        ctx.h, C.byref(g), C.byref(r), _dev_arg(ctx, kv, torch.uint8, "kv", blocks), kv_stride, n, per_block,
        _dev_arg(ctx, pos, i32, "pos"), _dev_arg(ctx, rot_pos, i32, "rot_pos", n), qp, qs, op, os_, kp, ks, vp, vs))
    return q_out


def kv_read(ctx, g, kv, kv_stride, pos, per_block=1, k=None, v=None):
    """The cache's rows at `pos` as fp32, codes times scale: (k [count][kvh *
    qk], v [count][kvh * vd]); zeros where pos is negative."""
    torch = _torch()
    n, f32 = pos.numel(), torch.float32
    if per_block < 1:
        raise ValueError(f"per_block {per_block} must be positive")
    blocks = kv_block_bytes(g) + (n - 1) // per_block * kv_stride if n else 0
    wk, wv = g.num_kv_heads * g.qk_head_dim, g.num_kv_heads * g.v_head_dim
    if k is None:
        k = _empty(ctx, (n, wk), f32)
    if v is None:
        v = _empty(ctx, (n, wv), f32)
    _check(lib().nd_kv_read(ctx.h, C.byref(g), _dev_arg(ctx, kv, torch.uint8, "kv", blocks), kv_stride, n, per_block,
                            _dev_arg(ctx, pos, torch.int32, "pos"), _dev_arg(ctx, k, f32, "k", n * wk),
                            _dev_arg(ctx, v, f32, "v", n * wv)))
    return k, v


# ---- drafted trees -------------------------------------------------------------

def tree_mask(parents):
    """The masks of trees of drafted tokens (int32 words, [..][nodes][ceil(nodes
    / 32)], a numpy array for the device): parents [..][nodes] holds each node's
    parent, an earlier node, or a negative number for a root; a node attends to
    its ancestors and itself."""
    up = np.asarray(parents)
    n = up.shape[-1]
    if n < 1 or (up >= np.arange(n)).any():
        raise ValueError("parents: every node's parent must come before it")
    flat = up.reshape(-1, n)
    see = np.zeros((flat.shape[0], n, (n + 31) // 32), np.uint32)
    rows = np.arange(flat.shape[0])
    for j in range(n):
        see[:, j] = np.where((flat[:, j] >= 0)[:, None], see[rows, np.maximum(flat[:, j], 0)], 0)
        see[:, j, j // 32] |= np.uint32(1 << (j % 32))
    return see.view(np.int32).reshape(up.shape + (-1,))


def _work_arg(ctx, work):
    if work is None:
        return None, 0
    p = _dev_arg(ctx, work, _torch().uint8, "work")
    return p, work.numel()


def attend_tree_i8(ctx, g, kv, kv_stride, base, lo, mask, q, length=None, scale=None, quant_query=False,
                   out=None, work=None):
    """Attention of every session's drafted tree (nd_attend_tree_i8): base [S]
    committed positions, lo [S][N] the first one each node attends to, mask
    [S][N][ceil(N / 32)] int32 words of the nodes it attends to, length [S]
    nodes there are; q [S][N][heads * qk] fp32, out [S][N][heads * v] (rows
    past a tree's length are left as they are, zeros in a new `out`).  work: a
    uint8 device tensor of attend_tree_i8_work() bytes, needed while a graph is
    captured."""
    torch = _torch()
    i32, f32 = torch.int32, torch.float32
    if q.dim() != 3:
        raise ValueError(f"q: shape {tuple(q.shape)}, expected [sessions][nodes][heads * qk]")
    s, n = q.shape[0], q.shape[1]
    wo = g.num_heads * g.v_head_dim
    if scale is None:
        scale = float(np.float32(1.0) / np.sqrt(np.float32(g.qk_head_dim)))
    if out is None:
        out = _empty(ctx, (s, n, wo), f32)
        if length is not None:
            with torch.cuda.stream(ctx.stream):
                out.zero_()
    blocks = kv_block_bytes(g) + (s - 1) * kv_stride if s else 0
    wp, wb = _work_arg(ctx, work)
    _check(lib().nd_attend_tree_i8(
        ctx.h, C.byref(g), _dev_arg(ctx, kv, torch.uint8, "kv", blocks), kv_stride, s, n,
        _dev_arg(ctx, base, i32, "base", s), _dev_arg(ctx, length, i32, "length", s),
        _dev_arg(ctx, lo, i32, "lo", s * n), _dev_arg(ctx, mask, i32, "mask", s * n * ((n + 31) // 32)),
        _dev_arg(ctx, q, f32, "q", s * n * g.num_heads * g.qk_head_dim), scale, int(bool(quant_query)),
        _dev_arg(ctx, out, f32, "out", s * n * wo), wp, wb))
    return out


def attend_tree_i8_work(ctx, g, sessions, nodes):
    """Bytes of `work` that attend_tree_i8 needs."""
    return lib().nd_attend_tree_i8_work(ctx.h, C.byref(g), sessions, nodes)


# ---- logits under rules --------------------------------------------------------

def logits_adjust(ctx, x, hist=None, hist_len=None, out_from=None, repeat=None, presence=None, frequency=None,
                  bias_id=None, bias=None, bias_len=None, mask=None, mask_row=None, out=None, pick=False,
                  write=True, work=None):
    """Rows of logits ([count][n] fp32, rows may be apart) under penalties for
    repeated tokens, biases and grammar masks (nd_logits_adjust): hist [count][
    m] int32 tokens (-1: none) with hist_len and out_from [count], repeat,
    presence and frequency [count] fp32, bias_id and bias [count][b] with
    bias_len [count], mask [rows][ceil(n / 32)] int32 words with mask_row
    [count].  Returns the new logits (`out`, which may be x); with pick=True
    (logits, next), next[i] the first maximum of row i, -1 where no token is
    left; with write=False next alone."""
    torch = _torch()
    i32, f32 = torch.int32, torch.float32
    count, n = x.shape
    xp, xs = _rows_arg(ctx, x, count, n, "x")
    m = b = rows = words = 0
    if hist is not None:
        if hist.dim() != 2 or hist.shape[0] != count:
            raise ValueError(f"hist: shape {tuple(hist.shape)}, expected {count} rows")
        m = hist.shape[1]
    if bias is not None and bias_id is not None:
        if bias.dim() != 2 or bias.shape[0] != count or bias.shape != bias_id.shape:
            raise ValueError(f"bias: shape {tuple(bias.shape)}, bias_id {tuple(bias_id.shape)}: [count][b] both")
        b = bias.shape[1]
    if mask is not None:
        if mask.dim() != 2 or mask.shape[1] < (n + 31) // 32:
            raise ValueError(f"mask: shape {tuple(mask.shape)}, expected rows of {(n + 31) // 32} words")
        rows, words = mask.shape
    rules = LogitsRules(
        _dev_arg(ctx, hist, i32, "hist"), m, _dev_arg(ctx, hist_len, i32, "hist_len", count),
        _dev_arg(ctx, out_from, i32, "out_from", count), _dev_arg(ctx, repeat, f32, "repeat", count),
        _dev_arg(ctx, frequency, f32, "frequency", count), _dev_arg(ctx, presence, f32, "presence", count),
        _dev_arg(ctx, bias_id, i32, "bias_id"), _dev_arg(ctx, bias, f32, "bias"), b,
        _dev_arg(ctx, bias_len, i32, "bias_len", count), _dev_arg(ctx, mask, i32, "mask"), words, rows,
        _dev_arg(ctx, mask_row, i32, "mask_row", count))
    yp = ys = None
    if write:
        if out is None:
            out = _empty(ctx, (count, n), f32)
        yp, ys = _rows_arg(ctx, out, count, n, "out")
    nxt = _empty(ctx, (count,), i32) if pick or not write else None
    wp, wb = _work_arg(ctx, work)
    _check(lib().nd_logits_adjust(ctx.h, xp, xs, count, n, C.byref(rules), yp, ys or 0,
                                  nxt.data_ptr() if nxt is not None else None, wp, wb))
    return (out, nxt) if write and pick else out if write else nxt


def logits_adjust_work(ctx, count, n):
    """Bytes of `work` that logits_adjust needs."""
    return lib().nd_logits_adjust_work(ctx.h, count, n)


# ---- Needle-3 forward on the device ----------------------------------------

class V3Cfg(C.Structure):
    _fields_ = [("vocab_size", C.c_int32), ("out_vocab", C.c_int32), ("d_model", C.c_int32),
                ("num_heads", C.c_int32), ("num_kv_heads", C.c_int32), ("num_layers", C.c_int32),
                ("qk_head_dim", C.c_int32), ("v_head_dim", C.c_int32), ("max_seq_len", C.c_int32),
                ("hada_n", C.c_int32), ("mhc_lanes", C.c_int32), ("rope_theta", C.c_float),
                ("sliding_window", C.c_int32), ("n_global", C.c_int32),
                ("global_layers", C.c_int32 * 64), ("qkv_conv_taps", C.c_int32),
                ("n_orders", C.c_int32), ("orders", C.c_int32 * 8), ("e_heads", C.c_int32),
                ("e_slots", C.c_int32), ("e_sub_dim", C.c_int32), ("n_sites", C.c_int32),
                ("sites", C.c_int32 * 64), ("e_conv_taps", C.c_int32),
                ("e_conv_dilation", C.c_int32), ("e_seed_heads", C.c_int32)]


class V3Record(C.Structure):
    _fields_ = [("kind", C.c_int32), ("data", C.c_void_p), ("len", _sz), ("out", _sz),
                ("inn", _sz), ("group", _sz), ("bits", _sz)]


def v3_cfg(g):
    c = V3Cfg()
    for k in ("vocab_size", "out_vocab", "d_model", "num_heads", "num_kv_heads", "num_layers",
              "qk_head_dim", "v_head_dim", "max_seq_len", "hada_n", "mhc_lanes",
              "sliding_window", "qkv_conv_taps", "e_heads", "e_slots", "e_sub_dim",
              "e_conv_taps", "e_conv_dilation", "e_seed_heads"):
        setattr(c, k, g[k])
    c.rope_theta = g["rope_theta"]
    c.n_global = len(g["global_layers"])
    for i, v in enumerate(g["global_layers"]):
        c.global_layers[i] = v
    c.n_orders = len(g["orders"])
    for i, v in enumerate(g["orders"]):
        c.orders[i] = v
    c.n_sites = len(g["sites"])
    for i, v in enumerate(g["sites"]):
        c.sites[i] = v
    return c


def geom_of_cfg(c):
    """The geometry dict (the keys v3_cfg reads) of an nd_v3_cfg."""
    g = {k: getattr(c, k) for k in (
        "vocab_size", "out_vocab", "d_model", "num_heads", "num_kv_heads", "num_layers",
        "qk_head_dim", "v_head_dim", "max_seq_len", "hada_n", "mhc_lanes", "sliding_window",
        "qkv_conv_taps", "e_heads", "e_slots", "e_sub_dim", "e_conv_taps", "e_conv_dilation",
        "e_seed_heads")}
    g["rope_theta"] = c.rope_theta
    g["global_layers"] = [c.global_layers[i] for i in range(c.n_global)]
    g["orders"] = [c.orders[i] for i in range(c.n_orders)]
    g["sites"] = [c.sites[i] for i in range(c.n_sites)]
    return g


def _container_bytes(data):
    if isinstance(data, (str, os.PathLike)):
        with open(data, "rb") as f:
            data = f.read()
    return np.frombuffer(data, np.uint8) if not isinstance(data, np.ndarray) else \
        np.ascontiguousarray(data, np.uint8)


def cact_v3_config(data):
    """A .cact v3 container (path or bytes) read as CactV3::from_bytes +
    config_from_geometry + V3Layout::derive (needle-infer/src/cact.rs:994-1030,
    v3.rs:25-386) do: returns (geometry dict, records up to final_norm).
    Host only; raises NeedleError with the reference's error variant."""
    buf = _container_bytes(data)
    cfg, n = V3Cfg(), _sz()
    _check(lib().nd_v3_cact_config(buf.ctypes.data_as(C.c_void_p), buf.size, C.byref(cfg),
                                   C.byref(n)))
    return geom_of_cfg(cfg), n.value


def v3_kv_bytes(geom, seq_len, kv_int8=True):
    """Key/value cache bytes of one session of `seq_len` positions
    (V3Config::kv_bytes_at, crates/needle-core/src/v3/config.rs:143-179).
    Host only."""
    cfg = v3_cfg(geom)
    return lib().nd_v3_kv_bytes(C.byref(cfg), seq_len, int(bool(kv_int8)))


def v3_ladder(num_layers, depth):
    """The blocks a `depth`-block rung keeps, ascending (ladder_layer_indices,
    crates/needle-core/src/v3/ladder.rs:67-74).  Host only."""
    kept = (C.c_int32 * max(int(depth), 1))()
    _check(lib().nd_v3_ladder(num_layers, depth, kept))
    return [kept[i] for i in range(depth)]


def cact_v3_config_at_depth(data, depth):
    """The geometry of a container's `depth`-block rung and the parent
    blocks it keeps (config_at_depth with model_from_cact_at_depth's
    checks, needle-infer/src/v3.rs:620-664).  Host only."""
    buf = _container_bytes(data)
    cfg = V3Cfg()
    kept = (C.c_int32 * max(int(depth), 1))()
    _check(lib().nd_v3_cact_config_at_depth(buf.ctypes.data_as(C.c_void_p), buf.size, depth,
                                            C.byref(cfg), kept))
    return geom_of_cfg(cfg), [kept[i] for i in range(depth)]


class V3Model:
    """A Needle-3 model on the device, from canonical container records
    (V3Layout::derive order, crates/needle-infer/src/v3.rs:236-330), or from a
    .cact v3 container with `from_cact` (model_from_cact, v3.rs:438-482; with
    `depth`, the ladder rung model_from_cact_at_depth slices, v3.rs:656-734)."""

    @classmethod
    def from_cact(cls, ctx, data, depth=None):
        buf = _container_bytes(data)
        if depth is None:
            geom, _ = cact_v3_config(buf)
        else:
            geom, _ = cact_v3_config_at_depth(buf, depth)
        self = cls.__new__(cls)
        self.ctx, self.geom = ctx, geom
        h = C.c_void_p()
        if depth is None:
            _check(lib().nd_v3_model_from_cact(ctx.h, buf.ctypes.data_as(C.c_void_p), buf.size,
                                               C.byref(h)))
        else:
            _check(lib().nd_v3_model_from_cact_at_depth(ctx.h, buf.ctypes.data_as(C.c_void_p),
                                                        buf.size, depth, C.byref(h)))
        self.h = h
        self.rows = lib().nd_v3_logit_rows(h)
        return self

    def __init__(self, ctx, geom, records, codebook):
        self.ctx, self.geom = ctx, geom
        cfg = v3_cfg(geom)
        keep = [np.ascontiguousarray(r["data"]) for r in records]
        arr = (V3Record * len(records))()
        for i, (r, buf) in enumerate(zip(records, keep)):
            arr[i] = V3Record(r["kind"], buf.ctypes.data, buf.nbytes, r["out"], r["inn"],
                              r["group"], r["bits"])
        cb = np.ascontiguousarray(codebook, np.float32)
        h = C.c_void_p()
        _check(lib().nd_v3_model_create(ctx.h, C.byref(cfg), cb.ctypes.data_as(C.c_void_p), cb.size,
                                        arr, len(records), C.byref(h)))
        self.h = h
        self.rows = lib().nd_v3_logit_rows(h)

    def close(self):
        if getattr(self, "h", None) and _lib is not None:
            _lib.nd_v3_model_free(self.h)
            self.h = None

    __del__ = close


class V3Batch:
    """`sessions` decode sessions stepped in lockstep on the device, with
    int8 KV caches (kv_int8=True, KvPrecision::Int8) or f32 ones
    (KvPrecision::F32, needle_v3_generate's default); with max_chunk > 1 a
    prompt is prefilled up to max_chunk positions per pass (the reference's
    chunked prefill, bit-identical to stepping).  The batch is stepped
    through `ctx` (the model's context by default): a model is shared by any
    number of threads, each stepping its own batches through its own
    context."""

    def __init__(self, model, sessions, max_len, hint=None, max_chunk=1, kv_int8=True, ctx=None):
        self.model, self.sessions, self.max_chunk = model, sessions, max_chunk
        self.ctx = ctx if ctx is not None else model.ctx
        self.kv_int8 = bool(kv_int8)
        h = C.c_void_p()
        _check(lib().nd_v3_batch_create_ex(self.ctx.h, model.h, sessions, max_len,
                                           hint or max_len, max_chunk, int(self.kv_int8),
                                           C.byref(h)))
        self.h = h

    def close(self):
        if getattr(self, "h", None) and _lib is not None:
            _lib.nd_v3_batch_free(self.h)
            self.h = None

    __del__ = close

    def positions(self):
        out = np.zeros(self.sessions, np.int32)
        _check(lib().nd_v3_positions(self.h, out.ctypes.data_as(C.c_void_p)))
        return out

    def set_graphs(self, on):
        """Single-position steps as one replayed HIP graph, or kernel by
        kernel (the default, faster on ROCm 7.2); the results are identical."""
        _check(lib().nd_v3_batch_set_graphs(self.h, int(bool(on))))

    def _logits_arg(self, logits):
        if logits is None:
            return None
        torch = _torch()
        return _arg(logits, torch.float32, "logits", self.sessions * self.model.rows)

    def step(self, tokens, logits=None, want_next=True):
        """Feed tokens[i] to session i (V3Model::decode_step); returns the greedy
        next tokens, and fills `logits` ([sessions][rows] device tensor) if given."""
        tok = np.ascontiguousarray(tokens, np.int32).reshape(self.sessions)
        nxt = np.zeros(self.sessions, np.int32) if want_next else None
        _check(lib().nd_v3_step(self.ctx.h, self.model.h, self.h,
                                tok.ctypes.data_as(C.c_void_p),
                                nxt.ctypes.data_as(C.c_void_p) if want_next else None,
                                self._logits_arg(logits)))
        return nxt

    def prefill(self, tokens, logits=None, want_next=True):
        """tokens [sessions][count]: count consecutive positions per session in
        one pass (V3Model::prefill); returns the greedy token after the last."""
        tok = np.ascontiguousarray(tokens, np.int32).reshape(self.sessions, -1)
        nxt = np.zeros(self.sessions, np.int32) if want_next else None
        _check(lib().nd_v3_prefill(self.ctx.h, self.model.h, self.h,
                                   tok.ctypes.data_as(C.c_void_p), tok.shape[1],
                                   nxt.ctypes.data_as(C.c_void_p) if want_next else None,
                                   self._logits_arg(logits)))
        return nxt

    def greedy(self, first, steps):
        """`steps` greedy steps from first[i] (V3Engine's loop, nd_v3_generate):
        returns [sessions][steps], each step's choice; the device feeds each
        step's choice to the next without a host round trip."""
        tok = np.ascontiguousarray(first, np.int32).reshape(self.sessions)
        out = np.zeros((self.sessions, steps), np.int32)
        _check(lib().nd_v3_generate(self.ctx.h, self.model.h, self.h,
                                    tok.ctypes.data_as(C.c_void_p), steps,
                                    out.ctypes.data_as(C.c_void_p)))
        return out

    @staticmethod
    def greedy_many(batches, firsts, steps):
        """greedy() for several batches of one model at once (nd_v3_generate_many):
        batch i on its own context's stream, the steps enqueued in turn from
        this thread; returns one [sessions][steps] array per batch."""
        n = len(batches)
        model = batches[0].model
        assert all(b.model is model for b in batches), "one model"
        toks = [np.ascontiguousarray(f, np.int32).reshape(b.sessions) for b, f in zip(batches, firsts)]
        outs = [np.zeros((b.sessions, steps), np.int32) for b in batches]
        ctxs = (C.c_void_p * n)(*[b.ctx.h.value for b in batches])
        bs = (C.c_void_p * n)(*[b.h.value for b in batches])
        fs = (C.c_void_p * n)(*[t.ctypes.data for t in toks])
        ts = (C.c_void_p * n)(*[o.ctypes.data for o in outs])
        _check(lib().nd_v3_generate_many(ctxs, model.h, bs, n, fs, steps, ts))
        return outs

    def generate(self, prompts, steps):
        """Prefill each session's prompt, max_chunk positions per pass (or by
        stepping; the reference proves the two bit-identical), then `steps`
        greedy tokens: the prefill's choice, then the device loop's."""
        prompts = np.asarray(prompts, np.int32).reshape(self.sessions, -1)
        nxt = None
        n = prompts.shape[1]
        for t0 in range(0, n, self.max_chunk):
            t1 = min(n, t0 + self.max_chunk)
            last = t1 == n
            if t1 - t0 == 1:
                nxt = self.step(prompts[:, t0], want_next=last)
            else:
                nxt = self.prefill(prompts[:, t0:t1], want_next=last)
        out = np.zeros((self.sessions, steps), np.int32)
        if steps > 0:
            out[:, 0] = nxt
        if steps > 1:
            out[:, 1:] = self.greedy(nxt, steps - 1)
        return out
