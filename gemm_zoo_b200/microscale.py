"""Microscaled 4-bit matrices (include/gemmzoo/microscale.h): quantisation and its inverse, the
product of two quantised matrices, and the gated feed-forward product.

    q  = mx_quantize(x, MX_NVFP4)                          # rows x k, blocks along k
    w  = mx_quantize(weight, MX_NVFP4, multiplier=256.0)   # n x k
    MxGemm(m, n, k, MX_NVFP4, torch.bfloat16)(q, w, None, d, 1 / 256.0, 0.0)

The reference (AD2605/gemm-zoo) has no counterpart: its narrowest type is 8 bits.
"""
from __future__ import annotations

import ctypes as C

from . import api
from .api import ACT_NONE, ACT_SILU, GZ_OK, Epilogue, GzError, ROW_MAJOR, _stream_handle, lib

MX_FP4, MX_NVFP4 = 16, 17
MX_CFG_AUTO, MX_CFG_PAIR, MX_CFG_SINGLE, MX_CFG_SWAP_M16, MX_CFG_SWAP_M32, MX_CFG_SWAP_M64 = 0, 1, 2, 3, 4, 5
MX_CFG_PAIR_N128, MX_CFG_SINGLE_N128 = 6, 7

EXPORTED_SYMBOLS = [
    "gz_mx_code_pitch", "gz_mx_scale_bytes", "gz_mx_quantize", "gz_mx_dequantize", "gz_mx_desc_validate",
    "gz_mx_plan_create", "gz_mx_plan_destroy", "gz_mx_plan_info_get", "gz_mx_gemm_run", "gz_mx_gated_run",
    "gz_mx_last_device_status",
]


class MxDesc(C.Structure):
    _fields_ = [
        ("struct_size", C.c_uint32), ("format", C.c_int32), ("out_type", C.c_int32), ("gated", C.c_int32),
        ("device", C.c_int32), ("config", C.c_int32), ("split", C.c_int32), ("flags", C.c_uint32),
        ("m", C.c_int64), ("n", C.c_int64), ("k", C.c_int64),
        ("pitch_a", C.c_int64), ("pitch_b", C.c_int64), ("ldc", C.c_int64), ("ldd", C.c_int64),
        ("wait_limit_ns", C.c_uint64),
    ]

    @classmethod
    def make(cls, format, out_type, m, n, k, gated=False, pitch_a=0, pitch_b=0, ldc=0, ldd=0, device=0,
             config=MX_CFG_AUTO, split=0, flags=0, wait_limit_ns=0):
        d = cls()
        d.struct_size = C.sizeof(cls)
        d.format, d.out_type, d.gated = format, out_type, int(gated)
        d.device, d.config, d.split, d.flags = device, config, split, flags
        d.m, d.n, d.k = m, n, k
        d.pitch_a, d.pitch_b, d.ldc, d.ldd = pitch_a, pitch_b, ldc, ldd
        d.wait_limit_ns = wait_limit_ns
        return d


class MxPlanInfo(C.Structure):
    _fields_ = [
        ("config", C.c_int32), ("split", C.c_int32), ("tile_m", C.c_int32), ("tile_n", C.c_int32),
        ("tile_k", C.c_int32), ("stages", C.c_int32), ("grid", C.c_int32), ("smem_bytes", C.c_int32),
        ("out_tma", C.c_int32), ("reserved", C.c_int32), ("tiles", C.c_int64),
    ]

    def as_dict(self):
        return {f: getattr(self, f) for f, _ in self._fields_}


_bound = None


def _bind():
    global _bound
    if _bound is not None:
        return _bound
    L = lib()
    vp, i32, i64, f32 = C.c_void_p, C.c_int32, C.c_int64, C.c_float
    fp = C.POINTER(f32)
    L.gz_mx_code_pitch.argtypes = [i64]
    L.gz_mx_scale_bytes.argtypes = [i32, i64, i64]
    L.gz_mx_quantize.argtypes = [vp, i32, i32, i64, i64, i64, i32, f32, vp, i64, vp, i32, vp]
    L.gz_mx_dequantize.argtypes = [vp, i64, vp, i32, i64, i64, f32, vp, i32, i32, i64, i32, vp]
    L.gz_mx_desc_validate.argtypes = [C.POINTER(MxDesc), C.c_int, C.POINTER(MxPlanInfo)]
    L.gz_mx_plan_create.argtypes = [C.POINTER(vp), C.POINTER(MxDesc)]
    L.gz_mx_plan_destroy.argtypes = [vp]
    L.gz_mx_plan_info_get.argtypes = [vp, C.POINTER(MxPlanInfo)]
    L.gz_mx_gemm_run.argtypes = [vp, vp, vp, vp, vp, vp, vp, fp, fp, C.POINTER(Epilogue), vp]
    L.gz_mx_gated_run.argtypes = [vp, vp, vp, vp, vp, vp, vp, vp, vp, fp, fp, i32, f32, vp]
    L.gz_mx_last_device_status.argtypes = [vp, vp, C.POINTER(C.c_uint32 * 4)]
    for name in EXPORTED_SYMBOLS:
        getattr(L, name).restype = C.c_int
    L.gz_mx_code_pitch.restype = i64
    L.gz_mx_scale_bytes.restype = i64
    _bound = L
    return L


def code_pitch(k: int) -> int:
    """Bytes of one packed row of codes."""
    return _bind().gz_mx_code_pitch(k)


def scale_bytes(format: int, rows: int, k: int) -> int:
    """Bytes of the scale array of a rows x k matrix."""
    return _bind().gz_mx_scale_bytes(format, rows, k)


class MxMatrix:
    """A quantised rows x k matrix: `codes` (uint8, rows x pitch bytes) and `scales` (uint8, flat, in tiles of
    128 rows x 4 blocks); the layout is that of include/gemmzoo/microscale.h.  The attributes are not replaced
    after construction, which checked them together; the tensors' contents are the caller's."""

    __slots__ = ("_codes", "_scales", "_key")  # _key: (rows, k, format, pitch, device), what a plan compares
    codes, scales = property(lambda self: self._codes), property(lambda self: self._scales)
    rows, k = property(lambda self: self._key[0]), property(lambda self: self._key[1])
    format, pitch = property(lambda self: self._key[2]), property(lambda self: self._key[3])
    device = property(lambda self: self._key[4])
    _codes_ptr, _scales_ptr = property(lambda self: self._codes.data_ptr()), property(lambda self: self._scales.data_ptr())

    def __init__(self, codes, scales, rows, k, format):
        import torch
        need = scale_bytes(format, rows, k)
        if need < 0:
            raise ValueError("MxMatrix: rows and k must be positive and format one of MX_FP4, MX_NVFP4")
        if not (isinstance(codes, torch.Tensor) and isinstance(scales, torch.Tensor) and codes.dtype == torch.uint8 and
                scales.dtype == torch.uint8):
            raise ValueError("MxMatrix: codes and scales are uint8 tensors")
        if not (codes.is_cuda and codes.device == scales.device):
            raise ValueError("MxMatrix: codes and scales must live on one CUDA device")
        pitch = codes.stride(0) if codes.dim() == 2 and rows > 1 else codes.shape[-1]
        packed = code_pitch(k)
        if (codes.dim() != 2 or codes.shape[0] != rows or codes.shape[1] < packed or codes.stride(1) != 1 or pitch % 16 or
                pitch < packed):
            raise ValueError(f"MxMatrix: codes must be rows x at least {packed} bytes, contiguous along a row, "
                             "rows a multiple of 16 bytes apart that do not overlap")
        if not scales.is_contiguous() or scales.numel() < need:
            raise ValueError(f"MxMatrix: scales must be {need} contiguous bytes")
        if codes.data_ptr() % 16 or scales.data_ptr() % 16:
            raise ValueError("MxMatrix: codes and scales must be 16-byte aligned")
        self._codes, self._scales = codes, scales
        self._key = (rows, k, format, pitch, codes.get_device())

    @classmethod
    def empty(cls, rows, k, format, device="cuda"):
        """Uninitialised storage (the functions that write a quantised matrix write all of it)."""
        import torch
        need, pitch = scale_bytes(format, rows, k), code_pitch(k)
        if need < 0:
            raise ValueError("MxMatrix: rows and k must be positive and format one of MX_FP4, MX_NVFP4")
        return cls(torch.empty(rows, pitch, dtype=torch.uint8, device=device),
                   torch.empty(need, dtype=torch.uint8, device=device), rows, k, format)


def tile_scales(linear, format):
    """rows x blocks scale bytes (one row after the other, as checkpoints hold them) -> the tiled array."""
    import torch
    if format not in (MX_FP4, MX_NVFP4):
        raise ValueError("tile_scales: format must be one of MX_FP4, MX_NVFP4")
    if linear.dim() != 2 or linear.element_size() != 1 or linear.numel() == 0:
        raise ValueError("tile_scales: rows x blocks scale bytes are needed")
    rows, blocks = linear.shape
    rg, bg = -(-rows // 128), -(-blocks // 4)
    s = torch.zeros(rg * 128, bg * 4, dtype=torch.uint8, device=linear.device)
    s[:rows, :blocks] = linear.view(torch.uint8)
    return s.view(rg, 4, 32, bg, 4).permute(0, 3, 2, 1, 4).reshape(-1)


def linear_scales(q: MxMatrix):
    """The inverse of tile_scales: the rows x blocks scale bytes of a quantised matrix."""
    blocks = -(-q.k // (16 if q.format == MX_NVFP4 else 32))
    rg, bg = -(-q.rows // 128), -(-blocks // 4)
    s = q.scales[:rg * bg * 512].view(rg, bg, 32, 4, 4).permute(0, 3, 2, 1, 4)
    return s.reshape(rg * 128, bg * 4)[:q.rows, :blocks].contiguous()


def _refuse_matrix(x, what):
    if x.dim() != 2 or not x.is_cuda:
        raise ValueError(f"{what}: a 2-D CUDA tensor is needed")
    if x.shape[1] > 1 and x.stride(1) != 1:
        raise ValueError(f"{what}: the last dimension must be contiguous")
    raise ValueError(f"{what}: rows overlap")


# The two calls below cost about as much on the host as on the GPU at the sizes of a single token, so they ask each
# thing of torch once.
def mx_quantize(x, format, layout=ROW_MAJOR, multiplier=1.0, out=None, stream=None):
    """Quantise x * multiplier along k (gz_mx_quantize).  x: 2-D, rows x k (ROW_MAJOR) or k x rows (COL_MAJOR).
    Returns `out`, or a new MxMatrix.  stream: None is the default stream, as everywhere in this package."""
    shape, strides = x.shape, x.stride()
    if len(shape) != 2 or not x.is_cuda or (strides[1] != 1 and shape[1] > 1) or (strides[0] < shape[1] and shape[0] > 1):
        _refuse_matrix(x, "mx_quantize")
    rows, k = shape if layout == ROW_MAJOR else (shape[1], shape[0])
    if out is None:
        import torch
        if stream is None:
            on = torch.cuda.default_stream(x.device)
        else:
            on = torch.cuda.ExternalStream(stream, x.device) if isinstance(stream, int) and stream else stream
        with torch.cuda.stream(on or torch.cuda.default_stream(x.device)):  # the allocator then knows the memory's stream
            out = MxMatrix.empty(rows, k, format, x.device)
    to = out._key
    if to[0] != rows or to[1] != k or to[2] != format or to[4] != x.get_device():
        raise ValueError("mx_quantize: out has another size, format or device")
    st = (_bound or _bind()).gz_mx_quantize(x.data_ptr(), api._torch_dtype_code(x.dtype), layout,
                                            strides[0] if shape[0] > 1 else 0, rows, k, format, multiplier, out._codes_ptr,
                                            to[3], out._scales_ptr, to[4], _stream_handle(stream))
    if st != GZ_OK:
        raise GzError(st, "gz_mx_quantize")
    return out


def mx_dequantize(q: MxMatrix, out, layout=ROW_MAJOR, multiplier=1.0, stream=None):
    """code * scale * multiplier into `out` (gz_mx_dequantize), a 2-D tensor in `layout`.  Returns `out`."""
    shape, strides = out.shape, out.stride()
    if len(shape) != 2 or not out.is_cuda or (strides[1] != 1 and shape[1] > 1) or (strides[0] < shape[1] and shape[0] > 1):
        _refuse_matrix(out, "mx_dequantize")
    rows, k = shape if layout == ROW_MAJOR else (shape[1], shape[0])
    q_rows, q_k, format, pitch, device = q._key
    if q_rows != rows or q_k != k or device != out.get_device():
        raise ValueError("mx_dequantize: out has another size or device")
    st = (_bound or _bind()).gz_mx_dequantize(q._codes_ptr, pitch, q._scales_ptr, format, rows, k, multiplier,
                                              out.data_ptr(), api._torch_dtype_code(out.dtype), layout,
                                              strides[0] if shape[0] > 1 else 0, device, _stream_handle(stream))
    if st != GZ_OK:
        raise GzError(st, "gz_mx_dequantize")
    return out


def mx_validate(desc: MxDesc, sm_count: int = 0):
    """Host-only validation.  Returns (status, MxPlanInfo)."""
    info = MxPlanInfo()
    st = _bind().gz_mx_desc_validate(C.byref(desc), sm_count, C.byref(info))
    return st, info


class _MxPlan:
    """Owns a gz_mx_plan."""

    def __init__(self, desc: MxDesc):
        self.desc = desc
        self._h = C.c_void_p()
        h = C.c_void_p()
        st = _bind().gz_mx_plan_create(C.byref(h), C.byref(desc))
        if st != GZ_OK:
            raise GzError(st, "gz_mx_plan_create")
        self._h = h

    def info(self) -> MxPlanInfo:
        info = MxPlanInfo()
        st = _bind().gz_mx_plan_info_get(self._h, C.byref(info))
        if st != GZ_OK:
            raise GzError(st, "gz_mx_plan_info_get")
        return info

    def device_status(self, stream=None):
        """(status, detail[4]) after synchronising `stream`."""
        detail = (C.c_uint32 * 4)()
        st = _bind().gz_mx_last_device_status(self._h, _stream_handle(stream), C.byref(detail))
        return st, list(detail)

    def destroy(self):
        if self._h:
            _bind().gz_mx_plan_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass

    def _refuse(self, name, q, key):
        got = getattr(q, "_key", None)
        raise ValueError(f"{name}: an MxMatrix of (rows, k, format, pitch, device) = {key} is needed, got {got or type(q)}")


def _out_code(t):
    return t if isinstance(t, int) else api._torch_dtype_code(t)


class _Dense:
    """What a torch tensor given for C or D must be: the plan reads or writes it by address.  (An address, an int, is taken as
    it is.)  These checks run in every call, beside kernels of a few microseconds, so they compare prepared values."""

    def __init__(self, name, code, rows, cols, ld, device):
        import torch
        self.name, self.ld, self.device = name, ld, device
        self.shape, self.strides = torch.Size((rows, cols)), (ld, 1)
        self.dtype = next((t for t, c in _torch_types().items() if c == code), None)

    def address(self, t):
        if isinstance(t, int):
            return t
        if t.stride() != self.strides or t.shape != self.shape or t.dtype is not self.dtype or t.get_device() != self.device:
            self._look_closer(t)
        return t.data_ptr()

    def _look_closer(self, t):
        rows, cols = self.shape
        ok = (t.shape == self.shape and t.dtype is self.dtype and t.get_device() == self.device and
              (t.stride(1) == 1 or cols == 1) and (t.stride(0) == self.ld or rows == 1))  # strides of one row mean nothing
        if not ok:
            raise ValueError(f"{self.name}: expected {tuple(self.shape)}, rows {self.ld} elements apart, {self.dtype}, on device "
                             f"{self.device}; got {tuple(t.shape)}, strides {t.stride()}, {t.dtype}, {t.device}")


def _torch_types():
    import torch
    api._torch_dtype_code(torch.float32)
    return api._TORCH_DT


def _check_vector(name, t, length, device):
    if t is None or not hasattr(t, "data_ptr"):
        return
    import torch
    if t.dtype != torch.float32 or t.numel() != length or not t.is_contiguous() or not t.is_cuda or t.get_device() != device:
        raise ValueError(f"{name}: {length} contiguous fp32 values on device {device} are needed")


class MxGemm(_MxPlan):
    """D[m x n] = act(alpha * row_scale * col_scale * A B^T + beta * C + bias) for quantised A (m x k) and
    B (n x k) (gz_mx_gemm_run).  pitch_a / pitch_b: bytes between rows of codes, ldc / ldd: elements between rows,
    0 = packed.  c and d: m x n tensors of the output type with those strides (or addresses)."""

    def __init__(self, m, n, k, format, out_dtype, ldc=0, ldd=0, pitch_a=0, pitch_b=0, device=0, config=MX_CFG_AUTO,
                 split=0, flags=0, wait_limit_ns=0):
        super().__init__(MxDesc.make(format, _out_code(out_dtype), m, n, k, False, pitch_a, pitch_b, ldc, ldd, device,
                                     config, split, flags, wait_limit_ns))
        out = self.desc.out_type
        self._m, self._n, self._device = m, n, device
        self._a = (m, k, format, pitch_a or code_pitch(k), device)
        self._b = (n, k, format, pitch_b or code_pitch(k), device)
        self._c, self._d = _Dense("c", out, m, n, ldc or n, device), _Dense("d", out, m, n, ldd or n, device)
        self._run = _bound.gz_mx_gemm_run

    def __call__(self, a: MxMatrix, b: MxMatrix, c, d, alpha, beta, bias=None, row_scale=None, col_scale=None,
                 activation=ACT_NONE, stream=None):
        if getattr(a, "_key", None) != self._a:
            self._refuse("a", a, self._a)
        if getattr(b, "_key", None) != self._b:
            self._refuse("b", b, self._b)
        dp = self._d.address(d)
        cp = None if c is None else self._c.address(c)
        ep = None
        if activation != ACT_NONE or bias is not None or row_scale is not None or col_scale is not None:
            _check_vector("bias", bias, self._n, self._device)
            _check_vector("row_scale", row_scale, self._m, self._device)
            _check_vector("col_scale", col_scale, self._n, self._device)
            ep = C.byref(Epilogue.make(bias, row_scale, col_scale, activation))
        st = self._run(self._h, a._codes_ptr, a._scales_ptr, b._codes_ptr, b._scales_ptr, cp, dp, C.byref(C.c_float(alpha)),
                       C.byref(C.c_float(beta)), ep, _stream_handle(stream))
        if st != GZ_OK:
            raise GzError(st, "gz_mx_gemm_run")


class MxGated(_MxPlan):
    """D[m x n] = act(alpha_gate * A G^T) * (alpha_up * A U^T) for quantised A (m x k), gate and up (n x k) in one
    launch (gz_mx_gated_run).  out_dtype: a torch type (or DT_* code) for a plain D, or MX_FP4 / MX_NVFP4 for an
    MxMatrix, which then holds D * out_multiplier."""

    def __init__(self, m, n, k, format, out_dtype, activation=ACT_SILU, ldd=0, pitch_a=0, pitch_b=0, device=0,
                 config=MX_CFG_AUTO, split=0, flags=0, wait_limit_ns=0):
        super().__init__(MxDesc.make(format, _out_code(out_dtype), m, n, k, True, pitch_a, pitch_b, 0, ldd, device,
                                     config, split, flags, wait_limit_ns))
        self.activation = activation
        out = self.desc.out_type
        self._a = (m, k, format, pitch_a or code_pitch(k), device)
        self._b = (n, k, format, pitch_b or code_pitch(k), device)
        self._quantised = out in (MX_FP4, MX_NVFP4)
        self._d = (m, n, out, ldd or code_pitch(n), device) if self._quantised else _Dense("d", out, m, n, ldd or n, device)
        self._run = _bound.gz_mx_gated_run

    def __call__(self, a: MxMatrix, gate: MxMatrix, up: MxMatrix, d, alpha_gate=1.0, alpha_up=1.0, out_multiplier=1.0,
                 stream=None):
        if getattr(a, "_key", None) != self._a:
            self._refuse("a", a, self._a)
        if getattr(gate, "_key", None) != self._b:
            self._refuse("gate", gate, self._b)
        if getattr(up, "_key", None) != self._b:
            self._refuse("up", up, self._b)
        if self._quantised:
            if getattr(d, "_key", None) != self._d:
                self._refuse("d", d, self._d)
            dp, ds = d._codes_ptr, d._scales_ptr
        else:
            dp, ds = self._d.address(d), None
        st = self._run(self._h, a._codes_ptr, a._scales_ptr, gate._codes_ptr, gate._scales_ptr, up._codes_ptr, up._scales_ptr,
                       dp, ds, C.byref(C.c_float(alpha_gate)), C.byref(C.c_float(alpha_up)), self.activation, out_multiplier,
                       _stream_handle(stream))
        if st != GZ_OK:
            raise GzError(st, "gz_mx_gated_run")
