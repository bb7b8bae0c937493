"""Single operators on CUDA tensors (the iec_ops_* calls of iec_cuda.h):
group normalisation over channels-last maps and layers in 8-bit floating
point, for networks built next to the four models.

    ops = iec.ops.Ops()
    codes, scales = ops.group_norm_fp8(x, 32, gamma, beta, act=iec.ops.SILU)   # x: n, h, w, c
    w, w_scales = ops.quantize_fp8(weights, block_rows=128)                    # once: n_out, c
    y = ops.matmul_fp8(codes, scales, w, w_scales, bias, residual=x.flatten(0, 2))

Tensors are torch tensors of the handle's device. Work is queued on
torch's current stream unless `stream` (an integer cudaStream_t) is given,
and the calls return without waiting. There is no CPU fallback.
"""

from __future__ import annotations

import ctypes

import torch

from . import IecError, ERR_INPUT, Options, _check, lib

NONE, RELU, GELU, SIGMOID, SILU = range(5)
BLOCK = 128  # values along a row that share a scale

_DTYPE = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_LEGACY_STREAM = 1  # cudaStreamLegacy: torch's default stream has the handle 0


def _bad(message: str):
    raise IecError(ERR_INPUT, message)


def _dtype(t, what: str) -> int:
    code = _DTYPE.get(t.dtype)
    if code is None:
        _bad(f"{what} is {t.dtype}: float16, bfloat16 or float32 are taken")
    return code


def _f32_vector(t, n: int, what: str):
    if t is None:
        return None
    if t.dtype is not torch.float32 or t.dim() != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1):
        _bad(f"{what} must be {n} contiguous float32 values")
    return t.data_ptr()


def _rows(t, rows: int, k: int, dtype, what: str) -> int:
    """The row stride of a rows x k matrix whose rows are contiguous."""
    if t.dtype is not dtype:
        _bad(f"{what} is {t.dtype}, not {dtype}")
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] != k:
        _bad(f"{what} is {tuple(t.shape)}, not {(rows, k)}")
    if k > 1 and t.stride(1) != 1:
        _bad(f"{what} must have contiguous rows")
    return t.stride(0) if rows > 1 else max(k, 1)


def _maps(t, what: str):
    """(maps, pixels, channels, pixel stride, map stride) of n x ... x c."""
    if t.dim() < 2:
        _bad(f"{what} must be maps x pixels (or height x width) x channels")
    shape, stride = t.shape, t.stride()
    n, c = shape[0], shape[-1]
    if c > 1 and stride[-1] != 1:
        _bad(f"{what} must have contiguous channels")
    pixels, step = 1, 0
    for size, s in zip(shape[-2:0:-1], stride[-2:0:-1]):
        if size == 1:
            continue
        if pixels > 1 and s != step * pixels:
            _bad(f"{what} must have its pixels at one stride")
        if pixels == 1:
            step = s
        pixels *= size
    return n, pixels, c, step if pixels > 1 else c, stride[0] if n > 1 else c


def empty_codes(rows: int, k: int, device):
    """Codes of a rows x k matrix as matmul_fp8 reads them: rows a multiple
    of 16 bytes apart."""
    return torch.empty((rows, -(-max(k, 1) // 16) * 16), dtype=torch.float8_e4m3fn, device=device)[:, :k]


class Ops:
    """A handle of one GPU for the operators (iec_ops in iec_cuda.h)."""

    def __init__(self, device: int = -1, timeout_ms: int = 0):
        L = lib()
        vp, sz, i32, f32 = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_float
        norm = [vp, vp, i32, sz, sz, sz, sz, sz, sz, vp, vp, f32, i32]
        L.iec_ops_device_name.restype = ctypes.c_char_p
        L.iec_ops_device_name.argtypes = [vp]
        L.iec_ops_free.argtypes = [vp]
        L.iec_ops_sync.argtypes = [vp, vp]
        L.iec_ops_group_norm.argtypes = norm + [vp, sz, sz, vp]
        L.iec_ops_group_norm_fp8.argtypes = norm + [vp, sz, vp, sz, vp]
        L.iec_ops_quantize_fp8.argtypes = [vp, vp, i32, sz, sz, sz, sz, vp, sz, vp, sz, vp]
        L.iec_ops_matmul_fp8.argtypes = [vp, vp, sz, vp, sz, vp, sz, vp, sz, vp, vp, sz, sz, sz, sz, i32, i32, vp, sz, vp]
        self._h = ctypes.c_void_p()
        opt = Options(device, timeout_ms, 0)
        _check(L.iec_ops_open(ctypes.byref(opt), ctypes.byref(self._h)))
        self._lib = L

    def close(self):
        if getattr(self, "_h", None):
            lib().iec_ops_free(self._h)
            self._h = None

    __del__ = close

    def gpu(self) -> str:
        """The device's name."""
        return self._lib.iec_ops_device_name(self._h).decode()

    def sync(self, stream=None):
        """Wait (bounded) for the stream's work and raise what went wrong."""
        _check(self._lib.iec_ops_sync(self._h, self._stream(stream)))

    @staticmethod
    def _stream(stream, device=None):
        if stream is None:
            stream = torch.cuda.current_stream(device).cuda_stream
        return stream or _LEGACY_STREAM

    def group_norm(self, x, groups: int, gamma=None, beta=None, eps: float = 1e-5, act: int = NONE, out=None,
                   stream=None):
        """Group normalisation and activation of channels-last maps (n, ...,
        c); `out` (default: a new tensor) may be `x`."""
        dtype = _dtype(x, "x")
        n, pixels, c, step, map_step = _maps(x, "x")
        if out is None:
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if out.dtype is not x.dtype or out.shape != x.shape:
            _bad("out must have the shape and type of x")
        _, _, _, out_step, out_map_step = _maps(out, "out")
        _check(self._lib.iec_ops_group_norm(
            self._h, x.data_ptr(), dtype, n, pixels, c, step, map_step, groups, _f32_vector(gamma, c, "gamma"),
            _f32_vector(beta, c, "beta"), eps, act, out.data_ptr(), out_step, out_map_step,
            self._stream(stream, x.device)))
        return out

    def group_norm_fp8(self, x, groups: int, gamma=None, beta=None, eps: float = 1e-5, act: int = NONE, codes=None,
                       scales=None, stream=None):
        """group_norm with its result as 8-bit rows, one per pixel: (codes
        n*pixels x c, scales ceil(c / 128) x n*pixels)."""
        dtype = _dtype(x, "x")
        n, pixels, c, step, map_step = _maps(x, "x")
        codes, code_step, scales, scale_step = self._fp8_out(codes, scales, n * pixels, c, n * pixels, x.device)
        _check(self._lib.iec_ops_group_norm_fp8(
            self._h, x.data_ptr(), dtype, n, pixels, c, step, map_step, groups, _f32_vector(gamma, c, "gamma"),
            _f32_vector(beta, c, "beta"), eps, act, codes.data_ptr(), code_step, scales.data_ptr(), scale_step,
            self._stream(stream, x.device)))
        return codes, scales

    def quantize_fp8(self, x, block_rows: int = 1, codes=None, scales=None, stream=None):
        """A rows x k matrix as 8-bit rows: (codes rows x k, scales
        ceil(k / 128) x rows), with block_rows 128 (weights) scales
        ceil(k / 128) x ceil(rows / 128)."""
        dtype = _dtype(x, "x")
        if x.dim() != 2:
            _bad("x must be rows x values")
        rows, k = x.shape
        step = _rows(x, rows, k, x.dtype, "x")
        scale_rows = rows if block_rows != BLOCK else -(-rows // BLOCK)
        codes, code_step, scales, scale_step = self._fp8_out(codes, scales, rows, k, scale_rows, x.device)
        _check(self._lib.iec_ops_quantize_fp8(self._h, x.data_ptr(), dtype, rows, k, step, block_rows,
                                              codes.data_ptr(), code_step, scales.data_ptr(), scale_step,
                                              self._stream(stream, x.device)))
        return codes, scales

    @staticmethod
    def _fp8_out(codes, scales, rows: int, k: int, scale_rows: int, device):
        if codes is None:
            codes = empty_codes(rows, k, device)
        code_step = _rows(codes, rows, k, torch.float8_e4m3fn, "codes")
        blocks = -(-k // BLOCK)
        if scales is None:
            scales = torch.empty((blocks, scale_rows), dtype=torch.float32, device=device)
        return codes, code_step, scales, _rows(scales, blocks, scale_rows, torch.float32, "scales")

    def matmul_fp8(self, a, a_scales, w, w_scales, bias=None, act: int = NONE, residual=None, out=None,
                   dtype=torch.float16, stream=None):
        """act(a w^T + bias) + residual for 8-bit rows a (m x k) and w (n x
        k, quantised with block_rows 128); `out` (default: a new tensor of
        `dtype`) may be `residual`."""
        if a.dim() != 2 or w.dim() != 2:
            _bad("a and w must be matrices")
        m, k = a.shape
        n = w.shape[0]
        fp8, blocks = torch.float8_e4m3fn, -(-k // BLOCK)
        a_step, w_step = _rows(a, m, k, fp8, "a"), _rows(w, n, k, fp8, "w")
        a_scale_step = _rows(a_scales, blocks, m, torch.float32, "a_scales")
        w_scale_step = _rows(w_scales, blocks, -(-n // BLOCK), torch.float32, "w_scales")
        if out is None:
            out = torch.empty((m, n), dtype=dtype, device=a.device)
        code = _dtype(out, "out")
        out_step = _rows(out, m, n, out.dtype, "out")
        res, res_step = None, 0
        if residual is not None:
            res, res_step = residual.data_ptr(), _rows(residual, m, n, out.dtype, "residual")
        _check(self._lib.iec_ops_matmul_fp8(
            self._h, a.data_ptr(), a_step, a_scales.data_ptr(), a_scale_step, w.data_ptr(), w_step,
            w_scales.data_ptr(), w_scale_step, _f32_vector(bias, n, "bias"), res, res_step, m, n, k, act, code,
            out.data_ptr(), out_step, self._stream(stream, a.device)))
        return out
