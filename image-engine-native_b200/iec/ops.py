"""Single operators on CUDA tensors (the iec_ops_* calls of iec_cuda.h):
group normalisation over channels-last maps and layers in 8-bit floating
point, for networks built next to the four models.

    ops = iec.ops.Ops()
    codes, scales = ops.group_norm_fp8(x, 32, gamma, beta, act=iec.ops.SILU)   # x: n, h, w, c
    w, w_scales = ops.quantize_fp8(weights, block_rows=128)                    # once: n_out, c
    y = ops.matmul_fp8(codes, scales, w, w_scales, bias, residual=x.flatten(0, 2))

Where all outputs are given, a call goes through the compiled binding
(binding/ops_binding.cpp); what does not fit there comes back here, where
outputs are allocated and arguments checked one by one.

Tensors are torch tensors of the handle's device. Work is queued on
torch's current stream unless `stream` (an integer cudaStream_t) is given,
and the calls return without waiting. Outputs that a call allocates belong
to the stream it is queued on, as under torch.cuda.stream; inputs of another
stream are the caller's to order. There is no CPU fallback.

The operators have no gradients: where torch records them (outside
torch.no_grad()), a tensor that requires one is refused.
"""

from __future__ import annotations

import ctypes
from contextlib import nullcontext
from struct import Struct
from struct import error as StructError

import torch

from . import ERR_INPUT, IecError, Options, _check, lib

try:
    from . import _ops_binding as _fast
except ImportError as e:
    raise ImportError("iec/_ops_binding.so is missing: build it with `make binding` or __graft_entry__.build()") from e

NONE, RELU, GELU, SIGMOID, SILU = range(5)
BLOCK = 128  # values along a row that share a scale

# The argument structs of iec_cuda.h, field by field.
GROUP_NORM = Struct("@P6n3P2nPnPnfii0P")
QUANTIZE = Struct("@P4nPnPni0P")
MATMUL = Struct("@PnPnPnPnPPnP4nii0P")

_DTYPE = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_F32, _FP8 = torch.float32, torch.float8_e4m3fn
_LEGACY_STREAM = 1  # cudaStreamLegacy: torch's default stream has the handle 0


def _bad(message: str):
    raise IecError(ERR_INPUT, message)


def _pack(layout, *values) -> bytes:
    """An argument struct."""
    try:
        return layout.pack(*values)
    except (StructError, OverflowError) as e:
        raise IecError(ERR_INPUT, f"an argument is no number of its type's range: {e}") from e


def _dtype(t, what: str) -> int:
    code = _DTYPE.get(t.dtype)
    if code is None:
        _bad(f"{what} is {t.dtype}: float16, bfloat16 or float32 are taken")
    return code


def _known(t, device: int, what: str):
    """Refuses a tensor of another device, or one whose gradient would be lost."""
    if t.get_device() != device:
        _bad(f"{what} is on {t.device}, the handle on cuda:{device}")
    if t.requires_grad and torch.is_grad_enabled():
        _bad(f"{what} requires a gradient, which the operators do not have: detach it or call under torch.no_grad()")


def _f32_vector(t, n: int, device: int, what: str) -> int:
    """The address of n contiguous floats, 0 for None."""
    if t is None:
        return 0
    _known(t, device, what)
    if t.dtype is not _F32 or t.shape != (n,) or (n > 1 and t.stride() != (1,)):
        _bad(f"{what} must be {n} contiguous float32 values")
    return t.data_ptr()


def _rows(t, shape, dtype, device: int, what: str) -> int:
    """The row stride of a matrix of `shape` whose rows are contiguous."""
    _known(t, device, what)
    if t.dtype is dtype and t.shape == shape:
        step, one = t.stride()
        if one == 1 or shape[1] <= 1:
            return step if shape[0] > 1 else max(shape[1], 1)
        _bad(f"{what} must have contiguous rows")
    _bad(f"{what} is {tuple(t.shape)} of {t.dtype}, not {tuple(shape)} of {dtype}")


def _maps(t, device: int, what: str):
    """(maps, pixels, channels, pixel stride, map stride) of n x ... x c."""
    _known(t, device, what)
    shape, stride = t.shape, t.stride()
    if len(shape) < 2:
        _bad(f"{what} must be maps x pixels (or height x width) x channels")
    n, c = shape[0], shape[-1]
    if c > 1 and stride[-1] != 1:
        _bad(f"{what} must have contiguous channels")
    pixels, step = 1, c
    for at in range(len(shape) - 2, 0, -1):
        size = shape[at]
        if size == 1:
            continue
        if pixels == 1:
            step = stride[at]
        elif stride[at] != step * pixels:
            _bad(f"{what} must have its pixels at one stride")
        pixels *= size
    return n, pixels, c, step, stride[0] if n > 1 else c


def _fp8_out(codes, scales, rows: int, k: int, scale_rows: int, device: int, stream):
    with _queued_on(stream, device):
        if codes is None:
            codes = empty_codes(rows, k, f"cuda:{device}")
        blocks = -(-k // BLOCK)
        if scales is None:
            scales = torch.empty((blocks, scale_rows), dtype=_F32, device=f"cuda:{device}")
    code_step = _rows(codes, (rows, k), _FP8, device, "codes")
    return codes, code_step, scales, _rows(scales, (blocks, scale_rows), _F32, device, "scales")


def _stream(stream, device: int) -> int:
    """`stream`, or torch's current one of the device."""
    if stream is None:
        stream = torch._C._cuda_getCurrentRawStream(device)
    return stream or _LEGACY_STREAM


def _queued_on(stream, device: int):
    """Makes `stream` torch's current one while outputs are allocated: memory
    that was just freed on torch's current stream may still be in use there,
    and what a call's kernels write must not be handed out again behind them."""
    if stream is None:
        return nullcontext()
    if stream in (0, _LEGACY_STREAM):
        return torch.cuda.stream(torch.cuda.default_stream(device))
    return torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device))


def empty_codes(rows: int, k: int, device):
    """Codes of a rows x k matrix as matmul_fp8 reads them: rows a multiple
    of 16 bytes apart."""
    return torch.empty((rows, -(-max(k, 1) // 16) * 16), dtype=_FP8, device=device)[:, :k]


class Ops:
    """A handle of one GPU for the operators (iec_ops in iec_cuda.h)."""

    def __init__(self, device: int = -1, timeout_ms: int = 0):
        L = lib()
        vp = ctypes.c_void_p
        L.iec_ops_device_name.restype = ctypes.c_char_p
        L.iec_ops_device_name.argtypes = [vp]
        L.iec_ops_free.argtypes = [vp]
        L.iec_ops_device.argtypes = [vp]
        L.iec_ops_sync.argtypes = [vp, vp]
        for f in (L.iec_ops_group_norm, L.iec_ops_group_norm_fp8, L.iec_ops_quantize_fp8, L.iec_ops_matmul_fp8):
            f.argtypes = [vp, ctypes.c_char_p, vp]
        self._lib = L
        self._h = vp()
        opt = Options(device, timeout_ms, 0)
        _check(L.iec_ops_open(ctypes.byref(opt), ctypes.byref(self._h)))
        self._device = L.iec_ops_device(self._h)
        self._handle = self._h.value  # for the binding; 0 once closed
        _fast.bind(*(ctypes.cast(f, vp).value for f in (L.iec_ops_group_norm, L.iec_ops_group_norm_fp8,
                                                        L.iec_ops_quantize_fp8, L.iec_ops_matmul_fp8)))

    def close(self):
        if getattr(self, "_h", None):
            self._handle = 0
            self._lib.iec_ops_free(self._h)
            self._h = None

    __del__ = close

    def gpu(self) -> str:
        """The device's name."""
        return self._lib.iec_ops_device_name(self._h).decode()

    def sync(self, stream=None):
        """Wait (bounded) for the stream's work and raise what went wrong."""
        _check(self._lib.iec_ops_sync(self._h, _stream(stream, self._device)))

    def group_norm(self, x, groups: int, gamma=None, beta=None, eps: float = 1e-5, act: int = NONE, out=None,
                   stream=None):
        """Group normalisation and activation of channels-last maps (n, ...,
        c); `out` (default: a new tensor) may be `x`."""
        if out is not None:
            status = _fast.group_norm(self._handle, self._device, stream, x, groups, gamma, beta, eps, act, out)
            if status == 0:
                return out
            if status > 0:
                _check(status)
        dtype = _dtype(x, "x")
        n, pixels, c, step, map_step = _maps(x, self._device, "x")
        if out is None:
            with _queued_on(stream, self._device):
                out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        elif out.dtype is not x.dtype or out.shape != x.shape:
            _bad("out must have the shape and type of x")
        _, _, _, out_step, out_map_step = _maps(out, self._device, "out")
        args = _pack(GROUP_NORM, x.data_ptr(), n, pixels, c, step, map_step, groups, _f32_vector(gamma, c, self._device, "gamma"),
                               _f32_vector(beta, c, self._device, "beta"), out.data_ptr(), out_step, out_map_step, 0, 0, 0, 0, eps,
                               dtype, act)
        status = self._lib.iec_ops_group_norm(self._h, args, _stream(stream, self._device))
        if status:
            _check(status)
        return out

    def group_norm_fp8(self, x, groups: int, gamma=None, beta=None, eps: float = 1e-5, act: int = NONE, codes=None,
                       scales=None, stream=None):
        """group_norm with its result as 8-bit rows, one per pixel: (codes
        n*pixels x c, scales ceil(c / 128) x n*pixels)."""
        if codes is not None and scales is not None:
            status = _fast.group_norm_fp8(self._handle, self._device, stream, x, groups, gamma, beta, eps, act, codes,
                                          scales)
            if status == 0:
                return codes, scales
            if status > 0:
                _check(status)
        dtype = _dtype(x, "x")
        n, pixels, c, step, map_step = _maps(x, self._device, "x")
        codes, code_step, scales, scale_step = _fp8_out(codes, scales, n * pixels, c, n * pixels, self._device,
                                                     stream)
        args = _pack(GROUP_NORM, x.data_ptr(), n, pixels, c, step, map_step, groups, _f32_vector(gamma, c, self._device, "gamma"),
                               _f32_vector(beta, c, self._device, "beta"), 0, 0, 0, codes.data_ptr(), code_step, scales.data_ptr(),
                               scale_step, eps, dtype, act)
        status = self._lib.iec_ops_group_norm_fp8(self._h, args, _stream(stream, self._device))
        if status:
            _check(status)
        return codes, scales

    def quantize_fp8(self, x, block_rows: int = 1, codes=None, scales=None, stream=None):
        """A rows x k matrix as 8-bit rows: (codes rows x k, scales
        ceil(k / 128) x rows), with block_rows 128 (weights) scales
        ceil(k / 128) x ceil(rows / 128)."""
        if codes is not None and scales is not None:
            status = _fast.quantize_fp8(self._handle, self._device, stream, x, block_rows, codes, scales)
            if status == 0:
                return codes, scales
            if status > 0:
                _check(status)
        dtype = _dtype(x, "x")
        shape = x.shape
        if len(shape) != 2:
            _bad("x must be rows x values")
        rows, k = shape
        step = _rows(x, shape, x.dtype, self._device, "x")
        scale_rows = rows if block_rows != BLOCK else -(-rows // BLOCK)
        codes, code_step, scales, scale_step = _fp8_out(codes, scales, rows, k, scale_rows, self._device, stream)
        args = _pack(QUANTIZE, x.data_ptr(), rows, k, step, block_rows, codes.data_ptr(), code_step, scales.data_ptr(),
                             scale_step, dtype)
        status = self._lib.iec_ops_quantize_fp8(self._h, args, _stream(stream, self._device))
        if status:
            _check(status)
        return codes, scales

    def matmul_fp8(self, a, a_scales, w, w_scales, bias=None, act: int = NONE, residual=None, out=None,
                   dtype=torch.float16, stream=None):
        """act(a w^T + bias) + residual for 8-bit rows a (m x k) and w (n x
        k, quantised with block_rows 128); `out` (default: a new tensor of
        `dtype`) may be `residual`."""
        if out is not None:
            status = _fast.matmul_fp8(self._handle, self._device, stream, a, a_scales, w, w_scales, bias, act, residual,
                                      out)
            if status == 0:
                return out
            if status > 0:
                _check(status)
        a_shape, w_shape = a.shape, w.shape
        if len(a_shape) != 2 or len(w_shape) != 2:
            _bad("a and w must be matrices")
        m, k = a_shape
        n, dev = w_shape[0], self._device
        blocks = -(-k // BLOCK)
        if out is None:
            with _queued_on(stream, self._device):
                out = torch.empty((m, n), dtype=dtype, device=a.device)
        code = _dtype(out, "out")
        res, res_step = 0, 0
        if residual is not None:
            res, res_step = residual.data_ptr(), _rows(residual, (m, n), out.dtype, dev, "residual")
        args = _pack(MATMUL, a.data_ptr(), _rows(a, a_shape, _FP8, dev, "a"),
                           a_scales.data_ptr(), _rows(a_scales, (blocks, m), _F32, dev, "a_scales"),
                           w.data_ptr(), _rows(w, (n, k), _FP8, dev, "w"),
                           w_scales.data_ptr(), _rows(w_scales, (blocks, -(-n // BLOCK)), _F32, dev, "w_scales"),
                           _f32_vector(bias, n, self._device, "bias"), res, res_step,
                           out.data_ptr(), _rows(out, (m, n), out.dtype, dev, "out"), m, n, k, act, code)
        status = self._lib.iec_ops_matmul_fp8(self._h, args, _stream(stream, self._device))
        if status:
            _check(status)
        return out
