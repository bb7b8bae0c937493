"""The single operators' entry points on the CPU: exported, refusing without
a GPU, and refusing handles that are not theirs before anything is read."""

import ctypes

import pytest


def test_no_gpu_is_a_gpu_error():
    import iec
    from iec import ops

    if iec.device_count() > 0:
        pytest.skip("a GPU is present")
    with pytest.raises(iec.IecError) as e:
        ops.Ops()
    assert e.value.code == iec.ERR_GPU
    assert "no CUDA device" in str(e.value)


def test_null_and_foreign_handles_are_input_errors():
    import iec

    L = iec.lib()
    assert L.iec_ops_open(None, None) == iec.ERR_INPUT
    assert L.iec_ops_sync(None, None) == iec.ERR_INPUT
    assert b"null" in L.iec_last_error()
    foreign = ctypes.create_string_buffer(64)
    assert L.iec_ops_sync(foreign, None) == iec.ERR_INPUT
    assert b"not a handle" in L.iec_last_error()
    L.iec_ops_free(None)
    L.iec_ops_free(foreign)


def test_tensor_views():
    """Which strides count as maps of pixels and as rows."""
    import torch

    import iec
    from iec import ops

    t = torch.zeros(2, 5, 7, 24)
    assert ops._maps(t, -1, "t") == (2, 35, 24, 24, 35 * 24)
    assert ops._maps(t[..., :10], -1, "t") == (2, 35, 10, 24, 35 * 24)
    assert ops._maps(t[:1], -1, "t")[:4] == (1, 35, 24, 24)
    assert ops._maps(t[:, :, :1], -1, "t") == (2, 5, 24, 7 * 24, 35 * 24)
    assert ops._maps(t[:, :1, :1], -1, "t")[:3] == (2, 1, 24)
    for bad in (t[:, :, ::2], t[:, :, :4], t.transpose(1, 2), t.transpose(2, 3), torch.zeros(4)):
        with pytest.raises(iec.IecError):
            ops._maps(bad, -1, "t")
    with pytest.raises(iec.IecError) as e:  # -1 is the device of CPU tensors
        ops._maps(t, 0, "t")
    assert "cpu" in str(e.value)
    codes = ops.empty_codes(3, 50, "cpu")
    assert codes.shape == (3, 50) and codes.stride(0) == 64
    assert ops._rows(codes, (3, 50), torch.float8_e4m3fn, -1, "codes") == 64
    with pytest.raises(iec.IecError):
        ops._rows(codes.t(), (50, 3), torch.float8_e4m3fn, -1, "codes")


def test_binding_leaves_what_does_not_fit():
    """The compiled fast path calls nothing for tensors of another device, of
    other shapes or types, or for missing arguments: it answers -1."""
    import torch

    from iec import _ops_binding as fast

    x = torch.zeros(2, 16)
    assert fast.quantize_fp8(0, 0, 5, x, 1, x, x) == -1
    assert fast.quantize_fp8(0, 0, 5, None, 1, x, x) == -1
    assert fast.quantize_fp8(0) == -1
    assert fast.group_norm(0, 0, 5, x, 1, None, None, 1e-5, 0, x) == -1
    assert fast.group_norm_fp8(0, 0, 5, x, 1, None, None, 1e-5, 0, x, x) == -1
    assert fast.matmul_fp8(0, 0, 5, x, x, x, x, None, 0, None, x) == -1
    assert fast.matmul_fp8("no handle", 0, 5, x, x, x, x, None, 0, None, x) == -1
