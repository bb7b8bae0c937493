"""Calls from a thread whose current CUDA context is not the device's primary
one, as a program that uses the driver API has it (GPU test)."""

import pytest

pytestmark = pytest.mark.gpu


def test_a_call_under_another_context_of_the_device():
    import torch

    driver = pytest.importorskip("cuda.bindings.driver")
    from iec.ops import Ops

    ops = Ops()
    x = torch.randn(1, 300, 64, device="cuda").half()
    out = torch.empty_like(x)
    want = ops.group_norm(x, 8)
    torch.cuda.synchronize()
    err, primary = driver.cuCtxGetCurrent()
    assert err == driver.CUresult.CUDA_SUCCESS
    err, device = driver.cuDeviceGet(0)
    assert err == driver.CUresult.CUDA_SUCCESS
    err, other = driver.cuCtxCreate(0, device)
    assert err == driver.CUresult.CUDA_SUCCESS
    try:
        err, now = driver.cuCtxGetCurrent()
        assert int(now) == int(other) != int(primary)
        ops.group_norm(x, 8, out=out)
        ops.sync()
    finally:
        driver.cuCtxSetCurrent(primary)
        driver.cuCtxDestroy(other)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    ops.close()
