"""The single operators on streams other than torch's current one: whose
memory the outputs are that a call allocates."""

from contextlib import contextmanager
from types import SimpleNamespace

import pytest


@pytest.fixture
def recorded(monkeypatch):
    """An Ops on CPU tensors with a library that does nothing, and the stream
    that was torch's current one at each allocation."""
    import torch

    from iec import ops as O

    current, seen = [None], []
    empty = torch.empty

    @contextmanager
    def stream(s):
        before, current[0] = current[0], s
        yield
        current[0] = before

    def recording_empty(shape, dtype=None, device=None):
        seen.append(current[0])
        return empty(shape, dtype=dtype)

    monkeypatch.setattr(torch, "empty", recording_empty)
    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda ptr, device=None: ("external", ptr, device))
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: ("default", device))
    o = object.__new__(O.Ops)
    o._h, o._handle, o._device = None, 0, -1
    o._lib = SimpleNamespace(**{f"iec_ops_{n}": lambda h, args, s: 0
                                for n in ("group_norm", "group_norm_fp8", "quantize_fp8", "matmul_fp8")})
    return o, seen


def calls(o):
    import torch

    x = torch.zeros(2, 4, 32)
    codes, scales = torch.zeros(5, 32).to(torch.float8_e4m3fn), torch.ones(1, 5)
    w, w_scales = torch.zeros(3, 32).to(torch.float8_e4m3fn), torch.ones(1, 1)
    return {
        "group_norm": (1, lambda **k: o.group_norm(x, 4, **k)),
        "group_norm_fp8": (2, lambda **k: o.group_norm_fp8(x, 4, **k)),
        "group_norm_fp8, codes given": (1, lambda **k: o.group_norm_fp8(x, 4, codes=torch.zeros(8, 32).to(torch.float8_e4m3fn), **k)),
        "quantize_fp8": (2, lambda **k: o.quantize_fp8(x[0], **k)),
        "matmul_fp8": (1, lambda **k: o.matmul_fp8(codes, scales, w, w_scales, **k)),
    }


NAMES = ["group_norm", "group_norm_fp8", "group_norm_fp8, codes given", "quantize_fp8", "matmul_fp8"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("stream,want", [(77, ("external", 77, -1)), (0, ("default", -1)), (1, ("default", -1))])
def test_outputs_belong_to_the_stream_of_the_call(recorded, name, stream, want):
    o, seen = recorded
    outputs, call = calls(o)[name]
    call(stream=stream)
    assert seen == [want] * outputs


@pytest.mark.parametrize("name", NAMES)
def test_outputs_belong_to_the_current_stream_by_default(recorded, monkeypatch, name):
    import torch

    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 0, raising=False)
    o, seen = recorded
    outputs, call = calls(o)[name]
    call()
    assert seen == [None] * outputs


@pytest.mark.gpu
def test_memory_freed_on_the_current_stream_is_not_handed_out():
    """A block just freed on torch's current stream may still be written there;
    a call on another stream gets one of that stream's."""
    import torch

    from iec.ops import Ops

    ops, side = Ops(), torch.cuda.Stream()
    x = torch.randn(4096, 1024, device="cuda").half()
    want, want_scales = ops.quantize_fp8(x)
    w, w_scales = ops.quantize_fp8(x[:1024], 128)
    y = ops.matmul_fp8(want, want_scales, w, w_scales)
    torch.cuda.synchronize()

    def freed(shape, dtype):
        """Addresses of blocks that the current stream has free."""
        some = [torch.empty(shape, dtype=dtype, device="cuda") for _ in range(8)]
        return {t.data_ptr() for t in some}

    taken = freed((4096, 1024), torch.uint8) | freed((8, 4096), torch.float32)
    codes, scales = ops.quantize_fp8(x, stream=side.cuda_stream)
    assert codes.data_ptr() not in taken and scales.data_ptr() not in taken
    taken = freed((4096, 1024), torch.float16)
    out = ops.matmul_fp8(codes, scales, w, w_scales, stream=side.cuda_stream)
    normed = ops.group_norm(x[None], 32, stream=side.cuda_stream)
    assert out.data_ptr() not in taken and normed.data_ptr() not in taken
    ops.sync(side.cuda_stream)
    assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales, want_scales)
    assert torch.equal(out, y) and torch.equal(normed, ops.group_norm(x[None], 32))
    ops.close()
