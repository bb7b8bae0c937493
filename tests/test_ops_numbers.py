"""Numbers that do not fit the operators' argument structs are input errors
like any other wrong argument."""

from types import SimpleNamespace

import pytest


def wrong(ops, device):
    import torch

    x = torch.zeros((2, 4, 48), device=device)
    rows = torch.zeros((6, 32), device=device)
    a, w = (torch.zeros((r, 32), device=device).to(torch.float8_e4m3fn) for r in (6, 8))
    sa, sw = torch.ones((1, 6), device=device), torch.ones((1, 1), device=device)
    y = torch.empty((6, 8), device=device)
    return {
        "eps beyond f32": lambda **k: ops.group_norm(x, 4, eps=1e40, **k),
        "act beyond int": lambda **k: ops.group_norm(x, 4, act=1 << 40, **k),
        "act by name": lambda **k: ops.group_norm(x, 4, act="silu", **k),
        "groups beyond size_t": lambda **k: ops.group_norm(x, 1 << 70, **k),
        "groups as a float": lambda **k: ops.group_norm(x, 4.0, **k),
        "8-bit rows, eps": lambda **k: ops.group_norm_fp8(x, 4, eps=-1e300),
        "block_rows beyond size_t": lambda **k: ops.quantize_fp8(rows, -(1 << 80)),
        "product, act": lambda **k: ops.matmul_fp8(a, sa, w, sw, act=-(1 << 33), **({"out": y} if k else {"dtype": y.dtype})),
    }


NAMES = ["eps beyond f32", "act beyond int", "act by name", "groups beyond size_t", "groups as a float", "8-bit rows, eps",
         "block_rows beyond size_t", "product, act"]


def check(ops, device, name, **given):
    import iec

    with pytest.raises(iec.IecError) as e:
        wrong(ops, device)[name](**given)
    assert e.value.code == iec.ERR_INPUT


@pytest.mark.parametrize("name", [n for n in NAMES if "eps" not in n])  # the library sees those as infinite
def test_numbers_out_of_range_are_input_errors(monkeypatch, name):
    """iec/ops.py on CPU tensors; the library would accept everything."""
    import torch

    from iec import ops as O

    o = object.__new__(O.Ops)
    o._h, o._handle, o._device = None, 0, -1
    o._lib = SimpleNamespace(**{f"iec_ops_{n}": lambda h, args, s: 0
                                for n in ("group_norm", "group_norm_fp8", "quantize_fp8", "matmul_fp8")})
    empty = torch.empty
    monkeypatch.setattr(O, "_stream", lambda s, d: 0)
    monkeypatch.setattr(torch, "empty", lambda shape, dtype=None, device=None: empty(shape, dtype=dtype))
    check(o, "cpu", name)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_the_same_with_outputs_given(name):
    import torch

    from iec.ops import Ops

    ops = Ops()
    out = torch.empty((2, 4, 48), device="cuda")
    check(ops, "cuda", name)
    check(ops, "cuda", name, out=out)
    ops.close()
