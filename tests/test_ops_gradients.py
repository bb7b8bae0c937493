"""The single operators have no gradients and say so, instead of returning
results without history."""

import pytest


def calls(ops, x, codes, scales, w, w_scales, bias, residual, outputs):
    """Every tensor of values that may require a gradient, in every call;
    `outputs`: with all outputs given, as the compiled binding takes them."""
    import torch

    fp8 = torch.float8_e4m3fn
    n, c = x.shape[0] * x.shape[1], x.shape[2]
    gamma = torch.ones(c, device=x.device)
    q = dict(codes=torch.zeros((n, c), device=x.device).to(fp8), scales=torch.ones((1, n), device=x.device)) if outputs else {}
    out = dict(out=torch.empty_like(x)) if outputs else {}
    y = dict(out=torch.empty_like(residual)) if outputs else {}
    kw = {} if outputs else dict(dtype=residual.dtype)
    rows = x[0]
    qr = dict(codes=q["codes"][: rows.shape[0]], scales=q["scales"][:, : rows.shape[0]]) if outputs else {}
    return {
        "x": [lambda t: ops.group_norm(t, 4, **out), lambda t: ops.group_norm_fp8(t, 4, **q),
              lambda t: ops.quantize_fp8(t[0], **qr)], "x_value": x,
        "gamma": [lambda t: ops.group_norm(x, 4, t, None, **out), lambda t: ops.group_norm_fp8(x, 4, t, None, **q)],
        "gamma_value": gamma,
        "beta": [lambda t: ops.group_norm(x, 4, gamma, t, **out), lambda t: ops.group_norm_fp8(x, 4, gamma, t, **q)],
        "beta_value": gamma,
        "scales": [lambda t: ops.matmul_fp8(codes, t, w, w_scales, **y, **kw)], "scales_value": scales,
        "bias": [lambda t: ops.matmul_fp8(codes, scales, w, w_scales, t, **y, **kw)], "bias_value": bias,
        "residual": [lambda t: ops.matmul_fp8(codes, scales, w, w_scales, bias, 0, t, **y, **kw)], "residual_value": residual,
    }


NAMES = ["x", "gamma", "beta", "scales", "bias", "residual"]


def check(ops, device, name, outputs):
    import torch

    import iec

    fp8 = torch.float8_e4m3fn
    c, m, n = 32, 8, 16
    args = dict(x=torch.randn(2, 4, c, device=device), codes=torch.zeros((m, c), device=device).to(fp8),
                scales=torch.ones((1, m), device=device), w=torch.zeros((n, c), device=device).to(fp8),
                w_scales=torch.ones((1, 1), device=device), bias=torch.zeros(n, device=device),
                residual=torch.zeros((m, n), device=device), outputs=outputs)
    table = calls(ops, **args)
    value = table[name + "_value"]
    for call in table[name]:
        needs = value.clone().requires_grad_()
        with pytest.raises(iec.IecError) as e:
            call(needs)
        assert e.value.code == iec.ERR_INPUT and "gradient" in str(e.value) and "no_grad" in str(e.value)
        with torch.no_grad():
            call(needs)
        call(needs.detach())


@pytest.mark.parametrize("name", NAMES)
def test_inputs_that_require_a_gradient_are_refused(name):
    """The checks of iec/ops.py, on CPU tensors and a library that does
    nothing."""
    from types import SimpleNamespace

    import torch

    from iec import ops as O

    o = object.__new__(O.Ops)
    o._h, o._handle, o._device = None, 0, -1
    o._lib = SimpleNamespace(**{f"iec_ops_{n}": lambda h, args, s: 0
                                for n in ("group_norm", "group_norm_fp8", "quantize_fp8", "matmul_fp8")})
    stream, empty = O._stream, torch.empty
    try:
        O._stream = lambda s, d: 0
        torch.empty = lambda shape, dtype=None, device=None: empty(shape, dtype=dtype)
        check(o, "cpu", name, False)
    finally:
        O._stream, torch.empty = stream, empty


@pytest.mark.gpu
@pytest.mark.parametrize("outputs", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_the_binding_refuses_them_too(name, outputs):
    from iec.ops import Ops

    ops = Ops()
    check(ops, "cuda", name, outputs)
    ops.close()
