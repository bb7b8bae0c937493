"""The operators run together as a network uses them (GPU test): the example
block against the same block in 64 bits without quantisation.

Four operands are rounded to e4m3 (both layers' rows and weights), each value
by up to 2^-4 of itself, evenly spread: 2^-4 / sqrt(3) in the mean square.
They are independent, so the added part may be off by twice that, 7.3 %."""

import importlib.util
import os

import pytest

from conftest import PKG

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,h,w,c,hidden,groups", [(2, 16, 24, 256, 512, 32), (1, 7, 5, 96, 384, 8), (1, 64, 64, 512, 2048, 32)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_pointwise_block(n, h, w, c, hidden, groups, dtype):
    import torch

    from iec.ops import Ops

    spec = importlib.util.spec_from_file_location("pointwise_block", os.path.join(PKG, "examples", "pointwise_block.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    ops = Ops()
    params = example.parameters(c, hidden, seed=c)
    block = example.PointwiseBlock(ops, groups, *params)
    g = torch.Generator(device="cuda")
    g.manual_seed(h)
    x = (torch.randn(n, h, w, c, generator=g, device="cuda") * 2 + 1).to(getattr(torch, dtype))
    want = example.reference(x.double(), groups, *[p.double() for p in params])
    # the result itself is rounded to the type of x, up to 2^-8 of it
    rounding = 2.0 ** -8 * want.norm() / (want - x.double()).norm() if dtype == "bfloat16" else 0.0
    off = (block(x).double() - want).norm() / (want - x.double()).norm()
    assert off <= 2 * 2.0 ** -4 / 3 ** 0.5 + rounding, off.item()
    ops.close()
