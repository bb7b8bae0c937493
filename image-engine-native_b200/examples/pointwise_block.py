"""A residual block of pointwise layers over channels-last maps, in 8-bit
floating point:

    y = x + W2 gelu(W1 silu(group_norm(x)) + b1) + b2

The normalised, activated map is written as 8-bit rows and never in 16 bits;
the first layer reads them, its result is quantised, and the second layer
adds the map back. Weights are quantised once. Run it to see the block's
time and its distance from the same block in 32 bits:

    python image-engine-native_b200/examples/pointwise_block.py
"""

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from iec import ops as O  # noqa: E402


class PointwiseBlock:
    """`w1` hidden x c, `w2` c x hidden, `gamma`, `beta`, `b2` c values, `b1`
    hidden values: float32 CUDA tensors."""

    def __init__(self, ops: O.Ops, groups: int, gamma, beta, w1, b1, w2, b2, eps: float = 1e-5):
        self.ops, self.groups, self.eps = ops, groups, eps
        self.gamma, self.beta, self.b1, self.b2 = gamma, beta, b1, b2
        self.w1, self.w2 = ops.quantize_fp8(w1, block_rows=128), ops.quantize_fp8(w2, block_rows=128)

    def __call__(self, x):
        """x: n x h x w x c, float16 or bfloat16, contiguous."""
        ops = self.ops
        rows = x.reshape(-1, x.shape[-1])
        normed = ops.group_norm_fp8(x, self.groups, self.gamma, self.beta, self.eps, O.SILU)
        hidden = ops.matmul_fp8(*normed, *self.w1, self.b1, O.GELU, dtype=x.dtype)
        out = ops.matmul_fp8(*ops.quantize_fp8(hidden), *self.w2, self.b2, residual=rows, dtype=x.dtype)
        return out.reshape(x.shape)


def reference(x, groups, gamma, beta, w1, b1, w2, b2, eps=1e-5):
    """The same block without quantisation, in the type of x."""
    n, h, w, c = x.shape
    v = x.reshape(n, h * w, groups, c // groups)
    v = v - v.mean((1, 3), keepdim=True)
    v = v / ((v * v).mean((1, 3), keepdim=True) + eps).sqrt()
    v = v.reshape(x.shape) * gamma + beta
    v = v * torch.sigmoid(v)
    v = torch.nn.functional.gelu(v @ w1.T + b1)
    return x + v @ w2.T + b2


def parameters(c: int, hidden: int, seed: int = 0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    return [1 + 0.2 * randn(c), 0.2 * randn(c), randn(hidden, c) / c ** 0.5, 0.1 * randn(hidden),
            randn(c, hidden) / hidden ** 0.5, 0.1 * randn(c)]


def main():
    ops = O.Ops()
    n, side, c, hidden, groups = 4, 64, 512, 2048, 32
    params = parameters(c, hidden)
    block = PointwiseBlock(ops, groups, *params)
    x = torch.randn(n, side, side, c, device="cuda").half()
    y = block(x)
    want = reference(x.double(), groups, *[p.double() for p in params])
    err = ((y.double() - want).norm() / (want - x.double()).norm()).item()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for _ in range(5):
        block(x)
    start.record()
    for _ in range(50):
        block(x)
    end.record()
    ops.sync()
    print(f"{ops.gpu()}: {n} x {side} x {side} x {c}, hidden {hidden}: {start.elapsed_time(end) / 50 * 1e3:.1f} us, "
          f"relative error of the added part {err:.3f}")


if __name__ == "__main__":
    main()
