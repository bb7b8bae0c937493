"""The single operators (group normalisation, e4m3 quantisation, the 8-bit
product) against their definitions in 64 bits (GPU tests).

Tolerances, u the output type's unit roundoff (2^-p for p significant
bits: 2^-11 f16, 2^-8 bf16, 2^-24 f32):
  norm     u |y| + 2^-19 (1 + |gamma| (|x| + |mean|) / sigma + |beta|): a few
           f32 roundings of x rstd gamma and of mean rstd gamma, statistics
           good to 2^-22, and an exponential good to 2^-21
  scales   2^-22 relative: one division of an exact maximum
  codes    the e4m3 value nearest to x 448 / amax, or its neighbour where
           that is within 2^-21 of half-way
  product  u |y| + 2^-16 S, S = sum over k of |a w| with the scales: a block's
           four tensor instructions each add 32 products and the running sum
           with at least 23 bits below the largest, 4 x 33 x 2^-23, about 2^-16
"""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

NONE, RELU, GELU, SIGMOID, SILU = range(5)
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
SMALL = {"f16": 2.0 ** -25, "bf16": 0.0, "f32": 0.0}  # half a subnormal step


@pytest.fixture(scope="module")
def ops():
    from iec.ops import Ops

    o = Ops()
    yield o
    o.close()


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def act64(v, act):
    if act == RELU:
        return torch.relu(v)
    if act == GELU:
        return 0.5 * v * torch.special.erfc(-v * 0.5 ** 0.5)
    if act == SIGMOID:
        return torch.sigmoid(v)
    if act == SILU:
        return v * torch.sigmoid(v)
    return v


def norm64(x, groups, gamma, beta, eps, act):
    """(y, tolerance of its f32 arithmetic) over x of n x pixels x c."""
    n, px, c = x.shape
    v = x.double().reshape(n, px, groups, c // groups)
    mean = v.mean((1, 3), keepdim=True)
    sigma = ((v - mean) ** 2).mean((1, 3), keepdim=True).add(eps).sqrt()
    y = ((v - mean) / sigma).reshape(n, px, c)
    size = ((v.abs() + mean.abs()) / sigma).reshape(n, px, c)
    if gamma is not None:
        y, size = y * gamma.double(), size * gamma.double().abs()
    if beta is not None:
        y, size = y + beta.double(), size + beta.double().abs()
    return act64(y, act), 2.0 ** -19 * (1 + size)


def e4m3_step(v):
    _, e = torch.frexp(v.abs())
    return torch.ldexp(torch.ones_like(v), torch.clamp_min(e - 1, -6) - 3)


def within(got, want, tol):
    err = (got.double() - want).abs()
    assert torch.isfinite(got.float()).all()
    worst = (err / tol).max().item()
    assert worst <= 1.0, worst


def check_codes(codes, scales, x, block_rows=1, slack=None):
    """codes, scales of x (rows x k, doubles); `slack`: how far each x may
    have been off before it was quantised."""
    rows, k = x.shape
    kb, rb = -(-k // 128), -(-rows // block_rows)
    full = torch.zeros(rb * block_rows, kb * 128, dtype=torch.float64, device=x.device)
    full[:rows, :k] = x.abs()
    amax = full.reshape(rb, block_rows, kb, 128).amax((1, 3))
    want = torch.where(amax < 2.0 ** -100, torch.ones_like(amax), amax / 448)
    each = want.repeat_interleave(block_rows, 0).repeat_interleave(128, 1)[:rows, :k]
    allowed = torch.zeros_like(x) if slack is None else slack
    top = torch.zeros_like(full)
    top[:rows, :k] = allowed
    top = top.reshape(rb, block_rows, kb, 128).amax((1, 3)) / 448
    assert scales.shape == (kb, rb)
    assert ((scales.t().double() - want).abs() <= 2.0 ** -22 * want + top).all()
    v = x / each
    err = (codes.double() - v).abs()
    moved = v.abs() * (top / want).repeat_interleave(block_rows, 0).repeat_interleave(128, 1)[:rows, :k]
    limit = e4m3_step(v) / 2 + 2.0 ** -21 * v.abs() + allowed / each + moved
    assert (err <= limit).all(), (err - limit).max().item()


NORMS = [
    # n, pixels, c, groups, pad, act, affine
    (1, 1, 32, 32, 0, NONE, True),       # one value a group: variance 0
    (1, 1, 512, 32, 0, SILU, True),
    (2, 7, 96, 8, 0, GELU, True),
    (3, 25, 293, 1, 0, SILU, False),     # odd channels
    (2, 33, 659, 1, 5, SIGMOID, True),
    (1, 130, 2, 2, 0, RELU, True),
    (4, 49, 320, 32, 40, RELU, True),    # groups of 10 channels, a slice
    (1, 1961, 814, 1, 8, NONE, True),
    (2, 961, 768, 32, 0, SILU, True),
    (9, 256, 512, 32, 0, SILU, True),
    (1, 4096, 64, 4, 0, GELU, True),
    (1, 70001, 128, 32, 0, SILU, True),
    (2, 16384, 520, 8, 24, SILU, True),
    (1, 300, 4096, 32, 0, SILU, True),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("n,pixels,c,groups,pad,act,affine", NORMS)
def test_group_norm(ops, n, pixels, c, groups, pad, act, affine, dtype):
    g = gen(n + pixels + c)
    x = (randn(g, n, pixels, c + pad) + randn(g, c + pad)).to(TYPES[dtype])[..., :c]
    gamma, beta = (1 + 0.3 * randn(g, c), 0.3 * randn(g, c)) if affine else (None, None)
    want, tol = norm64(x, groups, gamma, beta, 1e-5, act)
    got = ops.group_norm(x, groups, gamma, beta, 1e-5, act)
    assert got.shape == x.shape and got.dtype == x.dtype
    within(got, want, HALF[dtype] * want.abs() + SMALL[dtype] + tol)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("n,pixels,c,groups,pad,act,affine", NORMS)
def test_group_norm_fp8(ops, n, pixels, c, groups, pad, act, affine, dtype):
    g = gen(n + pixels + c + 1)
    x = (randn(g, n, pixels, c + pad) + randn(g, c + pad)).to(TYPES[dtype])[..., :c]
    gamma, beta = (1 + 0.3 * randn(g, c), 0.3 * randn(g, c)) if affine else (None, None)
    want, tol = norm64(x, groups, gamma, beta, 1e-5, act)
    codes, scales = ops.group_norm_fp8(x, groups, gamma, beta, 1e-5, act)
    check_codes(codes, scales, want.reshape(-1, c), slack=tol.reshape(-1, c))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("n,pixels,c,groups", [
    (1, 1024, 320, 32), (1, 1024, 960, 32), (2, 700, 768, 32), (1, 333, 992, 8),
    (1, 3, 1032, 3), (1, 1, 640, 32), (1, 90, 136, 17), (2, 500, 200, 8), (1, 2000, 416, 32),
    (1, 2304, 192, 6), (3, 400, 1000, 8), (1, 600, 1288, 7), (1, 64, 8184, 682), (1, 257, 264, 1)])
def test_group_norm_fp8_of_groups_across_blocks(ops, n, pixels, c, groups, dtype):
    """Groups that end inside the blocks of 128 channels, last blocks cut short."""
    g = gen(n + pixels + c + groups)
    wide = (randn(g, n, pixels, c + 8) + randn(g, c + 8)).to(TYPES[dtype])
    x = wide[..., :c]
    gamma, beta = 1 + 0.3 * randn(g, c), 0.3 * randn(g, c)
    want, tol = norm64(x, groups, gamma, beta, 1e-5, SILU)
    codes, scales = ops.group_norm_fp8(x, groups, gamma, beta, 1e-5, SILU)
    check_codes(codes, scales, want.reshape(-1, c), slack=tol.reshape(-1, c))
    again, same = ops.group_norm_fp8(x, groups, gamma, beta, 1e-5, SILU)
    assert torch.equal(codes.view(torch.uint8), again.view(torch.uint8)) and torch.equal(scales, same)
    # unaligned rows, the same bits
    odd = torch.empty(n, pixels, c + 1, device="cuda", dtype=x.dtype)[..., 1:]
    odd.copy_(x)
    into = torch.zeros((n * pixels, c + 3), device="cuda").to(torch.float8_e4m3fn)[:, 1:c + 1]
    _, same = ops.group_norm_fp8(odd, groups, gamma, beta, 1e-5, SILU, codes=into)
    assert torch.equal(codes.view(torch.uint8), into.view(torch.uint8)) and torch.equal(scales, same)


def test_group_norm_fp8_keeps_what_is_not_finite_within_its_group(ops):
    """Segments read their neighbours' channels; only the group's own count."""
    x = randn(gen(8), 1, 700, 320).half()
    x[0, 350, 125] = float("nan")  # group 12 of 10 channels, 120 to 129: both sides of a block's end
    codes, _ = ops.group_norm_fp8(x, 32)
    nan = torch.isnan(codes.float())  # through their scales, all of both blocks; none of the third
    assert nan[:, :256].all() and not nan[:, 256:].any()


@pytest.mark.parametrize("offset", [100.0, -3000.0])
def test_group_norm_keeps_its_digits_far_from_zero(ops, offset):
    """A mean thousands of deviations from zero: a variance from the mean of
    squares would be rounding noise."""
    x = offset + randn(gen(3), 2, 5000, 64)
    want, tol = norm64(x, 4, None, None, 1e-5, NONE)
    within(ops.group_norm(x, 4), want, tol)


def test_group_norm_of_constant_groups(ops):
    """Variance 0: beta through the activation, whatever the value."""
    x = torch.full((2, 50, 64), 3.25, device="cuda", dtype=torch.float16)
    beta = randn(gen(4), 64)
    got = ops.group_norm(x, 8, None, beta, 1e-5, SILU)
    want = act64(beta.double(), SILU).expand(2, 50, 64)
    within(got, want, 2.0 ** -11 * want.abs() + 2.0 ** -19)


@pytest.mark.parametrize("pixels", [9, 5000, 100000])
def test_group_norm_spreads_what_is_not_finite_within_its_group(ops, pixels):
    x = randn(gen(5), 2, pixels, 64).half()
    x[0, pixels // 2, 9] = float("nan")  # group 1 of 8 channels, map 0
    x[1, pixels - 1, 63] = float("inf")  # group 7, map 1
    got = ops.group_norm(x, 8)
    bad = torch.isnan(got).reshape(2, pixels, 8, 8).all(3).all(1)
    some = torch.isnan(got).reshape(2, pixels, 8, 8).any(3).any(1)
    want = torch.zeros(2, 8, dtype=torch.bool, device="cuda")
    want[0, 1] = want[1, 7] = True
    assert torch.equal(bad, want) and torch.equal(some, want)


@pytest.mark.parametrize("pixels,c", [(40, 96), (70000, 128)])
def test_group_norm_in_place_and_into_a_slice(ops, pixels, c):
    x = randn(gen(6), 2, pixels, c).half()
    want = ops.group_norm(x, 32, act=SILU)
    wide = torch.full((2, pixels, c + 24), 7.0, device="cuda", dtype=torch.float16)
    ops.group_norm(x, 32, act=SILU, out=wide[..., :c])
    assert torch.equal(wide[..., :c], want) and (wide[..., c:] == 7).all()
    ops.group_norm(x, 32, act=SILU, out=x)
    assert torch.equal(x, want)


def test_group_norm_takes_unaligned_maps(ops):
    """A tensor that starts 2 bytes past a vector's boundary."""
    base = randn(gen(7), 2 * 600 * 64 + 1).half()
    x = base[1:].reshape(2, 600, 64)
    assert torch.equal(ops.group_norm(x, 8, act=GELU), ops.group_norm(x.clone(), 8, act=GELU))


@pytest.mark.parametrize("pixels", [600, 60000])
@pytest.mark.parametrize("c", [64, 200])
def test_group_norm_fp8_takes_unaligned_maps(ops, pixels, c):
    """The same codes and scales from maps and into codes that start anywhere."""
    base = randn(gen(30), 2 * pixels * (c + 1) + 1).half()
    x = base[1:].reshape(2, pixels, c + 1)[..., :c]
    want, scales = ops.group_norm_fp8(x.clone(), 8, act=SILU)
    got = torch.zeros((2 * pixels, c + 3), device="cuda").to(torch.float8_e4m3fn)[:, 1:c + 1]
    _, other = ops.group_norm_fp8(x, 8, act=SILU, codes=got)
    assert torch.equal(got.view(torch.uint8), want.view(torch.uint8)) and torch.equal(other, scales)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("n,pixels,c,groups", [(1, 40, 5000, 4), (2, 300, 5001, 3), (1, 9, 30000, 6000), (3, 2, 65535, 15)])
def test_group_norm_of_many_channels(ops, n, pixels, c, groups, dtype):
    """Groups that straddle the kernels' tiles of channels."""
    g = gen(c)
    x = (randn(g, n, pixels, c) + randn(g, c)).to(TYPES[dtype])
    gamma, beta = 1 + 0.3 * randn(g, c), 0.3 * randn(g, c)
    want, tol = norm64(x, groups, gamma, beta, 1e-5, SILU)
    within(ops.group_norm(x, groups, gamma, beta, 1e-5, SILU), want, HALF[dtype] * want.abs() + SMALL[dtype] + tol)
    codes, scales = ops.group_norm_fp8(x, groups, gamma, beta, 1e-5, SILU)
    check_codes(codes, scales, want.reshape(-1, c), slack=tol.reshape(-1, c))


def test_group_norm_is_the_same_every_time(ops):
    x = randn(gen(8), 3, 9000, 128).half()
    first = ops.group_norm(x, 32, act=SILU)
    for _ in range(4):
        assert torch.equal(ops.group_norm(x, 32, act=SILU), first)


QUANTS = [(1, 1), (1, 16), (1, 2880), (3, 127), (7, 128), (22, 734), (130, 129), (129, 73), (300, 1000), (1000, 3545),
          (5000, 384)]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,k", QUANTS)
def test_quantize(ops, rows, k, block_rows, dtype):
    g = gen(rows + k)
    x = (randn(g, rows, k + 24) * torch.exp(randn(g, rows, 1))).to(TYPES[dtype])[:, :k]
    check_codes(*ops.quantize_fp8(x, block_rows), x.double(), block_rows)
    whole = x.contiguous()  # its rows may start anywhere
    check_codes(*ops.quantize_fp8(whole, block_rows), x.double(), block_rows)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("rows,k,block_rows", [(20000, 648, 1), (90001, 104, 1), (301, 1024, 1), (9000, 16, 1),
                                               (700, 648, 128), (129, 8, 128)])
def test_quantize_takes_rows_that_start_anywhere(ops, rows, k, block_rows, dtype):
    """The same codes and scales as from aligned rows, also of what is not
    finite, and into codes that start anywhere."""
    base = randn(gen(rows + k), rows, k + 1).to(TYPES[dtype])
    base[rows // 2, 3] = float("inf")
    base[rows - 1, k] = float("nan")
    base[0] = 0
    x = base[:, 1:]
    want, want_scales = ops.quantize_fp8(x.contiguous(), block_rows)
    got, scales = ops.quantize_fp8(x, block_rows)
    assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))
    assert torch.equal(scales.view(torch.int32), want_scales.view(torch.int32))
    wide = torch.zeros((rows, k + 3), device="cuda").to(torch.float8_e4m3fn)
    ops.quantize_fp8(x, block_rows, codes=wide[:, 1:k + 1])
    assert torch.equal(wide[:, 1:k + 1].view(torch.uint8), want.view(torch.uint8))
    assert (wide[:, 0].float() == 0).all() and (wide[:, k + 1:].float() == 0).all()


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_zeros_and_extremes(ops, block_rows):
    x = torch.zeros(5, 512, device="cuda")
    x[1, :128] = 2.0 ** -101  # below the least kept magnitude
    x[1, 128:256] = 2.0 ** -99
    x[2, 300] = 3.0e38
    x[3, 500] = float("inf")
    x[3, 390:400] = 1.0
    if block_rows == 1:
        x[4, 5] = float("nan")
        x[4, 6] = 1.0
    codes, scales = ops.quantize_fp8(x, block_rows)
    back = codes.float() * scales.t().repeat_interleave(block_rows, 0)[:5].repeat_interleave(128, 1)
    if block_rows == 1:
        assert (back[0] == 0).all() and (scales[:, 0] == 1).all()
        assert (back[1, :128] == 0).all() and (codes[1, 128:256].float() == 448).all()
        assert (back[1, 256:] == 0).all()
        assert torch.isnan(back[4, :128]).all() and (back[4, 128:] == 0).all()
        assert torch.isnan(back[3, 384:]).all() and (back[3, :384] == 0).all()
    else:
        assert (codes[1, 128:256].float() == 448).all()
        assert torch.isnan(back[:, 384:]).all()
    assert codes[2, 300].float() == 448 and abs(back[2, 300].item() / 3.0e38 - 1) < 1e-6


def operands(ops, g, m, n, k):
    a = randn(g, m, k) * torch.exp(randn(g, m, 1))
    w = randn(g, n, k)
    return ops.quantize_fp8(a), ops.quantize_fp8(w, 128)


def product64(a, sa, w, sw):
    """(a w^T, sum of magnitudes) in 64 bits."""
    n, k = w.shape
    x = a.double() * sa.t().double().repeat_interleave(128, 1)[:, :k]
    y = w.double() * sw.t().double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return x @ y.t(), x.abs() @ y.abs().t()


PRODUCTS = [
    # m, n, k
    (1, 1, 1), (1, 1, 16), (1, 4096, 4096), (1, 100, 1656), (2, 128, 128), (3, 777, 130), (8, 64, 960), (15, 33, 127),
    (16, 256, 384), (17, 129, 129), (31, 1059, 192), (33, 500, 2048), (64, 512, 512), (65, 136, 4000), (100, 39, 65),
    (127, 255, 256), (128, 128, 128), (129, 257, 385), (200, 1536, 384), (344, 159, 1317), (512, 512, 512),
    (1111, 777, 1000), (2048, 384, 1536), (4096, 1536, 384), (5000, 2050, 96),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_matmul(ops, m, n, k, dtype):
    g = gen(m + n + k)
    (a, sa), (w, sw) = operands(ops, g, m, n, k)
    want, size = product64(a, sa, w, sw)
    got = ops.matmul_fp8(a, sa, w, sw, dtype=TYPES[dtype])
    within(got, want, HALF[dtype] * want.abs() + SMALL[dtype] + 2.0 ** -16 * size)


@pytest.mark.parametrize("m,n,k", [(1, 200, 300), (20, 777, 512), (300, 136, 200), (1111, 777, 1000)])
@pytest.mark.parametrize("act", [NONE, RELU, GELU, SIGMOID, SILU])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_matmul_epilogue(ops, m, n, k, act, dtype):
    """Bias, activation (each with slope at most 1.13) and residual, the
    residual read from the output itself and from a wider matrix."""
    g = gen(m * 3 + act)
    (a, sa), (w, sw) = operands(ops, g, m, n, k)
    sa *= 0.1
    bias, res = randn(g, n), randn(g, m, n + 3).to(TYPES[dtype])[:, :n]
    raw, size = product64(a, sa, w, sw)
    v = act64(raw + bias.double(), act)
    want = v + res.double()
    tol = HALF[dtype] * want.abs() + SMALL[dtype] + 1.13 * 2.0 ** -16 * (size + bias.abs().double()) + 2.0 ** -19
    got = ops.matmul_fp8(a, sa, w, sw, bias, act, res, dtype=TYPES[dtype])
    within(got, want, tol)
    out = res.contiguous().clone()
    ops.matmul_fp8(a, sa, w, sw, bias, act, out, out=out)
    assert torch.equal(out, got)
    wide = torch.full((m, n + 5), 7.0, device="cuda", dtype=TYPES[dtype])
    ops.matmul_fp8(a, sa, w, sw, bias, act, res, out=wide[:, :n])
    assert torch.equal(wide[:, :n], got) and (wide[:, n:] == 7).all()


@pytest.mark.parametrize("m,n,k", [(4, 512, 4096), (1024, 512, 4096)])
def test_matmul_sums_in_32_bits(ops, m, n, k):
    """An f32 result of a long reduction is good to 2^-20 of its norm."""
    (a, sa), (w, sw) = operands(ops, gen(11), m, n, k)
    want, _ = product64(a, sa, w, sw)
    got = ops.matmul_fp8(a, sa, w, sw, dtype=torch.float32).double()
    assert ((got - want).norm() / want.norm()).item() <= 2.0 ** -20


@pytest.mark.parametrize("m", [3, 300])
def test_matmul_keeps_what_is_not_finite_in_its_rows(ops, m):
    x = randn(gen(12), m, 300).half()
    x[1, 200] = float("nan")
    x[2, 10] = float("inf")
    x[0] = 0
    a, sa = ops.quantize_fp8(x)
    w, sw = ops.quantize_fp8(randn(gen(13), 200, 300), 128)
    bad = torch.isnan(ops.matmul_fp8(a, sa, w, sw))
    want = torch.zeros(m, 200, dtype=torch.bool, device="cuda")
    want[1] = want[2] = True
    assert torch.equal(bad, want)
    assert (ops.matmul_fp8(a, sa, w, sw)[0] == 0).all()


@pytest.mark.parametrize("m,n,k", [(5, 300, 700), (700, 300, 700)])
def test_matmul_of_strided_operands(ops, m, n, k):
    """Operands and scales that are slices of wider ones give the same."""
    (a, sa), (w, sw) = operands(ops, gen(14), m, n, k)
    want = ops.matmul_fp8(a, sa, w, sw)

    def slice_of(t, more, off):
        wide = torch.zeros((t.shape[0], -(-t.shape[1] // 16) * 16 + more), dtype=torch.float32, device="cuda").to(t.dtype)
        part = wide[:, off:off + t.shape[1]]
        part.copy_(t)
        return part

    got = ops.matmul_fp8(slice_of(a, 64, 16), slice_of(sa, 5, 2), slice_of(w, 32, 0), slice_of(sw, 3, 1))
    assert torch.equal(got, want)


def test_no_rows_and_no_values(ops):
    """Sizes of zero: nothing is written, nothing is read."""
    half = dict(device="cuda", dtype=torch.float16)
    for n, px in [(0, 5), (5, 0)]:
        x = torch.empty((n, px, 32), **half)
        assert ops.group_norm(x, 4).shape == (n, px, 32)
        codes, scales = ops.group_norm_fp8(x, 4)
        assert codes.shape == (0, 32) and scales.shape == (1, 0)
    for rows, k in [(0, 40), (4, 0)]:
        codes, scales = ops.quantize_fp8(torch.empty((rows, k), **half))
        assert codes.shape == (rows, k)
    (a, sa), (w, sw) = operands(ops, gen(15), 6, 40, 64)
    assert ops.matmul_fp8(a[:0], sa[:, :0], w, sw).shape == (0, 40)
    assert ops.matmul_fp8(a, sa, w[:0], sw[:, :0]).shape == (6, 0)
    bias, res = randn(gen(16), 40), randn(gen(17), 6, 40).half()
    got = ops.matmul_fp8(a[:, :0], sa[:0], w[:, :0], sw[:0], bias, RELU, res)
    want = torch.relu(bias.double()) + res.double()
    within(got, want, 2.0 ** -10 * want.abs() + 2.0 ** -25)


def test_other_streams_and_graphs(ops):
    """Queued on the stream they are given, in its order; captured once the
    handle's scratch has its size."""
    x = randn(gen(18), 4, 64 * 64, 256).half()
    w, sw = ops.quantize_fp8(randn(gen(19), 512, 256), 128)

    def chain(out):
        codes, scales = ops.group_norm_fp8(x, 32, act=SILU)
        return ops.matmul_fp8(codes, scales, w, sw, out=out)

    want = chain(None)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    out = torch.zeros_like(want)
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        chain(out)
        copy = out.clone()
    ops.sync(side.cuda_stream)
    assert torch.equal(copy, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        chain(out)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_offsets_past_32_bits(ops):
    """Rows whose element offsets do not fit 32 bits."""
    step = 1 << 20
    wide = torch.empty((2100, step), device="cuda", dtype=torch.float16)  # 4.1 GiB
    x = wide[:, -512:]
    x.copy_(randn(gen(20), 2100, 512))
    assert torch.equal(ops.group_norm(x[None], 32, act=SILU), ops.group_norm(x.clone()[None], 32, act=SILU))
    ops.group_norm(x[None], 32, act=SILU, out=x[None])
    a, sa = ops.quantize_fp8(x)
    b, sb = ops.quantize_fp8(x.clone())
    assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)) and torch.equal(sa, sb)
    w, sw = ops.quantize_fp8(randn(gen(21), 256, 512), 128)
    want = ops.matmul_fp8(a, sa, w, sw)
    ops.matmul_fp8(a, sa, w, sw, out=wide[:, :256])
    assert torch.equal(wide[:, :256], want)
    codes = wide.view(torch.float8_e4m3fn)[:, -512:]  # offsets past 2^32 bytes
    codes.view(torch.uint8).copy_(a.view(torch.uint8))
    assert torch.equal(ops.matmul_fp8(codes, sa, w, sw), want)


def test_gamma_and_beta_from_the_product_before(ops):
    """An adaptive normalisation: gamma and beta are what a product queued just
    before writes. Every kernel may start while the one before it runs; none
    reads its inputs before that one is done. (The map takes two kernels.)"""
    x = randn(gen(22), 2, 40000, 256).half()
    (a, sa), (w, sw) = operands(ops, gen(23), 2, 256, 8192)
    big = randn(gen(24), 8192, 8192).half()
    for _ in range(3):
        both = torch.zeros((2, 256), device="cuda")
        torch.cuda.synchronize()
        ops.quantize_fp8(big)  # keeps the stream busy while the calls below are queued
        ops.matmul_fp8(a, sa, w, sw, out=both, dtype=torch.float32)
        got = ops.group_norm(x, 32, both[0], both[1], act=SILU)
        torch.cuda.synchronize()
        assert torch.equal(got, ops.group_norm(x, 32, both[0].clone(), both[1].clone(), act=SILU))


def test_a_graph_keeps_its_scratch(ops):
    """A captured call replays after larger calls on its stream."""
    x = randn(gen(25), 1, 30000, 256).half()
    side, out = torch.cuda.Stream(), torch.empty_like(x)
    with torch.cuda.stream(side):
        want = ops.group_norm(x, 32, act=SILU)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.group_norm(x, 32, act=SILU, out=out)
    with torch.cuda.stream(side):
        wide = randn(gen(26), 40, 600, 40003).half()  # one value at a time, a few MB of pairs
        ops.group_norm(wide, 40003, out=wide)
        del wide
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_launch_timing(ops):
    """The launch record covers the operators' handle."""
    import iec

    x = randn(gen(27), 2, 64, 64, 256).half()
    w, sw = ops.quantize_fp8(randn(gen(28), 512, 256), 128)
    iec.set_launch_timing(ops, True)
    codes, scales = ops.group_norm_fp8(x, 32)
    ops.matmul_fp8(codes, scales, w, sw)
    names = [r["name"] for r in iec.launch_timing(ops)]
    iec.set_launch_timing(ops, False)
    assert any(n.startswith("norm_") for n in names) and any("8192x512x256" in n for n in names)


def test_refusals(ops):
    import iec

    half = dict(device="cuda", dtype=torch.float16)
    x = torch.zeros((2, 4, 48), **half)

    def refused(call, *words):
        with pytest.raises(iec.IecError) as e:
            call()
        assert e.value.code == iec.ERR_INPUT
        for w in words:
            assert w in str(e.value), str(e.value)

    refused(lambda: ops.group_norm(x, 5), "5 groups", "48")
    refused(lambda: ops.group_norm(x, 0), "groups")
    refused(lambda: ops.group_norm(x, 4, eps=-1.0), "eps")
    refused(lambda: ops.group_norm(x, 4, eps=float("nan")), "eps")
    refused(lambda: ops.group_norm(x, 4, act=9), "activation")
    refused(lambda: ops.group_norm(x.double(), 4), "float64")
    refused(lambda: ops.group_norm(x.cpu(), 4), "cpu")
    refused(lambda: ops.group_norm(x, 4, gamma=torch.ones(48)), "gamma", "cpu")
    refused(lambda: ops.group_norm(x, 4, gamma=torch.ones(47, device="cuda")), "gamma")
    refused(lambda: ops.group_norm(x, 4, out=torch.empty((2, 4, 47), **half)), "out")
    refused(lambda: ops.group_norm(x.transpose(1, 2), 4), "channels")
    refused(lambda: ops.group_norm(x[:, :, None].expand(2, 4, 3, 48), 4), "stride")
    rows = torch.zeros((6, 96), **half)
    refused(lambda: ops.quantize_fp8(rows, 64), "64 rows")
    refused(lambda: ops.quantize_fp8(rows.t()), "rows")
    a, sa = ops.quantize_fp8(rows)
    w, sw = ops.quantize_fp8(rows, 128)
    refused(lambda: ops.matmul_fp8(a, sa, w[:, :80], sw), "w")
    refused(lambda: ops.matmul_fp8(a, sa[:, :5], w, sw), "a_scales")
    refused(lambda: ops.matmul_fp8(a[:, 8:], sa, w[:, 8:], sw), "16")
    odd = torch.zeros((6, 100), device="cuda").to(torch.float8_e4m3fn)[:, :96]
    refused(lambda: ops.matmul_fp8(odd, sa, w, sw), "16")
    refused(lambda: ops.matmul_fp8(a, sa, w, sw, bias=torch.ones(5, device="cuda")), "bias")
    refused(lambda: ops.matmul_fp8(a, sa, w, sw, residual=torch.ones((6, 6), device="cuda")), "residual")
    refused(lambda: ops.matmul_fp8(a, sa, w, sw, act=-1), "activation")
    refused(lambda: ops.matmul_fp8(a, sa, w, sw, dtype=torch.float64), "float64")
    L = iec.lib()
    f = np.zeros(1, np.float32).ctypes.data

    def raw(x=x.data_ptr(), rows=2, step=16, dtype=0):
        args = iec.ops.QUANTIZE.pack(x or 0, rows, 16, step, 1, f, 16, f, 2, dtype)
        return L.iec_ops_quantize_fp8(ops._h, args, None)

    assert raw(x=x.data_ptr() + 1) == iec.ERR_INPUT
    assert b"aligned" in L.iec_last_error()
    assert raw(dtype=7) == iec.ERR_INPUT
    assert raw(step=15) == iec.ERR_INPUT
    assert raw(x=None) == iec.ERR_INPUT
    assert raw(rows=1 << 40) == iec.ERR_INPUT
    assert L.iec_ops_quantize_fp8(ops._h, None, None) == iec.ERR_INPUT
    # the handle works on after a refusal
    assert torch.isfinite(ops.group_norm(x, 4)).all()
