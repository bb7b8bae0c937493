"""The 8-bit product where tests/test_ops_gpu.py does not reach (GPU tests):
scales at the ends of f32's range, as many columns as it takes."""

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

FP8 = torch.float8_e4m3fn


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


def product64(a, sa, w, sw):
    """(a w^T, sum of magnitudes) in 64 bits."""
    n, k = w.shape
    x = a.double() * sa.t().double().repeat_interleave(128, 1)[:, :k]
    y = w.double() * sw.t().double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return x @ y.t(), x.abs() @ y.abs().t()


SIZES = [(3, 40, 16), (5, 300, 700), (300, 200, 260), (20000, 130, 130), (8200, 1040, 300)]
TOP = 3.4028234663852886e38


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("a_exp,w_exp", [(66, 66), (-66, -66), (-109, -40), (119, 30), (40, -149), (100, 127), (-60, 50)])
def test_scales_at_the_ends_of_the_range(ops, m, n, k, a_exp, w_exp):
    """The two scales of a block count as their f32 product: cut off at the
    largest value, off by half a step of 2^-149 below 2^-126, which a block's sum
    of magnitudes multiplies. Sums of zero are 0 whatever the scales."""
    from iec.ops import empty_codes

    g = gen(m + n + k)
    a, w = empty_codes(m, k, "cuda"), empty_codes(n, k, "cuda")
    a.copy_(4 * randn(g, m, k))
    w.copy_(4 * randn(g, n, k))
    a.view(torch.uint8)[1] = 0
    w.view(torch.uint8)[2] = 0
    kb = -(-k // 128)
    sa = torch.full((kb, m), 2.0, device="cuda", dtype=torch.float64).pow(a_exp).float()
    sw = torch.full((kb, -(-n // 128)), 2.0, device="cuda", dtype=torch.float64).pow(w_exp).float()
    sa[:, 0] = 1.0  # a row in range among them
    got = ops.matmul_fp8(a, sa, w, sw, dtype=torch.float32).double()
    want, size = product64(a, sa, w, sw)
    plain = a.double().abs() @ w.double().abs().t()
    assert (got[1] == 0).all() and (got[:, 2] == 0).all()
    sure = size < TOP  # no partial sum overflows
    off = (got - want).abs() - 2.0 ** -16 * size - 2.0 ** -150 * plain - kb * 2.0 ** -149
    assert (off[sure] <= 0).all(), off[sure].max().item()
    assert torch.isfinite(got[sure]).all()
    if a_exp + w_exp > 128 and kb == 1:
        far = (want / 2.0 ** (a_exp + w_exp)).abs() >= 2  # twice the largest value, or more
        far[0] = False
        assert far.any() and (got[far] == want[far].sign() * float("inf")).all()


@pytest.mark.parametrize("m,n,k", SIZES)
def test_a_row_out_of_range_leaves_the_others_as_they_are(ops, m, n, k):
    g = gen(m + n)
    (a, sa), (w, sw) = ops.quantize_fp8(randn(g, m, k)), ops.quantize_fp8(randn(g, n, k), 128)
    want = ops.matmul_fp8(a, sa, w, sw, dtype=torch.float32)
    sa[:, 2] = 2.0 ** -140
    sa[0, 1] = float("inf")
    a.view(torch.uint8)[1, 0] = 127  # NaN, as in a row with an infinity
    got = ops.matmul_fp8(a, sa, w, sw, dtype=torch.float32)
    keep = torch.ones(m, dtype=torch.bool, device="cuda")
    keep[1] = keep[2] = False
    assert torch.equal(got[keep], want[keep])
    assert torch.isnan(got[1]).all() and (got[2].abs() <= 2.0 ** -100).all()


def test_infinite_scales_stay_infinite(ops):
    a, w = (torch.full((r, 16), 2.0, device="cuda").to(FP8) for r in (3, 4))
    w.view(torch.uint8)[1] = 0
    sa = torch.tensor([[1.0, float("inf"), float("nan")]], device="cuda")
    got = ops.matmul_fp8(a, sa, w, torch.ones((1, 1), device="cuda"), dtype=torch.float32)
    assert torch.equal(got[0], torch.tensor([64.0, 0.0, 64.0, 64.0], device="cuda"))
    assert torch.isnan(got[1, 1]) and (got[1, [0, 2, 3]] == float("inf")).all() and torch.isnan(got[2]).all()


def test_zero_weights_beside_the_largest_values(ops):
    """Quantised as a user does it: 1e38 times a weight of 0 is 0."""
    g = gen(9)
    x, weights = randn(g, 40, 256), 1e4 * randn(g, 130, 256)
    x[3] = 1e38 * x[3].sign()
    weights[7] = 0
    got = ops.matmul_fp8(*ops.quantize_fp8(x), *ops.quantize_fp8(weights, 128), dtype=torch.float32)
    assert (got[:, 7] == 0).all()


@pytest.mark.parametrize("m,n,k", [(2, 1 << 20, 32), (130, (1 << 20) - 127, 16), (1, (1 << 20) - 128, 144)])
def test_as_many_columns_as_it_takes(ops, m, n, k):
    g = gen(m)
    (a, sa), (w, sw) = ops.quantize_fp8(randn(g, m, k)), ops.quantize_fp8(randn(g, n, k), 128)
    got = ops.matmul_fp8(a, sa, w, sw).double()
    want, size = product64(a, sa, w, sw)
    assert ((got - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -25 + 2.0 ** -16 * size).all()


def test_one_column_more_is_refused(ops):
    import iec
    from iec.ops import empty_codes

    n = (1 << 20) + 1
    with pytest.raises(iec.IecError) as e:
        ops.matmul_fp8(empty_codes(1, 16, "cuda"), torch.ones((1, 1), device="cuda"), empty_codes(n, 16, "cuda"),
                       torch.ones((1, -(-n // 128)), device="cuda"))
    assert e.value.code == iec.ERR_INPUT and "columns" in str(e.value)


def kernels_of(ops, call):
    """What `call` returns and the kernels it launches, from the launch record."""
    import iec

    iec.set_launch_timing(ops, True)
    try:
        out = call()
        return out, [r["name"] for r in iec.launch_timing(ops)]
    finally:
        iec.set_launch_timing(ops, False)


NONE, RELU, GELU, SIGMOID, SILU = range(5)
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
SMALL = {"f16": 2.0 ** -25, "bf16": 0.0, "f32": 0.0}  # half a subnormal step
SINGLE, PAIR, SPLIT = "fp8_gemm_sm100<0>", "fp8_gemm_sm100<1>", "fp8_gemm_sm100<2>"
# m, n, k: rows of every type start on 16 bytes; tiles, and blocks along k, are cut short
TILES = [(2300, 2040, 1100, PAIR), (2304, 2048, 128, PAIR), (9400, 2040, 300, PAIR), (4090, 1528, 300, SINGLE), (100, 200, 2000, SPLIT)]


def act64(v, act):
    if act == RELU:
        return torch.relu(v)
    if act == GELU:
        return 0.5 * v * torch.special.erfc(-v * 0.5 ** 0.5)
    if act == SIGMOID:
        return torch.sigmoid(v)
    return v * torch.sigmoid(v) if act == SILU else v


def operands(ops, m, n, k):
    """Codes and scales whose products are about 1."""
    g = gen(m + n + k)
    (a, sa), (w, sw) = ops.quantize_fp8(randn(g, m, k) * k ** -0.5), ops.quantize_fp8(randn(g, n, k), 128)
    return a, sa, w, sw, randn(g, n)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("m,n,k,kernel", TILES)
def test_every_tile_shape_with_its_whole_epilogue(ops, m, n, k, kernel, dtype):
    """Each kernel against the 64-bit product, through TMA: bias, activation
    (slope at most 1.13, good to 2^-14 for 16 bits) and residual, the residual
    in a tensor of its own, in the output, and in a wider output whose other
    columns stay as they are."""
    a, sa, w, sw, bias = operands(ops, m, n, k)
    res = randn(gen(7), m, n).to(TYPES[dtype])
    raw, size = product64(a, sa, w, sw)
    raw = raw + bias.double()
    slack = 1.13 * 2.0 ** -16 * (size + bias.double().abs())

    def good(got, want, act):
        curve = 0.0 if act in (NONE, RELU) else 2.0 ** (-19 if dtype == "f32" else -14) * act64(raw, act).abs()
        off = (got.double() - want).abs() - HALF[dtype] * want.abs() - SMALL[dtype] - slack - curve
        assert (off <= 0).all(), off.max().item()

    got, names = kernels_of(ops, lambda: ops.matmul_fp8(a, sa, w, sw, bias, dtype=TYPES[dtype]))
    assert names == [f"{kernel} {m}x{n}x{k}"]
    good(got, raw, NONE)
    for act in (NONE, RELU, GELU, SIGMOID, SILU):
        want = act64(raw, act) + res.double()
        got, names = kernels_of(ops, lambda: ops.matmul_fp8(a, sa, w, sw, bias, act, res, dtype=TYPES[dtype]))
        assert names == [f"{kernel} {m}x{n}x{k}"]
        good(got, want, act)
        out = res.clone()
        ops.matmul_fp8(a, sa, w, sw, bias, act, out, out=out)
        assert torch.equal(out, got)
        wide = torch.full((m + 1, n + 16), 7.0, device="cuda", dtype=TYPES[dtype])
        wide[:m, :n] = res
        ops.matmul_fp8(a, sa, w, sw, bias, act, wide[:m, :n], out=wide[:m, :n])
        assert torch.equal(wide[:m, :n], got) and (wide[:m, n:] == 7).all() and (wide[m] == 7).all()
        odd = torch.full((m, n + 5), 7.0, device="cuda", dtype=TYPES[dtype])  # rows that start anywhere: no TMA
        ops.matmul_fp8(a, sa, w, sw, bias, act, res, out=odd[:, 2:n + 2])
        assert torch.equal(odd[:, 2:n + 2], got) and (odd[:, :2] == 7).all() and (odd[:, n + 2:] == 7).all()


@pytest.mark.parametrize("m,n,k,kernel", TILES)
def test_every_tile_shape_sums_in_32_bits(ops, m, n, k, kernel):
    a, sa, w, sw, _ = operands(ops, m, n, k)
    want, _ = product64(a, sa, w, sw)
    got, names = kernels_of(ops, lambda: ops.matmul_fp8(a, sa, w, sw, dtype=torch.float32))
    assert names == [f"{kernel} {m}x{n}x{k}"]
    assert ((got.double() - want).norm() / want.norm()).item() <= 2.0 ** -20
