"""The operators' activations alone, over their whole range (GPU tests): a
product without values along k is act(bias), a normalisation with gamma 0 is
act(beta).

Tolerances, u the output type's unit roundoff: for f32 2^-21 of the value, two
units each for an exponential, a sum, a quotient and a product. For 16 bits u +
2^-18: the exponent v log2(e) is rounded once, by up to 2^-17 / 2 at |v| = 87,
2^-18.5 of the exponential. Below -87.3 the sigmoid is less than
2^-126 and may be 0: 2^-119 of a SiLU, since |v| < 128 where that matters.
GELU: a Phi(-a), a = |v|, has its exponent a^2 log2(e) / 2 rounded twice, which
moves it by a^2 2^-24 of itself, next to 2^-20 for what else is rounded; for 16
bits its own form is good to 2^-14."""

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

NONE, RELU, GELU, SIGMOID, SILU = range(5)
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
SMALL = {"f16": 2.0 ** -25, "bf16": 0.0, "f32": 0.0}  # half a subnormal step
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def ops():
    from iec.ops import Ops

    o = Ops()
    yield o
    o.close()


def of_bias(ops, v, act, dtype, rows=1):
    """act(v) as rows x len(v), through a product with k = 0."""
    n, fp8 = v.numel(), torch.float8_e4m3fn
    a, w = (torch.zeros((r, 16), device="cuda").to(fp8)[:, :0] for r in (rows, n))
    sa, sw = (torch.zeros((0, c), device="cuda") for c in (rows, -(-n // 128)))
    return ops.matmul_fp8(a, sa, w, sw, v, act, dtype=TYPES[dtype])


def act64(v, act):
    if act == GELU:
        return 0.5 * v * torch.special.erfc(-v * 0.5 ** 0.5)
    return torch.sigmoid(v) if act == SIGMOID else v * torch.sigmoid(v)


def arguments():
    """Dense around 0, then every size, both signs."""
    sizes = torch.logspace(-12, 4.5, 20001, dtype=torch.float64)
    return torch.cat([torch.linspace(-110, 110, 100001, dtype=torch.float64), sizes, -sizes]).float().cuda()


def close(got, want, dtype, relative, tiny):
    top = {"f16": 65504.0, "bf16": 3.3895313892515355e38, "f32": 3.4028234663852886e38}[dtype]
    fits = want.abs() <= top
    off = (got.double() - want).abs() - (HALF[dtype] + relative) * want.abs() - SMALL[dtype] - tiny
    assert (off[fits] <= 0).all(), off[fits].max().item()
    assert (got[~fits].double() == want[~fits].sign() * INF).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("act", [SIGMOID, SILU])
@pytest.mark.parametrize("rows", [1, 300])
def test_sigmoid_and_silu_over_their_range(ops, act, dtype, rows):
    """One row takes the products that split k, 300 rows whole tiles."""
    v = arguments()
    got = of_bias(ops, v, act, dtype, rows)
    want = act64(v.double(), act)
    for y in (got[0], got[-1]):
        close(y, want, dtype, 2.0 ** -21 if dtype == "f32" else 2.0 ** -18, 2.0 ** -119)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_sigmoid_and_silu_of_the_largest(ops, dtype):
    """v / (1 + e^-v) and 1 / (1 + e^-v) as f32 has them."""
    v = torch.tensor([-1e2, -1e4, -1e20, -3e38, -INF, 1e2, 1e4, 1e20, 3e38, INF, NAN, 0.0], device="cuda")
    silu, sigmoid = (of_bias(ops, v, act, dtype)[0].float() for act in (SILU, SIGMOID))
    assert (sigmoid[:5].abs() <= 2.0 ** -126).all() and (sigmoid[5:10] == 1).all()
    assert torch.isnan(sigmoid[10]) and sigmoid[11] == 0.5
    assert (silu[:4].abs() <= 2.0 ** -119).all() and torch.isnan(silu[4])
    assert torch.equal(silu[5:10], v[5:10].to(TYPES[dtype]).float())
    assert torch.isnan(silu[10]) and silu[11] == 0


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 300])
def test_gelu_over_its_range(ops, dtype, rows):
    v = arguments()
    got = of_bias(ops, v, GELU, dtype, rows)
    want = act64(v.double(), GELU)
    relative = 2.0 ** (-20 if dtype == "f32" else -14) + torch.clamp_max(v.double().abs(), 14) ** 2 * 2.0 ** -23
    for y in (got[0], got[-1]):
        close(y, want, dtype, relative, 2.0 ** -119)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gelu_of_the_largest(ops, dtype):
    v = torch.tensor([-1e2, -1e4, -1e20, -3e38, 1e2, 1e4, 1e20, 3e38, INF, NAN, 0.0], device="cuda")
    got = of_bias(ops, v, GELU, dtype)[0].float()
    assert (got[:4] == 0).all() and torch.equal(got[4:9], v[4:9].to(TYPES[dtype]).float())
    assert torch.isnan(got[9]) and got[10] == 0
    least = of_bias(ops, torch.full((8,), -INF, device="cuda"), GELU, dtype)
    assert (torch.isnan(least) | (least == 0)).all()  # -inf 0, or its limit


@pytest.mark.parametrize("act,lo,hi", [(GELU, -6.0, 2.0), (GELU, -5.5, -4.5), (SILU, -12.0, -6.0), (SIGMOID, -70.0, -60.0)])
@pytest.mark.parametrize("pixels", [33, 9000])
def test_eight_bit_rows_of_tails(ops, act, lo, hi, pixels):
    """Whole blocks in an activation's tail keep the codes' precision: the
    value is within 2^-15 of itself before it is quantised, so codes and scales
    are off by no more than that beside their own rounding."""
    c = 256
    beta = torch.linspace(lo, hi, c, device="cuda")
    x = torch.zeros(1, pixels, c, device="cuda", dtype=torch.float16)
    codes, scales = ops.group_norm_fp8(x, 2, torch.zeros(c, device="cuda"), beta, act=act)
    want = act64(beta.double(), act).reshape(2, 128)
    top = want.abs().amax(1)
    assert ((scales.double() * 448 / top[:, None] - 1).abs() <= 2.0 ** -14).all()
    back = codes.double().reshape(pixels, 2, 128) * scales.double().t()[:, :, None]
    step = torch.clamp_min(want.abs() / 16, top[:, None] / 448 * 2.0 ** -10)  # half a step of the codes
    assert ((back - want).abs() <= step + 2.0 ** -14 * want.abs()).all()


@pytest.mark.parametrize("act", [GELU, SIGMOID, SILU])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_a_nan_or_infinity_leaves_its_neighbours_alone(ops, act, dtype):
    """Values that share a reciprocal."""
    v = torch.linspace(-9, 9, 64, device="cuda")
    want = of_bias(ops, v, act, dtype)[0]
    for at in (0, 1, 30, 31, 62, 63):
        for odd in (NAN, INF, -INF, -1e30, 1e30):
            u = v.clone()
            u[at] = odd
            got = of_bias(ops, u, act, dtype)[0]
            keep = torch.arange(64, device="cuda") != at
            assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("pixels", [40, 60000])
@pytest.mark.parametrize("c", [256, 254])
def test_eight_bit_rows_of_silu_far_below_zero(ops, pixels, c):
    """Blocks of SiLU values below 2^-100 are zeros with scale 1; those above
    it have their value, 2^-4 of it at most beside the code's own rounding."""
    x = torch.zeros(1, pixels, c, device="cuda", dtype=torch.float16)
    gamma, beta = torch.zeros(c, device="cuda"), torch.empty(c, device="cuda")
    beta[:128], beta[128:] = -60.0, -1e6
    codes, scales = ops.group_norm_fp8(x, 2, gamma, beta, act=SILU)
    want = act64(torch.tensor(-60.0, dtype=torch.float64), SILU).item()
    back = codes[:, :128].double() * scales[0].double()[:, None]
    assert ((back / want - 1).abs() <= 2.0 ** -4).all()
    assert (codes[:, 128:].float() == 0).all() and (scales[1] == 1).all()
