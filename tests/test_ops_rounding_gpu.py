"""What a whole block or group shares is as good as f32 lets it be (GPU
tests): a block's scale and factor are quotients rounded once, a group's 1 /
sqrt(variance + eps) nearly so."""

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(scope="module")
def ops():
    from iec.ops import Ops

    o = Ops()
    yield o
    o.close()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,k", [(40000, 128), (3000, 1024), (700, 1001), (5000, 31)])
def test_scales_and_factors_are_rounded_once(ops, rows, k, block_rows, dtype):
    """scale = amax / 448 and code = e4m3(x * (448 / amax)), each quotient the
    f32 value nearest to it (1 where amax is below 2^-100)."""
    g = torch.Generator(device="cuda")
    g.manual_seed(rows + k)
    x = (torch.randn(rows, k, generator=g, device="cuda") * torch.exp(8 * torch.randn(rows, 1, generator=g, device="cuda"))).to(TYPES[dtype])
    x = x.clamp(-6e4, 6e4)
    codes, scales = ops.quantize_fp8(x, block_rows)
    kb, rb = -(-k // 128), -(-rows // block_rows)
    full = torch.zeros(rb * block_rows, kb * 128, device="cuda")
    full[:rows, :k] = x.float().abs()
    amax = full.reshape(rb, block_rows, kb, 128).amax((1, 3))
    tiny, one = amax < 2.0 ** -100, torch.ones_like(amax)
    assert torch.equal(scales.t(), torch.where(tiny, one, (amax.double() / 448).float()))
    factor = torch.where(tiny, one, (448 / amax.double()).float()).repeat_interleave(block_rows, 0).repeat_interleave(128, 1)[:rows, :k]
    assert torch.equal(codes.view(torch.uint8), (x.float() * factor).to(torch.float8_e4m3fn).view(torch.uint8))


@pytest.mark.parametrize("pixels,c", [(64, 512), (64, 511), (16, 64)])
def test_a_groups_rstd_is_nearly_rounded_once(ops, pixels, c):
    """Groups of one channel that hold 1 and -1, equally often: every sum of
    them is exact, the mean 0, the variance 1, and 1 + eps has no rounding for
    multiples of 2^-22 below 3. The result is 1 / sqrt(1 + eps) itself, 2^-24 of
    it if it is rounded once; half as much again is left for a step towards it."""
    x = torch.ones(1, pixels, c, device="cuda")
    x[:, 1::2] = -1
    g = torch.Generator()
    g.manual_seed(pixels + c)
    worst = 0.0
    for j in torch.randint(1, 3 << 22, (400,), generator=g).tolist():
        eps = j * 2.0 ** -22
        got = ops.group_norm(x, c, eps=eps).double()
        assert (got[:, 1::2] == -got[:, :1]).all()
        worst = max(worst, ((got[:, 0::2] * (1 + eps) ** 0.5 - 1).abs()).max().item())
    assert worst <= 1.5 * 2.0 ** -24 + 2.0 ** -40, worst
