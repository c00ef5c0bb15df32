"""GPU: what a large number beside the others costs a linear of a few tokens: nothing where its code is zero.

Tolerance: that of the products (every product is exact; an fp32 sum is off by at most one unit 2^-23 of the sum of absolute terms for each of
K / 16 instructions and K / 128 + 16 additions; one rounding).  The absolute terms are those of the formula, x times code: a number met by
a code of zero has none, and a weight row of zeros gives zeros."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]
K, ROWS = 1024, 64


def _weights(gen, per_channel):
    """Codes with zeros at every 128th channel and in rows 3 and 40 throughout: (packed, scale, the numbers they stand for)."""
    codes = torch.randint(-8, 8, (ROWS, K), device="cuda", generator=gen)
    codes[:, 5::128] = 0
    codes[[3, 40]] = 0
    packed = ((codes[:, 0::2] & 15) | ((codes[:, 1::2] & 15) << 4)).to(torch.uint8).contiguous()
    scale = torch.full((ROWS,), 2.0 ** -6, device="cuda")
    if not per_channel:
        packed, scale = packed.view(ROWS, K // 128, 64).transpose(0, 1).contiguous(), scale.expand(K // 128, ROWS).contiguous()
    return packed, scale, codes.double() * 2.0 ** -6


def _tokens(gen, M, kind, ratio, dtype):
    """Tokens of a kind with one number of each 128 `ratio` times as large: 2^15 in fp16 at most, the others scaled down instead."""
    if kind == "normal":
        x = torch.randn(M, K, device="cuda", generator=gen)
    elif kind == "signs":
        x = torch.randint(0, 2, (M, K), device="cuda", generator=gen) * 2.0 - 1.0
    else:
        x = torch.randint(4, 9, (M, K), device="cuda", generator=gen) / 8.0
    top = float(ratio) if dtype == torch.bfloat16 else min(float(ratio), 2.0 ** 15)
    x = (x * (top / ratio)).to(dtype)
    x[:, 5::128] = top
    return x


def _product(x, w):
    x = x.double()
    return x @ w.T, (K / 16 + K / 128 + 16) * 2.0 ** -23 * (x.abs() @ w.abs().T)


def _check(out, ref, slack):
    half = torch.finfo(out.dtype).eps / 2
    err = (out.double() - ref).abs()
    bound = half * (ref.abs() + slack) + slack + (2.0 ** -25 if out.dtype == torch.float16 else 0)   # fp16: half a subnormal step
    assert (err <= bound).all(), (err - bound).max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("per_channel", [False, True])
@pytest.mark.parametrize("kind", ["normal", "signs", "eighths"])
@pytest.mark.parametrize("exponent", [4, 12, 16, 20, 24])
@pytest.mark.parametrize("M", [1, 8, 9])
def test_linear(M, exponent, kind, per_channel, dtype):
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(M + exponent)
    packed, scale, w = _weights(gen, per_channel)
    x = _tokens(gen, M, kind, 2 ** exponent, dtype)
    out = ops.w4a16_linear(x, packed, scale, ROWS, per_channel)
    ref, slack = _product(x, w)
    _check(out, ref, slack)
    assert not out[:, [3, 40]].any()
    # and each token by itself, whatever stands beside it
    for m in range(M):
        _check(ops.w4a16_linear(x[m:m + 1], packed, scale, ROWS, per_channel), ref[m:m + 1], slack[m:m + 1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("exponent", [12, 16, 20])
@pytest.mark.parametrize("M", [1, 8])
def test_gated(M, exponent, dtype):
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(exponent)
    packed, scale, w = _weights(gen, False)
    x = _tokens(gen, M, "normal", 2 ** exponent, dtype)
    out = ops.w4a16_gated_linear(x, packed, scale, ROWS // 2)
    y, slack = _product(x, w)
    (g, u), (dg, du) = y.chunk(2, -1), slack.chunk(2, -1)
    act = g * torch.sigmoid(g)
    # |d silu| <= 1.1; the activation itself is a handful of fp32 operations, the exponential's argument good to half a step of g
    _check(out, act * u, 1.1 * dg * u.abs() + act.abs() * du + 1.1 * dg * du + (16 + g.abs()) * 2.0 ** -23 * (act * u).abs())
    assert not out[:, [3, 8]].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_ones_beside_a_large_number(dtype):
    """127 ones under codes of one, and a number 2^25 times as large under a code of zero: 127."""
    from fp8_inference_toolkit_b200 import ops

    one = 1.0 if dtype == torch.bfloat16 else 2.0 ** -10
    x = torch.full((1, 128), one, device="cuda", dtype=dtype)
    x[0, 0] = one * 2.0 ** 25
    packed = torch.full((1, 16, 64), 0x11, dtype=torch.uint8, device="cuda")
    packed[:, :, 0] = 0x10
    out = ops.w4a16_linear(x, packed, torch.ones(1, 16, device="cuda"), 16)
    assert (out == 127 * one).all(), out
