"""GPU: rotary positions against the rotation in 64 bits.

Tolerance: half a step of the type for the one rounding, and of the two products 2^-21 of their factors' absolute sum: the angle is good to
2^-24 of half a turn (2^-22.3 rad), cosine and sine to 2 units of 2^-24, the scale and the two products to one each."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _turn(x, positions, freqs, interleaved, scale, inverse):
    """The rotation in 64 bits, and the sum of absolute values that its terms have."""
    x, R = x.double(), 2 * freqs.numel()
    angle = positions.double()[:, None, None] * freqs * (-1 if inverse else 1)
    c, s = angle.cos() * scale, angle.sin() * scale
    out, mag = x.clone(), torch.zeros_like(x)
    i = torch.arange(0, R, 2) if interleaved else torch.arange(R // 2)
    j = i + (1 if interleaved else R // 2)
    a, b = x[..., i], x[..., j]
    out[..., i], out[..., j] = a * c - b * s, b * c + a * s
    mag[..., i] = mag[..., j] = (a.abs() + b.abs()) * abs(scale)
    return out, mag


def _check(out, ref, mag):
    half = torch.finfo(out.dtype).eps / 2
    assert ((out.double() - ref).abs() <= half * ref.abs() + 2.0 ** -21 * mag * (mag != 0) + (2.0 ** -25 if out.dtype == torch.float16 else 0)).all()


CASES = [
    # tokens, heads, D, R, interleaved, scale, inverse
    (1, 1, 2, 2, False, 1.0, False), (1, 1, 2, 2, True, 1.0, True), (16, 40, 128, 128, False, 1.0, False), (777, 9, 96, 64, True, 1.0, True),
    (130, 3, 80, 40, False, 1.1386, False), (5, 7, 65, 64, True, 0.5, False), (5, 7, 65, 34, False, 1.0, True), (2500, 1, 64, 64, False, 1.0, False),
    (3, 64, 256, 64, True, 1.25, False), (33, 5, 12, 6, False, 1.0, False), (33, 5, 12, 6, True, 1.0, False), (9, 2, 128, 0, False, 1.0, False),
    (4, 300, 128, 128, True, 1.0, False),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,heads,D,R,interleaved,scale,inverse", CASES)
def test_rope(tokens, heads, D, R, interleaved, scale, inverse, index, dtype):
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(tokens + D)
    x = torch.randn(tokens, heads, D, device="cuda", generator=gen).to(dtype)
    positions = torch.randint(-5, 1 << 20, (tokens,), device="cuda", generator=gen).to(index)
    freqs = 1e4 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / max(R, 1))
    ref, mag = _turn(x, positions, freqs, interleaved, scale, inverse)
    out = ops.rope(x, positions, freqs, interleaved=interleaved, scale=scale, inverse=inverse)
    assert out.dtype == dtype and out.shape == x.shape
    _check(out, ref, mag)
    same = x.clone()
    assert ops.rope_(same, positions, freqs, interleaved, scale, inverse) is same
    assert torch.equal(same, out)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", ["heads of a wider buffer", "off by one", "odd rows", "heads first", "columns"])
def test_rope_takes_any_layout(layout, interleaved):
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(1)
    dense = torch.randn(21, 6, 64, device="cuda", generator=gen).to(torch.bfloat16)
    new = lambda *s: torch.full(s, 7.0, dtype=dense.dtype, device="cuda")  # noqa: E731
    whole, x = {
        "heads of a wider buffer": lambda: (b := new(21, 10, 64), b[:, 2:8]),
        "off by one": lambda: (b := new(21 * 6 * 64 + 1), b[1:].view(21, 6, 64)),
        "odd rows": lambda: (b := new(21, 6 * 64 + 3), b[:, 3:].unflatten(1, (6, 64))),
        "heads first": lambda: (b := new(6, 21, 64), b.transpose(0, 1)),
        "columns": lambda: (b := new(21, 64, 6), b.transpose(1, 2)),
    }[layout]()
    x.copy_(dense)
    positions = torch.arange(21, device="cuda") * 1000
    freqs, _ = ops.rope_frequencies(64, 1e6)
    want = ops.rope(dense, positions, freqs, interleaved)
    assert torch.equal(ops.rope(x, positions, freqs, interleaved), want) and torch.equal(x, dense)
    if layout == "columns":
        with pytest.raises(RuntimeError, match="contiguous"):
            ops.rope_(x, positions, freqs, interleaved)
        return
    outside = whole.clone()
    ops.rope_(x, positions, freqs, interleaved)
    assert torch.equal(x, want)
    x.copy_(dense)
    assert torch.equal(whole, outside)                  # what is not x stays as it was


@pytest.mark.parametrize("interleaved", [False, True])
def test_inverse_is_the_gradient(interleaved):
    """Against the derivative of the formula by autograd in 64 bits, and against differences of the formula."""
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(2)
    x, up = (torch.randn(11, 3, 48, device="cuda", generator=gen).to(torch.float16) for _ in range(2))
    positions = torch.randint(0, 30000, (11,), device="cuda", generator=gen)
    freqs, _ = ops.rope_frequencies(32, 1e4)
    grad = ops.rope(up, positions, freqs, interleaved, scale=1.2, inverse=True)
    grad[..., 32:] = up[..., 32:]

    def f(v):
        i = torch.arange(0, 32, 2) if interleaved else torch.arange(16)
        j = i + (1 if interleaved else 16)
        angle = positions.double()[:, None, None] * freqs
        c, s = angle.cos() * 1.2, angle.sin() * 1.2
        y = v.clone()
        y[..., i], y[..., j] = v[..., i] * c - v[..., j] * s, v[..., j] * c + v[..., i] * s
        return (y * up.double()).sum()

    v = x.double().requires_grad_()
    f(v).backward()
    mag = up.double().abs().amax(-1, keepdim=True).expand_as(v) * 2.4
    _check(grad, v.grad, mag)
    step = torch.randn(x.shape, device="cuda", generator=gen, dtype=torch.float64) * 1e-3
    with torch.no_grad():
        change = (f(v + step) - f(v - step)) / 2
    # the formula is linear: only the gradient's own rounding is left
    bound = ((torch.finfo(torch.float16).eps / 2) * v.grad.abs() + 2.0 ** -21 * mag + 2.0 ** -25).mul(step.abs()).sum()
    assert (change - (grad.double() * step).sum()).abs() <= bound + 1e-9


def test_frequencies():
    from fp8_inference_toolkit_b200 import ops

    plain, one = ops.rope_frequencies(128, 1e6)
    assert one == 1.0 and plain.dtype == torch.float64
    assert torch.allclose(plain, 1e6 ** (-torch.arange(0, 128, 2, dtype=torch.float64, device="cuda") / 128), rtol=1e-14)
    linear, _ = ops.rope_frequencies(128, 1e6, scaling="linear", factor=4.0)
    assert torch.equal(linear, plain / 4)
    base, _ = ops.rope_frequencies(128, 1e6, scaling="base", factor=4.0)
    assert base[0] == 1.0 and abs(base[-1].item() * 4 / plain[-1].item() - 1) < 1e-12
    parts, scale = ops.rope_frequencies(128, 1e6, scaling="by_parts", factor=4.0, trained_length=32768)
    turns = 32768 * plain / (2 * math.pi)
    assert torch.equal(parts[turns >= 32], plain[turns >= 32]) and torch.equal(parts[turns <= 1], plain[turns <= 1] / 4)
    between = (turns > 1) & (turns < 32)
    assert between.any() and (parts[between] < plain[between]).all() and (parts[between] > plain[between] / 4).all()
    assert scale == 1.0 + 0.1 * math.log(4.0)
    for bad in [dict(rotary_dim=3, theta=1e4), dict(rotary_dim=0, theta=1e4), dict(rotary_dim=4, theta=1e4, scaling="other"),
                dict(rotary_dim=4, theta=1e4, scaling="by_parts", factor=2.0), dict(rotary_dim=4, theta=1e4, factor=0.0)]:
        with pytest.raises(RuntimeError):
            ops.rope_frequencies(**bad)


def test_rope_of_nothing_and_refusals():
    from fp8_inference_toolkit_b200 import ops

    x = torch.randn(4, 2, 16, device="cuda").to(torch.bfloat16)
    at, (freqs, _) = torch.arange(4, device="cuda"), ops.rope_frequencies(16, 1e4)
    assert ops.rope(x[:0], at[:0], freqs).shape == (0, 2, 16) and ops.rope_(x[:, :0], at, freqs).shape == (4, 0, 16)
    for args, match in [((x.cpu(), at, freqs), "CUDA"), ((x.float(), at, freqs), "bfloat16"), ((x[0], at, freqs), "3D"), ((x, at[:3], freqs), "tokens"),
                        ((x, at.float(), freqs), "int32"), ((x, at, freqs.float()), "float64"), ((x, at.cpu(), freqs), "device"),
                        ((x, at, ops.rope_frequencies(18, 1e4)[0]), "fewer"), ((x.clone().requires_grad_(), at, freqs), "backward")]:
        with pytest.raises(RuntimeError, match=match):
            ops.rope(*args)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.rope_(x[:1].expand(4, 2, 16), at, freqs)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.rope_(x.view(-1)[:100].as_strided((4, 2, 16), (16, 16, 1)), at, freqs)
