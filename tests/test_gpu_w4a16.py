"""GPU: the int4-weight linear of a few 16-bit tokens and its gated form against the product in 64 bits.

Tolerance: products of a code and a 16-bit number are exact, so an fp32 sum is off by its additions: at most one unit 2^-23 of the sum of
absolute terms for each of the K / 16 tensor instructions (they may truncate), and for each of the K / 128 + 16 additions of groups,
warps and ranks; the result is rounded once (half a step of its type)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def _weights(gen, rows, K, per_channel):
    """(codes as held, scales as held, the numbers they stand for [rows, K] in 64 bits)."""
    codes = torch.randint(-8, 8, (rows, K), device="cuda", generator=gen)
    packed = ((codes[:, 0::2] & 15) | ((codes[:, 1::2] & 15) << 4)).to(torch.uint8)
    if per_channel:
        scale = torch.rand(rows, device="cuda", generator=gen) * 0.02 + 1e-3
        return packed.contiguous(), scale, codes.double() * scale.double()[:, None]
    G = K // 128
    scale = torch.rand(G, rows, device="cuda", generator=gen) * 0.02 + 1e-3
    packed = packed.view(rows, G, 64).transpose(0, 1).contiguous()
    return packed, scale, (codes.view(rows, G, 128).double() * scale.T.double()[..., None]).view(rows, K)


def _product(x, w):
    x = x.double()
    return x @ w.T, (x.shape[1] / 16 + x.shape[1] / 128 + 16) * 2.0 ** -23 * (x.abs() @ w.abs().T)


def _check(out, ref, slack):
    half = torch.finfo(out.dtype).eps / 2
    err = (out.double() - ref).abs()
    bound = half * (ref.abs() + slack) + slack + (2.0 ** -25 if out.dtype == torch.float16 else 0)   # fp16: half a subnormal step
    assert (err <= bound).all(), (err / bound).max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N,per_channel", [
    (1, 128, 1, False), (1, 64, 1, True), (1, 4096, 6144, False), (2, 4096, 4096, True), (3, 12288, 33, False), (5, 2560, 9728, True),
    (7, 192, 31, True), (8, 128 * 7, 16, False), (9, 128 * 9, 17, False), (16, 12288, 4096, False), (17, 1024, 1000, True),
    (31, 4096, 513, False), (32, 12288, 47, False), (32, 12288 + 64, 65, True), (33, 2048, 257, False), (100, 1024, 96, True),
    (1, 65536, 5, False), (32, 32768, 24, False),
])
def test_linear(M, K, N, per_channel, dtype):
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(M * 7 + K + N)
    x = torch.randn(M, K, device="cuda", generator=gen).to(dtype)
    packed, scale, w = _weights(gen, N, K, per_channel)
    out = ops.w4a16_linear(x, packed, scale, N, per_channel)
    assert out.shape == (M, N) and out.dtype == dtype
    _check(out, *_product(x, w))
    assert torch.equal(out, ops.w4a16_linear(x, packed, scale, N, per_channel))     # the same bits in every run


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,I,per_channel", [(1, 4096, 12288, False), (1, 128, 1, False), (4, 2048, 768, True), (13, 128 * 11, 39, False),
                                               (24, 2560, 9728, True), (32, 12288, 100, False), (40, 512, 20, True)])
def test_gated(M, K, I, per_channel, dtype):
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(M + K + I)
    x = torch.randn(M, K, device="cuda", generator=gen).to(dtype)
    packed, scale, w = _weights(gen, 2 * I, K, per_channel)
    w *= 0.25
    scale = scale * 0.25
    out = ops.w4a16_gated_linear(x, packed, scale, I, per_channel)
    y, slack = _product(x, w)
    (g, u), (dg, du) = y.chunk(2, -1), slack.chunk(2, -1)
    act = g * torch.sigmoid(g)
    # |d silu| <= 1.1; the activation itself is a handful of fp32 operations, the exponential's argument good to half a step of g
    _check(out, act * u, 1.1 * dg * u.abs() + act.abs() * du + 1.1 * dg * du + (16 + g.abs()) * 2.0 ** -23 * (act * u).abs())


def test_tokens_do_not_mix():
    """Padding tokens and the tokens of other grid rows have no part in a token's sums: finite ones beside NaN and infinity, and each by itself."""
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(37, 1024, device="cuda", generator=gen).to(torch.bfloat16)
    x[3], x[20] = float("nan"), float("inf")
    packed, scale, w = _weights(gen, 77, 1024, False)
    whole = ops.w4a16_linear(x, packed, scale, 77)
    single = torch.cat([ops.w4a16_linear(x[m:m + 1], packed, scale, 77) for m in range(37)])
    fine = [m for m in range(37) if m not in (3, 20)]
    for out in (whole, single):
        _check(out[fine], *_product(x[fine], w))
        assert out[3].isnan().all() and not out[20].isfinite().any()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("per_channel", [False, True])
def test_numbers_of_very_different_size(per_channel, dtype, gated):
    """A token's largest number, met by codes of zero, hides nothing of numbers 2^-30 to 2^-100 times as large beside it."""
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(11)
    M, K, rows = 5, 1024, 64
    codes_zero = torch.zeros(K, dtype=torch.bool, device="cuda")
    codes_zero[5::128] = True
    x = torch.randn(M, K, device="cuda", generator=gen)
    x[1] *= 2.0 ** -40 if dtype == torch.bfloat16 else 2.0 ** -13
    x[2] *= 2.0 ** -100 if dtype == torch.bfloat16 else 2.0 ** -16
    x[3] *= 2.0 ** 90 if dtype == torch.bfloat16 else 1.0
    x[:, 5::128] = 60000.0
    x[4] = 0.0
    x = x.to(dtype)
    codes = torch.randint(-8, 8, (rows, K), device="cuda", generator=gen)
    codes[:, codes_zero] = 0
    packed = ((codes[:, 0::2] & 15) | ((codes[:, 1::2] & 15) << 4)).to(torch.uint8).contiguous()
    scale = torch.full((rows,), 2.0 ** -6, device="cuda")
    if not per_channel:
        packed, scale = packed.view(rows, K // 128, 64).transpose(0, 1).contiguous(), scale.expand(K // 128, rows).contiguous()
    ref, slack = _product(x.double() * ~codes_zero, codes.double() * 2.0 ** -6)
    if not gated:
        _check(ops.w4a16_linear(x, packed, scale, rows, per_channel), ref, slack)
        return
    small = (ref[[0, 1, 2, 4]], slack[[0, 1, 2, 4]])
    (g, u), (dg, du) = small[0].chunk(2, -1), small[1].chunk(2, -1)
    out = ops.w4a16_gated_linear(x, packed, scale, rows // 2, per_channel)[[0, 1, 2, 4]]
    act = g * torch.sigmoid(g)
    _check(out, act * u, 1.1 * dg * u.abs() + act.abs() * du + (16 + g.abs()) * 2.0 ** -23 * (act * u).abs() + 2.0 ** -126)


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities(dtype):
    """One infinity in a token: its sign times the code's, not a number where the code is zero; other tokens keep their bits."""
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(12)
    x = torch.randn(3, 512, device="cuda", generator=gen).to(dtype)
    packed, scale, w = _weights(gen, 96, 512, False)
    clean = ops.w4a16_linear(x, packed, scale, 96)
    x[1, 300] = -float("inf")
    out = ops.w4a16_linear(x, packed, scale, 96)
    c = w[:, 300]
    assert (c == 0).any() and out[1, c == 0].isnan().all()
    assert torch.equal(out[1, c != 0].double(), -float("inf") * c[c != 0].sign())
    ref, slack = _product(x[[0, 2]], w)
    _check(out[[0, 2]], ref, slack)
    _check(clean[[0, 2]], ref, slack)


@pytest.mark.parametrize("layout", ["strided rows", "odd stride", "misaligned", "columns"])
def test_linear_takes_any_layout_of_tokens(layout):
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(6)
    dense = torch.randn(6, 512, device="cuda", generator=gen).to(torch.bfloat16)
    if layout == "strided rows":
        x = torch.zeros(6, 1024, dtype=dense.dtype, device="cuda")[:, 8:520].copy_(dense)
    elif layout == "odd stride":
        x = torch.zeros(6, 515, dtype=dense.dtype, device="cuda")[:, :512].copy_(dense)
    elif layout == "misaligned":
        x = torch.zeros(6 * 512 + 1, dtype=dense.dtype, device="cuda")[1:].view(6, 512).copy_(dense)
    else:
        x = torch.zeros(512, 6, dtype=dense.dtype, device="cuda").t().copy_(dense)
    packed, scale, _ = _weights(gen, 40, 512, False)
    assert torch.equal(ops.w4a16_linear(x, packed, scale, 40), ops.w4a16_linear(dense, packed, scale, 40))


def test_linear_of_nothing_and_refusals():
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(7)
    packed, scale, _ = _weights(gen, 8, 256, False)
    x = torch.randn(2, 256, device="cuda").to(torch.bfloat16)
    assert ops.w4a16_linear(x[:0], packed, scale, 8).shape == (0, 8)
    assert ops.w4a16_linear(x, packed[:, :0], scale[:, :0], 0).shape == (2, 0)
    for bad, match in [((x.cpu(), packed, scale, 8), "CUDA"), ((x.float(), packed, scale, 8), "bfloat16 or float16"), ((x[0], packed, scale, 8), "2D"),
                       ((x[:, :192].contiguous(), packed, scale, 8), "divisible"), ((x[:, :0], packed, scale, 8), "divisible"),
                       ((x, packed, scale, 9), "bytes"), ((x, packed, scale[:1], 8), "scale_b"), ((x, packed, scale.half(), 8), "float32"),
                       ((x, packed.to(torch.int8), scale, 8), "uint8"), ((x, packed.cpu(), scale, 8), "device"),
                       ((x, packed, scale.T.contiguous().T, 8), "contiguous"), ((x.clone().requires_grad_(), packed, scale, 8), "backward")]:
        with pytest.raises(RuntimeError, match=match):
            ops.w4a16_linear(*bad)
    with pytest.raises(RuntimeError, match="bytes"):
        ops.w4a16_gated_linear(x, packed, scale, 8)


def test_streams_and_graphs():
    """Two captured graphs and an eager call of the same shapes side by side: nothing is shared between calls."""
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(8)
    packed, scale, _ = _weights(gen, 512, 12288, False)
    xs = [torch.randn(16, 12288, device="cuda", generator=gen).to(torch.bfloat16) for _ in range(3)]
    want = [ops.w4a16_linear(x, packed, scale, 512) for x in xs]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for x, st in zip(xs, streams):
        st.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            outs.append(ops.w4a16_linear(x, packed, scale, 512))
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        eager = ops.w4a16_linear(xs[2], packed, scale, 512)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[2])
