"""GPU: linears of the Qwen3-shaped model that have smoothing factors or a bias (a calibrated layer put in, or loaded) keep them in prompts and steps."""
import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu
NAMES = ("qkv", "o", "gate_up", "down")


def _model(**kw):
    from fp8_inference_toolkit_b200.qwen3 import Qwen3Config, Qwen3Prefill

    torch.manual_seed(0)
    return Qwen3Prefill(Qwen3Config(hidden=1024, layers=2, q_heads=8, kv_heads=2, head_dim=128, inter=1536, vocab=64), seed=3, **kw)


def _ids():
    return torch.randint(0, 64, (2, 9), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))


def _step(model):
    from fp8_inference_toolkit_b200.qwen3 import DecodeCache

    return model.step(_ids(), DecodeCache(model.cfg, 2, 16, page_size=16))


@pytest.mark.parametrize("name", NAMES)
def test_smoothing_factors(name):
    """Factors of 4 are a fourth of the weights' scales, to the bit; the products of gate and up are rounded before SwiGLU where they have factors."""
    smoothed, scaled = _model(fused=False), _model(fused=False)
    wide = _model()
    for a, b, c in zip(smoothed.blocks, scaled.blocks, wide.blocks):
        for blk in (a, c):
            lin = getattr(blk, name)
            lin.smooth_scale = nn.Parameter(torch.full((lin.in_features,), 4.0, dtype=torch.bfloat16, device="cuda"), requires_grad=False)
        getattr(b, name).weight_scale.data.mul_(0.25)
    assert torch.equal(smoothed(_ids()), scaled(_ids()))
    got, want = _step(smoothed), _step(scaled)
    if name == "gate_up":
        # two more roundings a layer, of the two products (half a step 2^-8 each); the gated product is off by at most three of them
        assert (got.float() - want.float()).norm() <= 2 * 3 * 2 * 2.0 ** -8 * want.float().norm()
    else:
        assert torch.equal(got, want)
    # the fused layers leave their way where a factor would be lost (the output projection is a module there, too)
    if name != "o":
        assert torch.equal(wide(_ids()), scaled(_ids()))


@pytest.mark.parametrize("name", NAMES)
def test_biases(name):
    """A bias that is most of what a linear gives: lost, it would be the result that is off by its own size."""
    model, plain = _model(), _model()
    for blk in model.blocks:
        lin = getattr(blk, name)
        lin.bias = nn.Parameter(torch.randn(lin.out_features, device="cuda").mul(8).to(torch.bfloat16), requires_grad=False)
    got, without = _step(model).float(), _step(plain).float()
    # the same as the modules give with 16-bit activations, up to the roundings of the path (13 half steps of 2^-8 a layer, forward() one more)
    for blk in model.blocks:
        blk.fused = False
        for n in NAMES:
            getattr(blk, n).method.act_bits = 16
    want = model(_ids()).float()
    assert (got - want).norm() <= 2 * 14 * 2 * 2.0 ** -8 * want.norm() < (got - without).norm()
