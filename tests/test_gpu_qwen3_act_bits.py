"""GPU: a model whose linears keep 16-bit activations quantises none, in the prompt's layers as in a step's."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", ["4", "16"])
def test_prompts_follow_the_flag(bits, monkeypatch):
    from fp8_inference_toolkit_b200 import moe, ops
    from fp8_inference_toolkit_b200.qwen3 import DecodeCache, Qwen3Config, Qwen3Prefill

    monkeypatch.setenv("INT4TC_ACT_BITS", bits)
    cfg = Qwen3Config(hidden=1024, layers=2, q_heads=8, kv_heads=2, head_dim=128, inter=1536, vocab=64)
    model = Qwen3Prefill(cfg)
    calls = {"w4a16_linear": 0, "rmsnorm_int4_quant_grouped": 0, "moe_silu_mul_quant": 0, "linear": 0, "cutlass_int4_fused_grouped_gemm": 0}

    def counted(name, op):
        def call(*a, **kw):
            calls[name] += 1
            return op(*a, **kw)
        return call

    for name in calls:
        where = moe if name == "moe_silu_mul_quant" else ops
        monkeypatch.setattr(where, name, counted(name, getattr(where, name)))
    ids = torch.randint(0, 64, (2, 9), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    prompt = model(ids)
    cached = model.prefill(ids, DecodeCache(cfg, 2, 16, page_size=16))
    quantised = sum(n for name, n in calls.items() if name != "w4a16_linear")
    if bits == "16":
        assert quantised == 0 and calls["w4a16_linear"] == 2 * 4 * cfg.layers
        # the same layers as a step's, so the same values up to their roundings (bf16 half a step 2^-8 at 13 places a layer, as for a step;
        # forward() turns by bf16 tables: one place more)
        step = model.step(ids, DecodeCache(cfg, 2, 16, page_size=16)).float()
        for out in (prompt, cached):
            assert (out.float() - step).norm() <= 2 * 14 * cfg.layers * 2.0 ** -8 * step.norm()
    else:
        assert quantised > 0 and calls["w4a16_linear"] == 0
    ops.check_status()


@pytest.mark.parametrize("name", ["qkv", "gate_up", "down"])
def test_a_layer_given_a_linear_of_16_bits(name, monkeypatch):
    """A layer's own way is that of the linears it has, not of those it was built with."""
    from fp8_inference_toolkit_b200 import ops
    from fp8_inference_toolkit_b200.qwen3 import Qwen3Config, Qwen3Prefill

    cfg = Qwen3Config(hidden=1024, layers=1, q_heads=8, kv_heads=2, head_dim=128, inter=1536, vocab=64)
    model = Qwen3Prefill(cfg)
    getattr(model.blocks[0], name).method.act_bits = 16
    calls, op = [], ops.w4a16_linear
    monkeypatch.setattr(ops, "w4a16_linear", lambda *a: calls.append(1) or op(*a))
    assert model(torch.arange(9, device="cuda").view(1, 9)).isfinite().all() and len(calls) == 1
