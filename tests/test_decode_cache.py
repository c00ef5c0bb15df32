"""CPU: what a decoding cache takes as a step, and what it forgets (stand-ins for the layers and for the append)."""
import pytest
import torch
from torch import nn


class _Layer(nn.Module):
    """A layer of one key head of 8 that attends, or raises before or after it does."""

    def __init__(self, fails=None):
        super().__init__()
        self.fails = fails

    def _maybe(self, when):
        if self.fails == when:
            raise RuntimeError("the layer failed")

    def step(self, x, positions, freqs, attend):
        self._maybe("before")
        heads = x[:, :, None]
        attend(heads, heads, heads)
        self._maybe("after")
        return x

    def forward(self, x, cos, sin, attend):
        self._maybe("before")
        return x


@pytest.fixture
def decode(lib_built, monkeypatch):
    """(model of the given layers, cache, what was appended: layer's cache, rows and counts)."""
    from fp8_inference_toolkit_b200 import ops
    from fp8_inference_toolkit_b200.qwen3 import DecodeCache, Qwen3Config, Qwen3Prefill

    appended = []
    monkeypatch.setattr(ops, "kv_cache_append_", lambda kc, vc, k, v, table, lengths, select=None, counts=None: appended.append((kc, k, counts)))
    monkeypatch.setattr(ops, "tree_attention", lambda q, *a, **kw: q)

    def make(*layers, batch=2, tokens=12, page_size=4):
        cfg = Qwen3Config(hidden=8, layers=len(layers), q_heads=1, kv_heads=1, head_dim=8, inter=8, vocab=16)
        model = Qwen3Prefill.__new__(Qwen3Prefill)
        nn.Module.__init__(model)
        model.cfg, model.embed, model.blocks, model.norm = cfg, nn.Embedding(16, 8), nn.ModuleList(layers), nn.Identity()
        return model, DecodeCache(cfg, batch, tokens, page_size, device="cpu")

    return make, appended


IDS = torch.zeros(2, 3, dtype=torch.int64)


@pytest.mark.parametrize("when", ["before", "after"])
@pytest.mark.parametrize("layer", [0, 1, 2])
def test_a_step_that_raised_cannot_be_committed(decode, layer, when):
    make, appended = decode
    model, cache = make(_Layer(), _Layer(), _Layer())
    model.step(IDS, cache)
    model.blocks[layer].fails = when
    with pytest.raises(RuntimeError, match="failed"):
        model.step(IDS, cache)
    with pytest.raises(RuntimeError, match="no step"):
        cache.commit()
    assert not appended and cache.lengths.tolist() == [0, 0]
    model.blocks[layer].fails = None
    model.step(IDS, cache)
    cache.commit()
    assert len(appended) == 3 and cache.lengths.tolist() == [3, 3]


@pytest.mark.parametrize("fails", [None, "before"])
def test_prefill_forgets_the_step_before_it(decode, fails):
    make, appended = decode
    model, cache = make(_Layer(), _Layer())
    model.step(IDS, cache)
    model.blocks[1].fails = fails
    if fails:
        with pytest.raises(RuntimeError, match="failed"):
            model.prefill(IDS, cache)
    else:
        model.prefill(IDS, cache)
    with pytest.raises(RuntimeError, match="no step"):
        cache.commit()
    assert not appended
