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


def _cache(make, lengths, tokens=12):
    model, cache = make(_Layer(), _Layer(), batch=len(lengths), tokens=tokens)
    cache.lengths.copy_(torch.tensor(lengths))
    return model, cache


@pytest.mark.parametrize("lengths,counts,taken", [
    ([0, 5], None, [3, 3]), ([9, 10], None, [3, -1]), ([12, 11], [0, 1], [0, 1]), ([12, 11], [1, 2], [-1, -1]), ([0, 0], [4, -1], [-1, -1]),
    ([-1, 13], [1, 0], [-1, 0]), ([-2, 2 ** 31 - 1], [3, 3], [-1, -1]),
])
def test_lengths_count_what_was_appended(decode, lengths, counts, taken):
    """Full sequences, counts out of range and lengths out of range: such a sequence takes nothing and is reported by its count of -1."""
    make, appended = decode
    model, cache = _cache(make, lengths)
    model.step(IDS, cache)
    cache.commit(None if counts is None else torch.tensor(counts, dtype=torch.int32))
    assert [c.tolist() for _, _, c in appended] == [taken] * 2
    assert cache.lengths.tolist() == [n + max(0, t) for n, t in zip(lengths, taken)] and cache.lengths.dtype == torch.int32


@pytest.mark.parametrize("counts,taken,tokens", [(None, [3, 3], 12), ([3, 0], [3, 0], 12), ([4, 2], [0, 2], 12), ([-1, 1], [0, 1], 12), (None, [0, 0], 0)])
def test_lengths_count_what_a_prompt_appended(decode, counts, taken, tokens):
    make, _ = decode
    model, cache = _cache(make, [0, 0], tokens)
    model.prefill(IDS, cache, None if counts is None else torch.tensor(counts, dtype=torch.int32))
    assert cache.lengths.tolist() == taken


def test_pages_and_rows_that_do_not_exist(decode):
    make, appended = decode
    model, cache = _cache(make, [4, 3])
    cache.block_table[0, 1], cache.block_table[1, 2] = -1, 6       # 6 pages there are; the second page of sequence 1 is the last it needs
    model.step(IDS, cache)
    cache.commit()
    assert appended[0][2].tolist() == [-1, 3] and cache.lengths.tolist() == [4, 6]
    model.step(IDS, cache)
    cache.commit(torch.tensor([0, 2], dtype=torch.int32), torch.tensor([[9, 9, 9], [0, 2, 9]], dtype=torch.int32))
    assert appended[-1][2].tolist() == [0, 2] and cache.lengths.tolist() == [4, 8]
    cache.block_table[1, 2] = 5
    model.step(IDS, cache)
    cache.commit(torch.tensor([0, 2], dtype=torch.int32), torch.tensor([[0, 0, 0], [0, 3, 0]], dtype=torch.int32))
    assert appended[-1][2].tolist() == [0, -1] and cache.lengths.tolist() == [4, 8]


def test_a_cache_without_room(decode):
    make, appended = decode
    model, cache = _cache(make, [0, 0], tokens=0)
    model.step(IDS, cache)
    cache.commit()
    assert appended[0][2].tolist() == [-1, -1] and cache.lengths.tolist() == [0, 0]


def test_counts_and_rows_of_another_kind_are_refused(decode):
    make, appended = decode
    model, cache = _cache(make, [0, 0])
    model.step(IDS, cache)
    for counts, select in [(torch.ones(2), None), (torch.ones(1, dtype=torch.int32), None), (None, torch.zeros(2, 3)),
                           (None, torch.zeros(2, 2, dtype=torch.int32)), (None, torch.zeros(1, 3, dtype=torch.int32))]:
        with pytest.raises(RuntimeError, match="counts must be" if counts is not None else "select must be"):
            cache.commit(counts, select)
    assert not appended and cache.lengths.tolist() == [0, 0]
    cache.commit()
    assert cache.lengths.tolist() == [3, 3]


def test_prompts_go_into_empty_sequences(decode, monkeypatch):
    """A prompt's positions begin at 0 and it sees itself only: a sequence that holds tokens takes none; without tokens it is left alone."""
    make, _ = decode
    model, cache = _cache(make, [4, 0])
    model.prefill(IDS, cache)
    assert cache.lengths.tolist() == [4, 3]
    model.prefill(IDS, cache, torch.tensor([0, 1], dtype=torch.int32))
    assert cache.lengths.tolist() == [4, 3]
    asked = []
    monkeypatch.setattr(type(cache), "append", lambda self, layer, k, v, counts=None, select=None: asked.append(counts.tolist()))
    monkeypatch.setattr(_Layer, "forward", lambda self, x, cos, sin, attend: attend(self, x))
    monkeypatch.setattr(_Layer, "_turned_heads", lambda self, qkv, positions, freqs: (qkv[:, None],) * 3, raising=False)
    cache.lengths.copy_(torch.tensor([0, 1]))
    model.prefill(IDS, cache, torch.tensor([2, 1], dtype=torch.int32))
    assert asked and set(map(tuple, asked)) == {(2, -1)} and cache.lengths.tolist() == [2, 1]
    asked.clear()
    model.prefill(IDS, cache, torch.tensor([0, 0], dtype=torch.int32))
    assert set(map(tuple, asked)) == {(0, 0)} and cache.lengths.tolist() == [2, 1]
