"""GPU: a decoding cache that cannot take a step's tokens keeps its lengths and rows, and says so."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _cache(lengths, batch=3, tokens=32):
    from fp8_inference_toolkit_b200.qwen3 import DecodeCache, Qwen3Config

    cache = DecodeCache(Qwen3Config(layers=2, kv_heads=2, head_dim=64), batch, tokens, page_size=16)
    cache.lengths.copy_(torch.tensor(lengths))
    gen = torch.Generator(device="cuda").manual_seed(1)
    cache.pending = [tuple(torch.randn(batch, 4, 2, 64, device="cuda", generator=gen).to(torch.bfloat16) for _ in range(2)) for _ in range(2)]
    return cache


@pytest.mark.parametrize("case", ["full", "count", "negative count", "row", "page"])
def test_a_sequence_that_cannot_take_its_tokens(case):
    from fp8_inference_toolkit_b200 import ops

    cache = _cache([5, 30 if case == "full" else 14, 20])
    rows, counts, select = cache.pending, None, None
    if case == "page":
        cache.block_table[1, 1] = 6
    elif case == "row":
        counts = torch.tensor([4, 3, 2], dtype=torch.int32, device="cuda")
        select = torch.tensor([[0, 1, 2, 3], [0, 2, 4, 0], [1, 3, 9, 9]], dtype=torch.int32, device="cuda")
    elif "count" in case:
        counts = torch.tensor([4, 5 if case == "count" else -1, 4], dtype=torch.int32, device="cuda")
    before = cache.lengths.tolist()
    ops.check_status()
    cache.commit(counts, select)
    taken = [4, 0, 2 if case == "row" else 4]
    assert cache.lengths.tolist() == [n + t for n, t in zip(before, taken)]
    with pytest.raises(RuntimeError, match="out of range"):
        ops.check_status()
    for held, new in zip(zip(cache.k, cache.v), rows):
        for cached, value in zip(held, new):
            want = torch.zeros_like(cached)
            for b in (0, 2):
                for i in range(taken[b]):
                    at = before[b] + i
                    want[int(cache.block_table[b, at // 16]), at % 16] = value[b, i if select is None else int(select[b, i])]
            assert torch.equal(cached, want)


def test_a_prompt_for_a_sequence_that_is_not_empty():
    """It takes none of its tokens and says so; the others take theirs, and one without tokens is no fault."""
    from fp8_inference_toolkit_b200 import ops
    from fp8_inference_toolkit_b200.qwen3 import DecodeCache, Qwen3Config, Qwen3Prefill

    cfg = Qwen3Config(hidden=512, layers=1, q_heads=4, kv_heads=2, head_dim=128, inter=512, vocab=64)
    model, cache = Qwen3Prefill(cfg), DecodeCache(cfg, 3, 32, page_size=16)
    ids = torch.arange(24, device="cuda").view(3, 8)
    model.prefill(ids, cache, torch.tensor([8, 0, 5], dtype=torch.int32, device="cuda"))
    ops.check_status()
    held = cache.k[0].clone()
    model.prefill(ids.flip(1), cache, torch.tensor([0, 8, 8], dtype=torch.int32, device="cuda"))
    assert cache.lengths.tolist() == [8, 8, 5]
    assert torch.equal(cache.k[0][:2], held[:2]) and torch.equal(cache.k[0][4:], held[4:]) and cache.k[0][2, :8].any()
    with pytest.raises(RuntimeError, match="out of range"):
        ops.check_status()
