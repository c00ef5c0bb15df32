"""GPU: the decoding path of the Qwen3-shaped model near enough to the same layers in 64 bits to tell them from wrong ones: a lost mask, position,
norm, rotation or cached token, gate for up, other heads.

The embedding is small, so that the layers make the result, and the norms' weights are not one.  Tolerance of each token's 2-norm: the path
rounds to bf16 at 13 places a layer (two norms at two places each, QKV, query and key norm, rotation, attention and its weights, output
projection, both sums, gated product, down projection).  A rounding is off by at most half a step, 2^-8 of a value; as independent uniform
errors, sqrt(13 * LAYERS) * 2^-8 / sqrt(3) together.  Three times that is allowed; the references that are wrong on purpose have to be off by
three times the tolerance."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
LAYERS = 2
NEAR = 3 * math.sqrt(13 * LAYERS) * 2.0 ** -8 / math.sqrt(3)


def _model(per_channel=False):
    from fp8_inference_toolkit_b200.qwen3 import Qwen3Config, Qwen3Prefill

    torch.manual_seed(0)
    cfg = Qwen3Config(hidden=1024, layers=LAYERS, q_heads=8, kv_heads=2, head_dim=128, inter=1536, vocab=512, rope_theta=1e6)
    model = Qwen3Prefill(cfg, device="cuda", per_channel=per_channel, seed=3)
    model.embed.weight.data.mul_(0.02)
    for name, p in model.named_parameters():
        if "ln" in name or "norm" in name:
            p.data.copy_(torch.rand(p.shape, device="cuda") + 0.5)
    return model


def _weight(lin):
    """[N, K] in 64 bits."""
    codes = lin.weight_int4.to(torch.int64)
    codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    codes = torch.where(codes > 7, codes - 16, codes).double() * lin.weight_scale.double()[..., None]
    return codes if codes.dim() == 2 else codes.transpose(0, 1).flatten(1)


def _reference(model, ids, positions, visible, cached=None, wrong=""):
    """One sequence: ids and positions [n], visible [n, m + n] over m cached tokens (``cached``: keys and values [m, kv_heads, D] of each layer) and
    these -> (hidden [n, hidden], keys and values [n, kv_heads, D] of each layer) in 64 bits."""
    cfg, n = model.cfg, len(ids)
    x, made = model.embed.weight[ids].double(), []
    f = cfg.rope_theta ** (-torch.arange(0, cfg.head_dim, 2, dtype=torch.float64, device="cuda") / cfg.head_dim)
    c, s = ((positions.double()[:, None] * f).cos()[:, None], (positions.double()[:, None] * f).sin()[:, None])

    def turn(y):
        a, b = y.chunk(2, -1)
        return y if wrong == "rotation" else torch.cat((a * c - b * s, b * c + a * s), -1)

    def norm(y, m):
        y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + m.eps)
        return y if wrong == "norm weights" else y * m.weight.double()

    for layer, blk in enumerate(model.blocks):
        qkv = (norm(x, blk.ln1) @ _weight(blk.qkv).T).view(n, -1, cfg.head_dim)
        q, k, v = qkv.split([cfg.q_heads, cfg.kv_heads, cfg.kv_heads], 1)
        if wrong != "head norms":
            q, k = norm(q, blk.q_norm), norm(k, blk.k_norm)
        q, k = turn(q), turn(k)
        made.append((k, v))
        if cached is not None:
            k, v = (torch.cat((old.double(), new)) for old, new in zip(cached[layer], (k, v)))
        times = cfg.q_heads // cfg.kv_heads
        k, v = (t.repeat(1, times, 1) if wrong == "heads" else t.repeat_interleave(times, 1) for t in (k, v))
        p = torch.softmax((torch.einsum("ihd,jhd->hij", q, k) * cfg.head_dim ** -0.5).masked_fill(~visible, -math.inf), -1)
        x = x + torch.einsum("hij,jhd->ihd", p, v).reshape(n, -1) @ _weight(blk.o).T
        g, u = (norm(x, blk.ln2) @ _weight(blk.gate_up).T).chunk(2, -1)
        if wrong == "gate for up":
            g, u = u, g
        x = x + (g * torch.sigmoid(g) * u) @ _weight(blk.down).T
    return norm(x, model.norm), made


def _off(out, ref):
    """Of the token that is off most, by its 2-norm."""
    out, ref = out.double().flatten(1), ref.flatten(1)
    return ((out - ref).norm(dim=1) / ref.norm(dim=1)).max()


def _chain(n):
    return torch.ones(n, n, dtype=torch.bool, device="cuda").tril()


def _tree(parents):
    mask = torch.zeros(len(parents), len(parents), dtype=torch.bool)
    for i, parent in enumerate(parents):
        if parent >= 0:
            mask[i] = mask[parent]
        mask[i, i] = True
    return mask.cuda()


def _held(cache, b, n):
    """Keys and values [n, kv_heads, D] of sequence b's first n tokens, layer by layer."""
    pages = cache.block_table[b].long()
    return [tuple(c[layer][pages].flatten(0, 1)[:n] for c in (cache.k, cache.v)) for layer in range(LAYERS)]


def _sees_all(n, mask):
    """[T, n + T]: n cached tokens, and the mask."""
    return torch.cat((torch.ones(len(mask), n, dtype=torch.bool, device="cuda"), mask), 1)


def _tokens(seed, *shape):
    return torch.randint(0, 512, shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


@pytest.mark.parametrize("per_channel", [False, True])
def test_chain_token_and_tree(per_channel):
    """A chain of ten from nothing, a token, a tree of which a path is kept, a token: each against the whole text so far."""
    from fp8_inference_toolkit_b200 import ops
    from fp8_inference_toolkit_b200.qwen3 import DecodeCache

    model = _model(per_channel)
    cache = DecodeCache(model.cfg, 2, 40, page_size=16)
    texts = [torch.empty(0, dtype=torch.int64, device="cuda") for _ in range(2)]

    def chain(ids):
        out = model.step(ids, cache)
        for b in range(2):
            whole = torch.cat((texts[b], ids[b]))
            n = len(whole)
            ref, _ = _reference(model, whole, torch.arange(n, device="cuda"), _chain(n))
            assert _off(out[b], ref[-ids.shape[1]:]) <= NEAR

    ids = _tokens(1, 2, 10)
    chain(ids)
    cache.commit(torch.tensor([10, 7], dtype=torch.int32, device="cuda"))
    texts = [ids[0], ids[1, :7]]
    ids = _tokens(2, 2, 1)
    chain(ids)
    cache.commit()
    texts = [torch.cat((t, i)) for t, i in zip(texts, ids)]
    ids, mask = _tokens(3, 2, 5), _tree([-1, 0, 0, 2, -1])
    out = model.step(ids, cache, mask)
    for b in range(2):
        n = len(texts[b])
        visible = torch.zeros(n + 5, n + 5, dtype=torch.bool, device="cuda")
        visible[:n, :n], visible[n:] = _chain(n), _sees_all(n, mask)
        positions = torch.cat((torch.arange(n, device="cuda"), n + mask.sum(-1) - 1))
        args = model, torch.cat((texts[b], ids[b])), positions, visible
        ref = _reference(*args)[0][n:]
        assert _off(out[b], ref) <= NEAR
        # what this has to tell apart
        as_chain, lost, first_lost = visible.clone(), visible.clone(), visible.clone()
        as_chain[n:, n:] = _chain(5)
        lost[n:, n - 1] = False
        first_lost[n:, 0] = False
        wrongs = [_reference(*args, wrong=w) for w in ("rotation", "norm weights", "head norms", "heads", "gate for up")]
        wrongs += [_reference(*args[:3], v) for v in (as_chain, lost, first_lost)]
        wrongs.append(_reference(*args[:2], torch.arange(n + 5, device="cuda"), visible))
        assert all(_off(w[n:], ref) > 3 * NEAR for w, _ in wrongs), [_off(w[n:], ref).item() for w, _ in wrongs]
    cache.commit(torch.tensor([3, 1], dtype=torch.int32, device="cuda"), torch.tensor([[0, 2, 3, 0, 0], [4, 0, 0, 0, 0]], dtype=torch.int32, device="cuda"))
    texts = [torch.cat((texts[0], ids[0, [0, 2, 3]])), torch.cat((texts[1], ids[1, [4]]))]
    chain(_tokens(4, 2, 2))
    ops.check_status()


@pytest.mark.parametrize("per_channel,act_bits", [(False, 4), (True, 4), (False, 16), (True, 16)])
def test_step_after_a_prompt(per_channel, act_bits, monkeypatch):
    """A ragged batch of prompts, then a tree: against the layers over the keys and values that the prompts left; with 16-bit activations these are
    the prompt's in 64 bits, too."""
    from fp8_inference_toolkit_b200 import ops
    from fp8_inference_toolkit_b200.qwen3 import DecodeCache

    monkeypatch.setenv("INT4TC_ACT_BITS", str(act_bits))
    model = _model(per_channel)
    cache = DecodeCache(model.cfg, 2, 64, page_size=16)
    ids, lengths = _tokens(5, 2, 40), [40, 25]
    out = model.prefill(ids, cache, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    if act_bits == 16:
        for b, n in enumerate(lengths):
            ref, made = _reference(model, ids[b, :n], torch.arange(n, device="cuda"), _chain(n))
            assert _off(out[b, :n], ref) <= NEAR
            for held, want in zip(_held(cache, b, n), made):
                assert all(_off(h, w) <= NEAR for h, w in zip(held, want))
    new, mask = _tokens(6, 2, 4), _tree([-1, 0, 0, 1])
    out = model.step(new, cache, mask)
    for b, n in enumerate(lengths):
        held = _held(cache, b, n)
        ref, _ = _reference(model, new[b], n + mask.sum(-1) - 1, _sees_all(n, mask), held)
        assert _off(out[b], ref) <= NEAR
        fewer = [tuple(t[1:] for t in kv) for kv in held]
        assert _off(_reference(model, new[b], n + mask.sum(-1) - 1, _sees_all(n - 1, mask), fewer)[0], ref) > NEAR
        assert _off(_reference(model, new[b], mask.sum(-1) - 1, _sees_all(n, mask), held)[0], ref) > 3 * NEAR
    ops.check_status()
