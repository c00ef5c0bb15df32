"""GPU: the decoding path of the Qwen3-shaped model (16-bit activations over the packed weights, rotary positions, paged cache, tree
attention) as a whole, against the same layers in 64 bits with the weights that the codes stand for.

Tolerance: the path rounds to bf16 (half a step 2^-8 of a value) at 11 places a layer (two norms at two places each, QKV, query and
key norm, rotation, attention and its weights, output projection, both sums, gated product, down projection); as relative errors of
the 2-norm these add up to at most 13 * 2^-8 a layer, and no operation of these layers is steeper than linear by much at N(0, 1)
inputs: twice that is allowed."""
import pytest
import torch

pytestmark = pytest.mark.gpu
LAYERS = 2


def _model(per_channel=False):
    from fp8_inference_toolkit_b200.qwen3 import Qwen3Config, Qwen3Prefill

    torch.manual_seed(0)
    cfg = Qwen3Config(hidden=1024, layers=LAYERS, q_heads=8, kv_heads=2, head_dim=128, inter=1536, vocab=512, rope_theta=1e6)
    return Qwen3Prefill(cfg, device="cuda", per_channel=per_channel, seed=3)


def _weight(lin):
    """[N, K] in 64 bits."""
    codes = lin.weight_int4.to(torch.int64)
    codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    codes = torch.where(codes > 7, codes - 16, codes).double() * lin.weight_scale.double()[..., None]
    return codes if codes.dim() == 2 else codes.transpose(0, 1).flatten(1)


def _norm(x, m):
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + m.eps) * m.weight.double()


def _reference(model, ids, positions, visible):
    """One sequence: ids and positions [n], visible [n, n] -> hidden [n, hidden] in 64 bits."""
    cfg = model.cfg
    n = len(ids)
    x = model.embed.weight[ids].double()
    f = cfg.rope_theta ** (-torch.arange(0, cfg.head_dim, 2, dtype=torch.float64, device="cuda") / cfg.head_dim)
    c, s = ((positions.double()[:, None] * f).cos()[:, None], (positions.double()[:, None] * f).sin()[:, None])

    def turn(y):
        a, b = y.chunk(2, -1)
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    for blk in model.blocks:
        qkv = (_norm(x, blk.ln1) @ _weight(blk.qkv).T).view(n, -1, cfg.head_dim)
        q, k, v = qkv.split([cfg.q_heads, cfg.kv_heads, cfg.kv_heads], 1)
        q, k = turn(_norm(q, blk.q_norm)), turn(_norm(k, blk.k_norm))
        k, v = (t.repeat_interleave(cfg.q_heads // cfg.kv_heads, 1) for t in (k, v))
        score = torch.einsum("ihd,jhd->hij", q, k) * cfg.head_dim ** -0.5
        p = torch.softmax(score.masked_fill(~visible, -float("inf")), -1)
        x = x + torch.einsum("hij,jhd->ihd", p, v).reshape(n, -1) @ _weight(blk.o).T
        g, u = (_norm(x, blk.ln2) @ _weight(blk.gate_up).T).chunk(2, -1)
        x = x + (g * torch.sigmoid(g) * u) @ _weight(blk.down).T
    return _norm(x, model.norm)


def _near(out, ref):
    rel = (out.double() - ref).norm() / ref.norm()
    assert rel <= 2 * 13 * LAYERS * 2.0 ** -8, rel


def _chain(n):
    return torch.ones(n, n, dtype=torch.bool, device="cuda").tril()


@pytest.mark.parametrize("per_channel", [False, True])
def test_tokens_chains_and_trees(per_channel):
    """Two sequences from nothing: a chain of seven, single tokens, a tree of which a path is kept, and what follows it."""
    from fp8_inference_toolkit_b200 import ops
    from fp8_inference_toolkit_b200.qwen3 import DecodeCache

    model = _model(per_channel)
    cache = DecodeCache(model.cfg, 2, 60, page_size=16)
    gen = torch.Generator(device="cuda").manual_seed(1)
    texts = [torch.empty(0, dtype=torch.int64, device="cuda") for _ in range(2)]

    def tokens(T):
        return torch.randint(0, 512, (2, T), device="cuda", generator=gen)

    def check_chain(ids, out):
        for b in range(2):
            whole = torch.cat((texts[b], ids[b]))
            n = len(whole)
            _near(out[b], _reference(model, whole, torch.arange(n, device="cuda"), _chain(n))[-ids.shape[1]:])

    ids = tokens(7)
    check_chain(ids, model.step(ids, cache))
    cache.commit(torch.tensor([7, 4], dtype=torch.int32, device="cuda"))
    texts = [ids[0], ids[1, :4]]
    for _ in range(3):
        ids = tokens(1)
        check_chain(ids, model.step(ids, cache))
        cache.commit()
        texts = [torch.cat((t, i)) for t, i in zip(texts, ids)]
    # node:     0  1  2  3  4
    parents = [-1, 0, 0, 2, -1]
    mask = torch.zeros(5, 5, dtype=torch.bool)
    for i, parent in enumerate(parents):
        if parent >= 0:
            mask[i] = mask[parent]
        mask[i, i] = True
    mask = mask.cuda()
    ids = tokens(5)
    out = model.step(ids, cache, mask)
    for b in range(2):
        n = len(texts[b])
        visible = torch.zeros(n + 5, n + 5, dtype=torch.bool, device="cuda")
        visible[:n, :n], visible[n:, :n], visible[n:, n:] = _chain(n), True, mask
        positions = torch.cat((torch.arange(n, device="cuda"), n + mask.sum(-1) - 1))
        _near(out[b], _reference(model, torch.cat((texts[b], ids[b])), positions, visible)[n:])
    # kept: 0, 2, 3 of the first, 4 of the second
    cache.commit(torch.tensor([3, 1], dtype=torch.int32, device="cuda"), torch.tensor([[0, 2, 3, 0, 0], [4, 0, 0, 0, 0]], dtype=torch.int32, device="cuda"))
    texts = [torch.cat((texts[0], ids[0, [0, 2, 3]])), torch.cat((texts[1], ids[1, [4]]))]
    assert cache.lengths.tolist() == [len(t) for t in texts]
    ids = tokens(2)
    check_chain(ids, model.step(ids, cache))
    with pytest.raises(RuntimeError, match="no step"):
        cache.commit()
        cache.commit()
    ops.check_status()


def test_prefill_then_step():
    """A ragged batch of prompts (the 4-bit activations of the prefill path), then a token: the cache holds what the prompts' layers made."""
    from fp8_inference_toolkit_b200.qwen3 import DecodeCache

    model = _model()
    cache = DecodeCache(model.cfg, 2, 64, page_size=16)
    gen = torch.Generator(device="cuda").manual_seed(2)
    ids = torch.randint(0, 512, (2, 40), device="cuda", generator=gen)
    counts = torch.tensor([40, 25], dtype=torch.int32, device="cuda")
    out = model.prefill(ids, cache, counts)
    assert cache.lengths.tolist() == [40, 25]
    # prompts one by one give the same rows: padding has no part
    other = DecodeCache(model.cfg, 1, 64, page_size=16)
    alone = model.prefill(ids[1:, :25], other)
    # (tiles of another row count, split K: the same values up to the roundings of the path)
    assert (alone[0].float() - out[1, :25].float()).norm() <= 2 * 13 * LAYERS * 2.0 ** -8 * alone.float().norm()
    for layer in range(LAYERS):
        for c, o in ((cache.k, other.k), (cache.v, other.v)):
            mine = c[layer][cache.block_table[1].long()].flatten(0, 1)
            assert not mine[25:].any() and (mine[:25].float() - o[layer].flatten(0, 1)[:25].float()).norm() <= 2 * 13 * LAYERS * 2.0 ** -8 * mine.float().norm()
    # forward() turns by bf16 tables (half a step 2^-8 of cosine and sine): as near
    assert (model(ids).float() - out.float())[0].norm() <= 2 * 14 * LAYERS * 2.0 ** -8 * out[0].float().norm()
    token = torch.randint(0, 512, (2, 1), device="cuda", generator=gen)
    assert model.step(token, cache).isfinite().all()


def test_step_in_a_graph():
    """A captured step and commit, replayed: lengths move on the device, and the results are those of eager steps."""
    from fp8_inference_toolkit_b200.qwen3 import DecodeCache

    model = _model()
    gen = torch.Generator(device="cuda").manual_seed(4)
    first, tokens = torch.randint(0, 512, (2, 9), device="cuda", generator=gen), torch.randint(0, 512, (5, 2, 1), device="cuda", generator=gen)
    caches = [DecodeCache(model.cfg, 2, 40, page_size=8) for _ in range(2)]
    for cache in caches:
        model.step(first, cache)
        cache.commit()
    eager = []
    for ids in tokens:
        eager.append(model.step(ids, caches[0]))
        caches[0].commit()
    ids, side, graph = tokens[0].clone(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        out = model.step(ids, caches[1])
        caches[1].commit()
    torch.cuda.synchronize()
    for t, want in zip(tokens, eager):
        ids.copy_(t)
        graph.replay()
        assert torch.equal(out, want)
    assert torch.equal(caches[0].lengths, caches[1].lengths) and torch.equal(caches[0].k[1], caches[1].k[1])


@pytest.mark.parametrize("per_channel,smooth", [(False, False), (True, False), (False, True)])
def test_linear_module_with_16_bit_activations(per_channel, smooth, monkeypatch):
    from fp8_inference_toolkit_b200.linear import W4A4Linear

    lin = torch.nn.Linear(512, 96, bias=True, device="cuda", dtype=torch.bfloat16)
    x = torch.randn(2, 3, 512, device="cuda").to(torch.bfloat16)
    stats = {"calibration_stats": {"l": {"input_absmax": x.flatten(0, 1).abs().amax(0).float()}}, "layer_name": "l"} if smooth else {}
    monkeypatch.setenv("INT4TC_ACT_BITS", "16")
    m = W4A4Linear.from_linear(lin, per_channel=per_channel, **stats)
    assert m.method.act_bits == 16
    out = m(x)
    v = x.double() if not smooth else (x / m.smooth_scale).double()
    w = _weight(m)
    ref = v @ w.T
    half = 2.0 ** -8
    slack = (512 / 16 + 512 / 128 + 16) * 2.0 ** -23 * (v.abs() @ w.abs().T)
    bound = half * (ref.abs() + slack) + slack
    total = ref + m.bias.double()
    assert ((out.double() - total).abs() <= bound + half * (total.abs() + bound)).all()
    for bad in (dict(act_bits=8), dict(act_bits=16, asymmetric=True), dict(act_bits=16, clip_ratio=0.9)):
        with pytest.raises(ValueError):
            W4A4Linear(128, 8, device="cuda", **bad)
