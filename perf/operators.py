"""The operators of a decoding step over 4-bit weights and a paged cache, as timed cases.

``listed()`` names typical points, ``draw()`` spreads over the ranges around them.  ``run()`` is one call of an operator: of the
framework's entry point where ``own`` is true, else the same mathematics in elementary torch operations (32 bits, rounded
once at the end).  ``exact()`` states the operators in 64 bits.
"""
import math
import random

import torch

own = False

GROUP = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one user decoding: the fused QKV projection of one token, bound by latency
        {"name": "linear_decode_1", "op": "linear", "M": 1, "K": 4096, "N": 6144, "scales": "group", "dtype": "bf16"},
        # a tree of sixteen drafts through the long-K down projection
        {"name": "linear_drafts_16", "op": "linear", "M": 16, "K": 12288, "N": 4096, "scales": "group", "dtype": "bf16"},
        # one token through gate and up projection and SwiGLU, the widest matrix of the model: weight bytes count
        {"name": "gated_decode_1", "op": "gated", "M": 1, "K": 4096, "N": 12288, "scales": "group", "dtype": "bf16"},
        # three users' trees of eight drafts, another model's widths, one scale a row
        {"name": "gated_drafts_24", "op": "gated", "M": 24, "K": 2560, "N": 9728, "scales": "channel", "dtype": "fp16"},
        # query and key heads of a tree of sixteen drafts far into a text, in the fused QKV buffer's rows
        {"name": "rope_drafts_16", "op": "rope", "tokens": 16, "heads": 40, "D": 128, "R": 128, "skip": 8, "far": 32768, "interleaved": False,
         "factor": 1.0, "inverse": False, "dtype": "bf16"},
        # a prefill batch of prompts in a context stretched to four times its trained length
        {"name": "rope_prefill_8192", "op": "rope", "tokens": 8192, "heads": 40, "D": 128, "R": 128, "skip": 8, "far": 131072, "interleaved": False,
         "factor": 4.0, "inverse": False, "dtype": "bf16"},
        # back through neighbouring pairs on two thirds of a head of 96: the gradient, or keys moved to other positions
        {"name": "rope_partial_777", "op": "rope", "tokens": 777, "heads": 9, "D": 96, "R": 64, "skip": 0, "far": 8192, "interleaved": True,
         "factor": 1.0, "inverse": True, "dtype": "fp16"},
        # one user decoding plain tokens a page or so after a thousand others: latency
        {"name": "attend_decode_1", "op": "attend", "B": 1, "T": 1, "heads": 32, "kv_heads": 8, "D": 128, "page": 16, "length": 1001, "tree": False,
         "dtype": "bf16"},
        # one user's tree of sixteen drafts behind a long text
        {"name": "attend_tree_long", "op": "attend", "B": 1, "T": 16, "heads": 32, "kv_heads": 8, "D": 128, "page": 64, "length": 32765, "tree": True,
         "dtype": "bf16"},
        # a serving batch: trees of eight drafts behind texts of every length up to eight thousand
        {"name": "attend_tree_batch", "op": "attend", "B": 32, "T": 8, "heads": 32, "kv_heads": 8, "D": 128, "page": 16, "length": 8191, "tree": True,
         "dtype": "bf16"},
        # the accepted paths of a batch of trees of eight drafts go into their pages
        {"name": "append_accepted_32", "op": "append", "B": 32, "T": 8, "kv_heads": 8, "D": 128, "page": 16, "length": 1000, "accepted": True,
         "dtype": "bf16"},
        # a prompt's keys and values go into fresh pages
        {"name": "append_prompt_8000", "op": "append", "B": 1, "T": 8000, "kv_heads": 8, "D": 128, "page": 64, "length": 0, "accepted": False,
         "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["linear", "gated", "rope", "attend", "attend", "append"])
    dtype = rng.choice(["bf16", "fp16"])
    if op in ("linear", "gated"):
        scales = rng.choice(["group", "group", "channel"])
        K = GROUP * _log(rng, 4, 96) + (64 if scales == "channel" and rng.random() < 0.3 else 0)
        # rows of weights: any number, even odd ones, up to the widest matrix with its bytes below that one's
        N = min(_log(rng, 64, 12288), 12288 * 4096 // K)
        N = N if rng.random() < 0.3 else (N + 7) // 8 * 8
        return {"op": op, "M": _log(rng, 1, 32), "K": K, "N": N, "scales": scales, "dtype": dtype}
    if op == "rope":
        D = rng.choice([32, 64, 80, 96, 128, 128, 192, 256])
        R = rng.choice([D, D, D // 2, D // 4 * 2])
        heads = rng.randint(1, 64)
        tokens = min(_log(rng, 1, 8192), 8192 * 40 * 128 // (heads * D))
        return {"op": op, "tokens": tokens, "heads": heads, "D": D, "R": R, "skip": rng.choice([0, 0, 1, 8]), "far": _log(rng, 64, 1 << 20),
                "interleaved": rng.random() < 0.5, "factor": rng.choice([1.0, 1.0, 4.0, 8.0]), "inverse": rng.random() < 0.3, "dtype": dtype}
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    D = rng.choice([64, 80, 96, 128, 128])
    page = rng.choice([1, 8, 16, 16, 24, 64, 256])
    if op == "attend":
        T, group = (1 if rng.random() < 0.25 else _log(rng, 2, 64)), rng.choice([1, 2, 4, 4, 7, 8])
        B = _log(rng, 1, 64)
        most = min(32 * 8192 * 8 * 128 // (B * kv_heads * D), 32 * 8192 * 8 * 32 * 128 // (B * T * kv_heads * group * D), 32768)
        return {"op": op, "B": B, "T": T, "heads": kv_heads * group, "kv_heads": kv_heads, "D": D, "page": page, "length": _log(rng, 1, max(2, most)),
                "tree": T > 1 and rng.random() < 0.7, "dtype": dtype}
    accepted = rng.random() < 0.6
    B = _log(rng, 1, 64) if accepted else _log(rng, 1, 8)
    T = _log(rng, 1, 64) if accepted else _log(rng, 16, 8192 // B)
    return {"op": op, "B": B, "T": T, "kv_heads": kv_heads, "D": D, "page": page, "length": _log(rng, 1, 1000) if accepted else 0, "accepted": accepted,
            "dtype": dtype}


def _lengths(case):
    """Cache lengths of the batch, from an eighth of the longest to the longest."""
    B, most = case["B"], case["length"]
    return [most if B == 1 else most // 8 + (most - most // 8) * b // (B - 1) for b in range(B)]


def _counts(case):
    """How many of its T new tokens each sequence appends: all of a prompt, of a tree the accepted path (none up to all)."""
    B, T = case["B"], case["T"]
    return [(1 + 3 * b) % (T + 1) if case["accepted"] else T for b in range(B)]


def _activations(gen, M, K, dtype):
    """N(0, 1) with 8 channels per 4096 scaled by 20 (at least one)."""
    x = torch.randn(M, K, device="cuda", generator=gen)
    hot = torch.randperm(K, device="cuda", generator=gen)[: max(1, round(K * 8 / 4096))]
    x[:, hot] *= 20.0
    return x.to(dtype)


def _pages(gen, case, tokens):
    """A cache with room for `tokens` of each sequence, its pages handed out in no order, some of them nobody's."""
    each = -(-tokens // case["page"])
    count = case["B"] * each + 3
    table = torch.randperm(count, device="cuda", generator=gen)[: case["B"] * each].view(case["B"], each).to(torch.int32)
    shape = (count, case["page"], case["kv_heads"], case["D"])
    return (*(torch.randn(shape, device="cuda", generator=gen, dtype=DTYPES[case["dtype"]]) for _ in range(2)), table)


def _tree(rng, T):
    """Rows of a random tree's ancestor mask: a node sees itself, its parent, and so on up to a root."""
    rows = []
    for i in range(T):
        parent = rng.randint(max(-1, i - 4), i - 1)
        row = list(rows[parent]) if parent >= 0 else [False] * T
        row[i] = True
        rows.append(row)
    return rows


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] in ("linear", "gated"):
        M, K = case["M"], case["K"]
        rows = case["N"] * (2 if case["op"] == "gated" else 1)
        s["x"] = _activations(gen, M, K, dtype)
        w = torch.randn(rows, K, device="cuda", generator=gen) * 0.02
        if case["scales"] == "group":
            w = w.view(rows, K // GROUP, GROUP).transpose(0, 1)           # group-major: [G, rows, 128]
        scale = w.abs().amax(-1) / 7
        codes = torch.round(w / scale[..., None]).clamp(-8, 7).to(torch.int32) & 15
        s["w"] = (codes[..., 0::2] | codes[..., 1::2] << 4).to(torch.uint8).contiguous()
        s["scale"] = scale.contiguous()
        return s
    if case["op"] == "rope":
        tokens, heads, D, R = case["tokens"], case["heads"], case["D"], case["R"]
        s["buffer"] = torch.randn(tokens, (heads + case["skip"]) * D, device="cuda", generator=gen).to(dtype)
        s["x"] = s["buffer"].view(tokens, heads + case["skip"], D)[:, :heads]
        first = torch.randint(0, max(1, case["far"] - min(tokens, 1024)), ((tokens + 1023) // 1024,), device="cuda", generator=gen)
        at = torch.arange(tokens, device="cuda")
        s["positions"] = first[at // 1024] + at % 1024                   # texts of 1024 tokens, each from a place of its own
        f = 1e6 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
        if case["factor"] != 1.0:
            # blended by how often a pair turns within the trained length: slow pairs are stretched, fast ones stay
            turns = case["far"] / case["factor"] * f / (2 * math.pi)
            keep = ((turns - 1) / 31).clamp(0, 1)
            f = f * keep + f / case["factor"] * (1 - keep)
        s["freqs"], s["rescale"] = f, 1.0 if case["factor"] == 1.0 else 0.1 * math.log(case["factor"]) + 1.0
        return s
    B, T, Hk, D = case["B"], case["T"], case["kv_heads"], case["D"]
    order = list(range(B))
    rng.shuffle(order)
    lengths = _lengths(case)
    s["lengths"] = torch.tensor([lengths[b] for b in order], dtype=torch.int32, device="cuda")
    # new keys and values as slices of the fused projection's rows
    Hq = case.get("heads", Hk)
    qkv = torch.randn(B, T, (Hq + 2 * Hk) * D, device="cuda", generator=gen).to(dtype).view(B, T, Hq + 2 * Hk, D)
    s["q"], s["k"], s["v"] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], qkv[:, :, Hq + Hk:]
    if case["op"] == "attend":
        s["k_cache"], s["v_cache"], s["table"] = _pages(gen, case, max(1, case["length"]))
        s["mask"] = torch.tensor([_tree(rng, T) for _ in range(B)], device="cuda") if case["tree"] else None
        return s
    s["k_cache"], s["v_cache"], s["table"] = _pages(gen, case, case["length"] + T)
    s["counts"] = s["select"] = None
    if case["accepted"]:
        counts = _counts(case)
        s["counts"] = torch.tensor([counts[b] for b in order], dtype=torch.int32, device="cuda")
        paths = [sorted(rng.sample(range(T), counts[b])) + [0] * (T - counts[b]) for b in order]
        s["select"] = torch.tensor(paths, dtype=torch.int32, device="cuda")
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        from fp8_inference_toolkit_b200 import ops

        s, case = state, state["case"]
        if op == "linear":
            return ops.w4a16_linear(s["x"], s["w"], s["scale"], case["N"], case["scales"] == "channel")
        if op == "gated":
            return ops.w4a16_gated_linear(s["x"], s["w"], s["scale"], case["N"], case["scales"] == "channel")
        if op == "rope":
            return ops.rope(s["x"], s["positions"], s["freqs"], interleaved=case["interleaved"], scale=s["rescale"], inverse=case["inverse"])
        if op == "attend":
            return ops.tree_attention(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], tree_mask=s["mask"])
        ops.kv_cache_append_(s["k_cache"], s["v_cache"], s["k"], s["v"], s["table"], s["lengths"], counts=s["counts"], select=s["select"])
        return s["k_cache"], s["v_cache"]
    return {"linear": _linear, "gated": _gated, "rope": _rope, "attend": _attend, "append": _append}[op](state)


def _product(s):
    """x times the transposed weights in 32 bits: [M, rows]."""
    w = s["w"]
    codes = torch.stack((w & 15, w >> 4), -1).flatten(-2).to(torch.int32)
    codes = (codes ^ 8) - 8
    w = codes * s["scale"][..., None]                                     # [rows, K], or [G, rows, 128]
    if w.dim() == 3:
        w = w.transpose(0, 1).flatten(1)
    return s["x"].float() @ w.T


def _linear(s):
    return _product(s).to(s["x"].dtype)


def _gated(s):
    gate, up = _product(s).chunk(2, -1)
    return (gate / (1 + torch.exp(-gate)) * up).to(s["x"].dtype)


def _rope(s):
    case, x = s["case"], s["x"]
    R = case["R"]
    angle = s["positions"].double()[:, None] * s["freqs"]                 # [tokens, R / 2]; far positions need 64 bits
    cos, sin = (t.float()[:, None] * s["rescale"] for t in (angle.cos(), angle.sin()))
    if case["inverse"]:
        sin = -sin
    turned, rest = x[..., :R].float(), x[..., R:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if case["interleaved"] else turned.chunk(2, -1)
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((a, b), -1).flatten(-2) if case["interleaved"] else torch.cat((a, b), -1)
    return torch.cat((turned.to(x.dtype), rest), -1)


def _attend(s):
    case = s["case"]
    B, T, Hq, Hk, D = (case[k] for k in ("B", "T", "heads", "kv_heads", "D"))
    # [B, Hk, cache and new tokens, D]
    k, v = (torch.cat((cache[s["table"]].flatten(1, 2), new), 1).transpose(1, 2).float() for cache, new in ((s["k_cache"], s["k"]), (s["v_cache"], s["v"])))
    room = k.shape[2] - T
    q = s["q"].float().view(B, T, Hk, Hq // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)
    old = (torch.arange(room, device=q.device) < s["lengths"][:, None])[:, None].expand(B, T, room)
    new = torch.ones(T, T, dtype=torch.bool, device=q.device).tril().expand(B, T, T) if s["mask"] is None else s["mask"]
    seen = torch.cat((old, new), -1)[:, None, None]                       # [B, 1, 1, T, cache and new tokens]
    score = (q @ k.transpose(2, 3) * D ** -0.5).view(B, Hk, Hq // Hk, T, room + T)
    score = torch.where(seen, score, -math.inf)
    weight = torch.exp(score - score.amax(-1, keepdim=True))
    weight = weight / weight.sum(-1, keepdim=True)
    out = (weight.flatten(2, 3) @ v).view(B, Hk, Hq // Hk, T, D)
    return out.permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D).to(s["q"].dtype)


def _append(s):
    case = s["case"]
    B, T, page = case["B"], case["T"], case["page"]
    i = torch.arange(T, device="cuda").expand(B, T)
    at = s["lengths"][:, None].long() + i
    slot = s["table"].long().gather(1, at // page) * page + at % page     # [B, T]
    take = i if s["select"] is None else s["select"].long()
    rows = torch.arange(B, device="cuda")[:, None]
    k, v = s["k"][rows, take], s["v"][rows, take]
    if s["counts"] is not None:
        kept = i < s["counts"][:, None]
        slot, k, v = slot[kept], k[kept], v[kept]
    s["k_cache"].flatten(0, 1)[slot] = k
    s["v_cache"].flatten(0, 1)[slot] = v
    return s["k_cache"], s["v_cache"]


def work(case):
    op = case["op"]
    if op in ("linear", "gated"):
        M, K, N = case["M"], case["K"], case["N"]
        rows = N * (2 if op == "gated" else 1)
        scales = K // GROUP if case["scales"] == "group" else 1
        return {"bytes": rows * K // 2 + 4 * rows * scales + 2 * M * K + 2 * M * N, "flops": 2 * M * rows * K}
    if op == "rope":
        values = case["tokens"] * case["heads"] * case["D"]
        return {"bytes": 4 * values + 8 * case["tokens"] + 4 * case["R"], "flops": 3 * values}
    B, T, Hk, D = case["B"], case["T"], case["kv_heads"], case["D"]
    if op == "attend":
        Hq, cached = case["heads"], sum(_lengths(case))
        pages = sum(-(-n // case["page"]) for n in _lengths(case))
        masks = B * T * T if case["tree"] else 0
        return {"bytes": 4 * (cached + B * T) * Hk * D + 4 * B * T * Hq * D + 4 * pages + 4 * B + masks, "flops": 4 * T * Hq * D * (cached + B * T)}
    moved = sum(_counts(case))
    return {"bytes": 8 * moved * Hk * D + 8 * moved, "flops": 0}


def exact(case, seed):
    if case["op"] == "append":
        return None                                                       # copies
    s = prepare(case, seed)
    dtype = torch.float64
    if case["op"] in ("linear", "gated"):
        rows = s["w"].shape[-2]
        low, high = s["w"].to(torch.int64) % 16, s["w"].to(torch.int64) // 16
        codes = torch.empty(*s["w"].shape[:-1], 2 * s["w"].shape[-1], dtype=dtype, device="cuda")
        codes[..., 0::2], codes[..., 1::2] = low, high
        codes[codes > 7] -= 16
        if case["scales"] == "group":
            y = torch.zeros(case["M"], rows, dtype=dtype, device="cuda")
            for g in range(codes.shape[0]):
                y += s["x"][:, g * GROUP:(g + 1) * GROUP].to(dtype) @ codes[g].T * s["scale"][g].to(dtype)
        else:
            y = s["x"].to(dtype) @ codes.T * s["scale"].to(dtype)
        if case["op"] == "linear":
            return y
        gate, up = y[:, :case["N"]], y[:, case["N"]:]
        return gate * torch.sigmoid(gate) * up
    if case["op"] == "rope":
        R, x = case["R"], s["x"].to(dtype)
        first = torch.arange(0, R, 2, device="cuda") if case["interleaved"] else torch.arange(R // 2, device="cuda")
        second = first + (1 if case["interleaved"] else R // 2)
        z = torch.complex(x[..., first], x[..., second])
        angle = s["positions"].to(dtype)[:, None] * s["freqs"] * (-1 if case["inverse"] else 1)
        z = z * torch.polar(torch.full_like(angle, s["rescale"]), angle)[:, None]
        x[..., first], x[..., second] = z.real, z.imag
        return x
    out = torch.empty(s["q"].shape, dtype=dtype, device="cuda")
    T, group = case["T"], case["heads"] // case["kv_heads"]
    for b, length in enumerate(s["lengths"].tolist()):
        pages = s["table"][b].long()
        for h in range(case["kv_heads"]):
            k, v = (torch.cat((cache[pages, :, h].reshape(-1, case["D"])[:length], new[b, :, h])).to(dtype)
                    for cache, new in ((s["k_cache"], s["k"]), (s["v_cache"], s["v"])))
            hidden = torch.zeros(T, length + T, dtype=dtype, device="cuda")
            mask = s["mask"][b] if s["mask"] is not None else torch.ones(T, T, device="cuda").tril().bool()
            hidden[:, length:][~mask] = -math.inf
            for j in range(h * group, (h + 1) * group):
                score = s["q"][b, :, j].to(dtype) @ k.T / math.sqrt(case["D"]) + hidden
                out[b, :, j] = torch.softmax(score, -1) @ v
    return out
