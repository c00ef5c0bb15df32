"""GPU: attention of a few new tokens over a paged cache, and appending to it, against the softmax in 64 bits.

Tolerance (half = half a step of the type): the kernel's weights are w (1 + d) with |d| <= half + e, normalised by their own sum, so a
result moves by at most (half + e) / (1 - half - e) * sum p |v - out|; e is the exponent's error: a score of D products, summed in
fp32 by D / 16 tensor instructions and scaled (2^-23 of the absolute sum each), and 2^-22 of the exponential; sums of weighted values
over L keys in parts are off by 2^-23 of the absolute sum for each of L / 16 instructions and 600 joins at most; then one rounding."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def _pages(gen, B, page, width, Hk, D, dtype, heads_first=False, spare=3):
    count = B * width + spare
    shape = (count, Hk, page, D) if heads_first else (count, page, Hk, D)
    k, v = (torch.randn(shape, device="cuda", generator=gen).to(dtype) for _ in range(2))
    if heads_first:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    return k, v, torch.randperm(count, device="cuda", generator=gen)[: B * width].view(B, width).to(torch.int32)


def _tree(gen, B, T):
    mask = torch.zeros(B, T, T, dtype=torch.bool)
    for b in range(B):
        for i in range(T):
            parent = int(torch.randint(max(-1, i - 4), i, (1,), generator=gen)) if i else -1
            if parent >= 0:
                mask[b, i] = mask[b, parent]
            mask[b, i, i] = True
    return mask.cuda()


def _reference(q, k, v, k_cache, v_cache, table, lengths, mask=None, scale=None):
    """(result, its tolerance) [B, T, heads, D] in 64 bits; what a token does not see is left out, not weighted by zero."""
    B, T, H, D = q.shape
    Hk, half = k.shape[2], torch.finfo(q.dtype).eps / 2
    scale = D ** -0.5 if scale is None else scale
    out, tol = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    for b in range(B):
        n = int(lengths[b])
        at = torch.arange(n, device="cuda")
        pages, slots = table[b].long()[at // k_cache.shape[1]], at % k_cache.shape[1]
        for t in range(T):
            seen = (torch.arange(T, device="cuda") <= t) if mask is None else (mask[b, t] if mask.dim() == 3 else mask[t])
            kk, vv = (torch.cat((c[pages, slots], new[b][seen])).double() for c, new in ((k_cache, k), (v_cache, v)))   # [keys, Hk, D]
            if len(kk) == 0:
                continue
            kk, vv = (a.repeat_interleave(H // Hk, 1).transpose(0, 1) for a in (kk, vv))                                # [H, keys, D]
            qq = q[b, t].double()[:, None]
            p = torch.softmax((qq * kk).sum(-1) * scale, -1)
            o = (p[..., None] * vv).sum(1)
            e = ((qq * kk).abs().sum(-1) * abs(scale)).amax(-1) * (D / 16 + 4) * 2.0 ** -23 + 2.0 ** -22
            d = (half + e)[:, None]
            spread = (p[..., None] * (vv - o[:, None]).abs()).sum(1)
            sums = (p[..., None] * vv.abs()).sum(1) * (len(kk[0]) / 16 + 600) * 2.0 ** -23
            out[b, t] = o
            tol[b, t] = half * o.abs() + (1 + half) * (d / (1 - d) * spread + sums) + (2.0 ** -25 if q.dtype == torch.float16 else 0)
    return out, tol


def _check(out, ref, tol):
    fine = ref.isfinite()
    assert torch.equal(out.isnan(), ref.isnan()) and torch.equal(out[~fine & ~ref.isnan()].double(), ref[~fine & ~ref.isnan()])
    err = (out.double() - ref).abs()[fine]
    assert (err <= tol[fine]).all(), (err / tol[fine]).max()


def _new(gen, B, T, H, Hk, D, dtype):
    qkv = torch.randn(B, T, H + 2 * Hk, D, device="cuda", generator=gen).to(dtype)
    return qkv[:, :, :H], qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:]


CASES = [
    # B, T, heads, kv_heads, D, page, lengths, tree
    (1, 1, 1, 1, 64, 16, [0], False),
    (1, 1, 32, 8, 128, 16, [1001], False),
    (3, 1, 8, 8, 64, 1, [5, 0, 129], False),
    (2, 5, 4, 4, 128, 16, [63, 64], True),
    (4, 8, 8, 2, 128, 16, [0, 1, 300, 57], True),
    (2, 16, 32, 8, 128, 64, [700, 1300], True),
    (1, 64, 8, 2, 128, 24, [500], True),
    (2, 64, 7, 1, 64, 8, [65, 2], False),
    (2, 33, 14, 2, 80, 24, [100, 31], True),
    (3, 7, 8, 1, 96, 256, [1, 255, 257], True),
    (5, 3, 6, 3, 8, 3, [0, 1, 2, 3, 64], True),
    (40, 2, 4, 2, 64, 16, [3 * b for b in range(40)], False),
    (1, 16, 8, 2, 128, 64, [20000], True),
]


def _roomy(table, page):
    """The table with room for 64 thousand tokens, what is not used of it not a page: the work is shared out in another way."""
    wide = torch.full((table.shape[0], -(-65536 // page)), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    return wide


@pytest.mark.parametrize("room", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,H,Hk,D,page,lengths,tree", CASES)
def test_attention(B, T, H, Hk, D, page, lengths, tree, dtype, room):
    """With a table that just holds the sequences, and with one that has room for many more tokens."""
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(B * 1000 + T)
    width = max(1, -(-max(lengths) // page)) + 1
    kc, vc, table = _pages(gen, B, page, width, Hk, D, dtype)
    q, k, v = _new(gen, B, T, H, Hk, D, dtype)
    if room:
        table = _roomy(table, page)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    mask = _tree(torch.Generator().manual_seed(T), B, T) if tree else None
    out = ops.tree_attention(q, k, v, kc, vc, table, n, tree_mask=mask)
    assert out.shape == q.shape and out.dtype == dtype and out.is_contiguous()
    _check(out, *_reference(q, k, v, kc, vc, table, n, mask))
    assert torch.equal(out, ops.tree_attention(q, k, v, kc, vc, table, n, tree_mask=mask))      # the same bits in every run
    ops.check_status()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("room", [False, True])
@pytest.mark.parametrize("T,H", [(1, 4), (6, 4), (20, 4), (40, 8)])
def test_large_scores_and_scales(T, H, dtype, room):
    """Scores of hundreds: the running maximum moves by more than an exponential holds; also a negative scale and a scale of zero."""
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(T)
    kc, vc, table = _pages(gen, 2, 16, 20, 2, 64, dtype)
    q, k, v = _new(gen, 2, T, H, 2, 64, dtype)
    table = _roomy(table, 16) if room else table
    n = torch.tensor([313, 100], dtype=torch.int32, device="cuda")
    mask = _tree(torch.Generator().manual_seed(3), 2, T)
    for scale in (4.0, -0.5, 0.0):
        _check(ops.tree_attention(q, k, v, kc, vc, table, n, mask, scale), *_reference(q, k, v, kc, vc, table, n, mask, scale))


@pytest.mark.parametrize("room", [False, True])
@pytest.mark.parametrize("T,H", [(4, 2), (12, 2), (40, 2)])
def test_rows_that_see_nothing(T, H, room):
    """An empty row of the mask: zeros without a cache, the cache alone with one."""
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(T)
    kc, vc, table = _pages(gen, 3, 16, 5, 1, 128, torch.bfloat16)
    q, k, v = _new(gen, 3, T, H, 1, 128, torch.bfloat16)
    mask = _tree(torch.Generator().manual_seed(1), 3, T)
    mask[:, T // 2] = False
    mask[1] = False
    table = _roomy(table, 16) if room else table
    n = torch.tensor([0, 0, 70], dtype=torch.int32, device="cuda")
    out = ops.tree_attention(q, k, v, kc, vc, table, n, mask)
    assert not out[1].any() and not out[0, T // 2].any() and out[2, T // 2].any()
    _check(out, *_reference(q, k, v, kc, vc, table, n, mask))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("room", [False, True])
@pytest.mark.parametrize("T,H", [(5, 2), (13, 2), (60, 1), (30, 8)])
def test_what_is_not_seen_has_no_part(T, H, dtype, room):
    """NaN and infinities in unused slots, foreign pages and unseen nodes change nothing; in a seen node they reach the rows that see it,
    and those only."""
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(T)
    kc, vc, table = _pages(gen, 2, 16, 10, 1, 64, dtype)
    q, k, v = (t.contiguous() for t in _new(gen, 2, T, H, 1, 64, dtype))
    n = torch.tensor([77, 0], dtype=torch.int32, device="cuda")
    mask = _tree(torch.Generator().manual_seed(2), 2, T)
    mask[:, :, T - 1] = False                      # nobody sees the last node, itself included
    table = _roomy(table, 16) if room else table
    clean = ops.tree_attention(q, k, v, kc, vc, table, n, mask)
    used = torch.zeros(kc.shape[:2], dtype=torch.bool, device="cuda")
    at = torch.arange(77, device="cuda")
    used[table[0].long()[at // 16], at % 16] = True
    for cache in (kc, vc):
        cache[~used] = float("nan")
    k[:, T - 1], v[:, T - 1] = float("nan"), float("inf")
    assert torch.equal(ops.tree_attention(q, k, v, kc, vc, table, n, mask), clean)
    v[0, 1, 0, 3], v[1, 0, 0, 5], v[1, 0, 0, 6], k[0, 2, 0, 0] = float("nan"), float("inf"), -float("inf"), float("nan")
    out = ops.tree_attention(q, k, v, kc, vc, table, n, mask)
    _check(out, *_reference(q, k, v, kc, vc, table, n, mask))
    blind = ~mask[0, :, 1] & ~mask[0, :, 2]
    assert blind.any() and torch.equal(out[0, blind], clean[0, blind])
    assert out.isnan().any() and (out == float("inf")).any()


@pytest.mark.parametrize("layout", ["heads first", "wide rows", "odd strides", "misaligned", "shared mask"])
def test_layouts(layout):
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(4)
    dtype, B, T, H, Hk, D = torch.bfloat16, 2, 6, 8, 4, 64
    kc, vc, table = _pages(gen, B, 16, 9, Hk, D, dtype, heads_first=layout == "heads first")
    q, k, v = (t.contiguous() for t in _new(gen, B, T, H, Hk, D, dtype))
    n = torch.tensor([130, 47], dtype=torch.int32, device="cuda")
    mask = _tree(torch.Generator().manual_seed(4), B, T)
    want = ops.tree_attention(q, k, v, kc.contiguous(), vc.contiguous(), table, n, mask)
    if layout == "wide rows":
        wide = torch.full((B, 20), -1, dtype=torch.int32, device="cuda")
        wide[:, 4:13] = table
        table = wide[:, 4:13]
        q, k, v = (torch.zeros(T, B, t.shape[2] + 3, D, dtype=dtype, device="cuda")[:, :, 1:1 + t.shape[2]].transpose(0, 1).copy_(t) for t in (q, k, v))
    elif layout == "odd strides":
        q, k, v = (torch.zeros(B, T, t.shape[2], D + 1, dtype=dtype, device="cuda")[..., :D].copy_(t) for t in (q, k, v))
    elif layout == "misaligned":
        q, k, v = (torch.zeros(t.numel() + 1, dtype=dtype, device="cuda")[1:].view(t.shape).copy_(t) for t in (q, k, v))
    elif layout == "shared mask":
        mask = mask[0]
        want = ops.tree_attention(q, k, v, kc, vc, table, n, mask.expand(B, T, T))
    assert torch.equal(ops.tree_attention(q, k, v, kc, vc, table, n, mask), want)


def test_offsets_past_32_bits():
    """A cache of more than 2^31 elements, its last pages in use."""
    from fp8_inference_toolkit_b200 import ops

    pages, page, Hk, D = 2100, 1024, 8, 128                       # 2.2e9 elements each
    k_cache, v_cache = (torch.zeros(pages, page, Hk, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    gen = torch.Generator(device="cuda").manual_seed(9)
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device="cuda")
    n = torch.tensor([2500], dtype=torch.int32, device="cuda")
    rows = torch.randn(2, 1, 2500, Hk, D, device="cuda", generator=gen).to(torch.bfloat16)
    ops.kv_cache_append_(k_cache, v_cache, rows[0], rows[1], table, torch.zeros_like(n))
    at = torch.arange(2500, device="cuda")
    where = table[0].long()[at // page], at % page
    assert torch.equal(k_cache[where], rows[0, 0]) and torch.equal(v_cache[where], rows[1, 0])
    q, k, v = _new(gen, 1, 4, 8, Hk, D, torch.bfloat16)
    _check(ops.tree_attention(q, k, v, k_cache, v_cache, table, n), *_reference(q, k, v, k_cache, v_cache, table, n))
    ops.check_status()


@pytest.mark.parametrize("room", [False, True])
@pytest.mark.parametrize("bad", ["page", "negative page", "length", "negative length"])
def test_out_of_range_is_reported(bad, room):
    """Nothing outside the cache is read, the call before and after stay right, and check_status raises once."""
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(10)
    kc, vc, table = _pages(gen, 2, 16, 6, 2, 64, torch.bfloat16)
    q, k, v = _new(gen, 2, 3, 4, 2, 64, torch.bfloat16)
    table = _roomy(table, 16) if room else table
    n = torch.tensor([90, 40], dtype=torch.int32, device="cuda")
    want = ops.tree_attention(q, k, v, kc, vc, table, n)
    ops.check_status()
    t2, n2 = table.clone(), n.clone()
    if "page" in bad:
        t2[0, 2] = kc.shape[0] if bad == "page" else -1
    else:
        n2[0] = table.shape[1] * 16 + 1 if bad == "length" else -5
    out = ops.tree_attention(q, k, v, kc, vc, t2, n2)
    assert torch.equal(out[1], want[1])
    with pytest.raises(RuntimeError, match="out of range"):
        ops.check_status()
    ops.check_status()
    k0, v0 = kc.clone(), vc.clone()
    n3 = torch.tensor([40 if "page" in bad else n2[0].item(), 10], dtype=torch.int32, device="cuda")
    ops.kv_cache_append_(kc, vc, k, v, t2, n3)
    with pytest.raises(RuntimeError, match="out of range"):
        ops.check_status()
    changed = torch.zeros(kc.shape[:2], dtype=torch.bool, device="cuda")
    changed[table[1, 0].long(), 10:13] = True
    assert torch.equal(kc[~changed], k0[~changed]) and torch.equal(vc[~changed], v0[~changed]) and torch.equal(kc[changed], k[1])


@pytest.mark.parametrize("B,T,Hk,D,page,lengths,picked", [
    (1, 1, 1, 8, 1, [0], False), (3, 5, 2, 64, 16, [0, 14, 31], True), (2, 300, 8, 128, 64, [0, 7], False), (4, 7, 3, 33, 4, [3, 0, 9, 1], True),
    (2, 9, 1, 2, 24, [20, 23], True), (64, 4, 8, 128, 16, [b for b in range(64)], True),
])
def test_append(B, T, Hk, D, page, lengths, picked):
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(T)
    width = -(-(max(lengths) + T) // page)
    kc, vc, table = _pages(gen, B, page, width, Hk, D, torch.float16)
    _, k, v = _new(gen, B, T, Hk, Hk, D, torch.float16)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    counts = select = None
    if picked:
        counts = torch.tensor([b % (T + 1) for b in range(B)], dtype=torch.int32, device="cuda")
        select = torch.stack([torch.randperm(T, device="cuda", generator=gen).sort().values for _ in range(B)]).to(torch.int32)
        select = torch.cat((select, torch.full((B, 2), -9, dtype=torch.int32, device="cuda")), 1)     # columns past T are nobody's
        select[0] = 10 ** 6                                                                           # counts[0] = 0: not read
    want_k, want_v = kc.clone(), vc.clone()
    for b in range(B):
        for i in range(T if counts is None else int(counts[b])):
            at = lengths[b] + i
            where = int(table[b, at // page]), at % page
            src = i if select is None else int(select[b, i])
            want_k[where], want_v[where] = k[b, src], v[b, src]
    ops.kv_cache_append_(kc, vc, k, v, table, n, select=select, counts=counts)
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v) and n.tolist() == lengths
    ops.check_status()


def test_append_then_attend_equals_attention_with_all_tokens_at_once():
    """Tokens one by one, each appended after its attention, against the same tokens as one chain."""
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(12)
    kc, vc, table = _pages(gen, 2, 16, 8, 2, 128, torch.bfloat16)
    q, k, v = _new(gen, 2, 12, 8, 2, 128, torch.bfloat16)
    n = torch.tensor([60, 15], dtype=torch.int32, device="cuda")
    ref, tol = _reference(q, k, v, kc, vc, table, n)
    _check(ops.tree_attention(q, k, v, kc, vc, table, n), ref, tol)
    for t in range(12):
        new = [a[:, t:t + 1] for a in (q, k, v)]
        _check(ops.tree_attention(*new, kc, vc, table, n), ref[:, t:t + 1], tol[:, t:t + 1])
        ops.kv_cache_append_(kc, vc, new[1], new[2], table, n)
        n += 1


def test_graphs_and_streams():
    """Replays read lengths and tables as they are then; two captured graphs and an eager call do not disturb one another."""
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(13)
    sets, wants = [], []
    for _ in range(3):
        kc, vc, table = _pages(gen, 4, 16, 40, 2, 128, torch.bfloat16)
        q, k, v = _new(gen, 4, 8, 8, 2, 128, torch.bfloat16)
        n = torch.tensor([600, 3, 250, 77], dtype=torch.int32, device="cuda")
        sets.append((q, k, v, kc, vc, table, n))
        wants.append([ops.tree_attention(q, k, v, kc, vc, table, m) for m in (n, n.flip(0).contiguous())])
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for s, st in zip(sets, streams):
        st.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            outs.append(ops.tree_attention(*s))
        graphs.append(graph)
    for turn in range(2):
        torch.cuda.synchronize()
        for _ in range(10):
            for graph, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    graph.replay()
            eager = ops.tree_attention(*sets[2])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], wants[0][turn]) and torch.equal(outs[1], wants[1][turn]) and torch.equal(eager, wants[2][turn])
        for s in sets:
            s[6].copy_(s[6].flip(0).clone())


def _shifted(cache):
    """A cache of the same shape that begins 8 bytes off."""
    return torch.empty(cache.numel() + 4, dtype=cache.dtype, device="cuda")[4:].view(cache.shape)


def test_refusals():
    from fp8_inference_toolkit_b200 import ops

    gen = torch.Generator(device="cuda").manual_seed(14)
    kc, vc, table = _pages(gen, 2, 16, 4, 2, 64, torch.bfloat16)
    q, k, v = _new(gen, 2, 3, 4, 2, 64, torch.bfloat16)
    n = torch.tensor([5, 6], dtype=torch.int32, device="cuda")
    good = dict(q=q, k=k, v=v, k_cache=kc, v_cache=vc, block_table=table, lengths=n)
    assert ops.tree_attention(**{**good, "q": q[:, :0], "k": k[:, :0], "v": v[:, :0]}).shape == (2, 0, 4, 64)
    for change, match in [
        (dict(q=q.cpu()), "CUDA"), (dict(q=q.float()), "bfloat16"), (dict(q=q.half()), "dtype"), (dict(q=q[:, :, :3]), "multiple of kv_heads"),
        (dict(q=q[:, :2]), r"\[B, T"), (dict(q=q[0]), "4D"), (dict(v=v[:, :2]), "same shape"), (dict(k_cache=kc[..., :32]), "same shape and strides"),
        (dict(v_cache=vc.transpose(1, 2).contiguous().transpose(1, 2)), "strides"), (dict(k_cache=kc[:, :, :1], v_cache=vc[:, :, :1]), "kv_heads"),
        (dict(block_table=table.long()), "int32"), (dict(block_table=table[:1]), "int32"), (dict(lengths=n.long()), "int32"), (dict(lengths=n[:1]), "int32"),
        (dict(lengths=n.cpu()), "device"), (dict(tree_mask=torch.ones(2, 3, 3, device="cuda")), "bool"),
        (dict(tree_mask=torch.ones(2, 3, 4, device="cuda", dtype=torch.bool)), "tree_mask"), (dict(q=q.clone().requires_grad_()), "backward"),
        (dict(k_cache=_shifted(kc), v_cache=_shifted(vc)), "16-byte"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            ops.tree_attention(**{**good, **change})
    q65, k65, v65 = _new(gen, 2, 65, 4, 2, 64, torch.bfloat16)
    with pytest.raises(RuntimeError, match="64 new tokens"):
        ops.tree_attention(**{**good, "q": q65, "k": k65, "v": v65})
    wide = [t.repeat(1, 1, 1, 4) for t in (q, k, v, kc, vc)]
    with pytest.raises(RuntimeError, match="128 elements"):
        ops.tree_attention(*wide, table, n)
    base = (kc, vc, k, v, table, n)
    for extra, match in [(dict(counts=n.long()), "counts"), (dict(counts=n[:1]), "counts"), (dict(select=torch.zeros(2, 2, dtype=torch.int32, device="cuda")), "columns"),
                         (dict(select=torch.zeros(2, 3, device="cuda", dtype=torch.int64)), "select")]:
        with pytest.raises(RuntimeError, match=match):
            ops.kv_cache_append_(*base, **extra)
