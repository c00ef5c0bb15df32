"""CPU: the C entry points of the decoding operators refuse what they cannot serve before any CUDA call."""
import struct

import pytest


def _cabi(lib_built):
    from fp8_inference_toolkit_b200 import _cabi

    return _cabi


LINEAR = dict(x=4096, w=4096, scale=4096, out=4096, dtype=0, M=1, K=128, ldx=128, N=8, per_channel=0, gated=0)   # addresses that nothing reads


@pytest.mark.parametrize("change,match", [
    (dict(dtype=2), "bfloat16"), (dict(M=-1), "size"), (dict(K=0), "size"), (dict(K=192, ldx=192), "divisible"), (dict(K=96, ldx=96, per_channel=1), "multiple of 64"),
    (dict(K=1 << 21, ldx=1 << 21), "too large"), (dict(x=4098), "aligned"), (dict(ldx=130), "aligned"), (dict(x=0), "null"),
])
def test_linear(lib_built, change, match):
    c = _cabi(lib_built)
    assert c.lib.i4tc_w4a16_linear(struct.pack("@4P7q", *{**LINEAR, **change}.values()), 0, None) < 0 and match in c.last_error()
    assert c.lib.i4tc_w4a16_linear(None, 0, None) < 0
    assert c.lib.i4tc_w4a16_linear(struct.pack("@4P7q", *{**LINEAR, "M": 0}.values()), 0, None) == 0


ROPE = dict(x=4096, positions=8192, freqs=16384, out=1 << 20, dtype=0, tokens=1, heads=1, D=8, R=8, xt=8, xh=8, ot=8, oh=8, long=0, inter=0, inverse=0)


@pytest.mark.parametrize("change,match", [
    (dict(dtype=2), "bfloat16"), (dict(R=7), "even"), (dict(R=10), "even"), (dict(positions=0), "null"), (dict(out=4096, ot=16), "strides"),
    (dict(x=4097), "aligned"), (dict(long=1, positions=8196), "aligned"), (dict(D=4096), "size"),
])
def test_rope(lib_built, change, match):
    c = _cabi(lib_built)
    assert c.lib.i4tc_rope(struct.pack("@4P12qd", *{**ROPE, **change}.values(), 1.0), 0, None) < 0 and match in c.last_error()
    assert c.lib.i4tc_rope(None, 0, None) < 0
    assert c.lib.i4tc_rope(struct.pack("@4P12qd", *{**ROPE, "tokens": 0}.values(), 1.0), 0, None) == 0


ATTENTION = ("q k v k_cache v_cache table lengths mask out scratch bytes dtype batch tokens heads kv_heads D pages page width "
             "qb qt qh nb nt nh ps ss hs ts mb").split()
GOOD = dict(q=4096, k=4096, v=4096, k_cache=4096, v_cache=4096, table=4096, lengths=4096, mask=0, out=4096, scratch=4096, bytes=0, dtype=0, batch=1, tokens=1,
            heads=2, kv_heads=1, D=64, pages=4, page=16, width=4, qb=128, qt=128, qh=64, nb=64, nt=64, nh=64, ps=1024, ss=64, hs=64, ts=4, mb=0)


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf")])
def test_attention_scale(lib_built, scale):
    c = _cabi(lib_built)
    assert c.lib.i4tc_tree_attention(struct.pack("@10P21qd", *GOOD.values(), scale), 0, None) < 0 and "finite" in c.last_error()


@pytest.mark.parametrize("change,match", [
    (dict(dtype=2), "bfloat16"), (dict(batch=-1), "size"), (dict(tokens=65), "64 new"), (dict(D=136), "128 elements"), (dict(D=12), "multiple of 8"),
    (dict(kv_heads=0), "multiple of kv_heads"), (dict(heads=3, kv_heads=2), "multiple of kv_heads"), (dict(page=0), "size"), (dict(q=0), "null"),
    (dict(table=0), "null"), (dict(k=4104), "aligned"), (dict(ss=60), "aligned"), (dict(qt=127), "aligned"),
])
def test_attention(lib_built, change, match):
    c = _cabi(lib_built)
    assert list(GOOD) == ATTENTION
    args = struct.pack("@10P21qd", *{**GOOD, **change}.values(), 0.125)
    assert c.lib.i4tc_tree_attention(args, 0, None) < 0 and match in c.last_error()
    assert c.lib.i4tc_tree_attention(None, 0, None) < 0
    assert c.lib.i4tc_tree_attention(struct.pack("@10P21qd", *{**GOOD, "tokens": 0}.values(), 0.125), 0, None) == 0


APPEND = dict(k=4096, v=4096, k_cache=4096, v_cache=4096, table=4096, lengths=4096, counts=0, select=0, element=2, batch=1, tokens=1, kv_heads=1, D=64, pages=4, page=16,
              width=4, nb=64, nt=64, nh=64, ps=1024, ss=64, hs=64, ts=4, sel=0)


@pytest.mark.parametrize("change,match", [(dict(element=4), "bfloat16"), (dict(tokens=-1), "size"), (dict(page=0), "size"), (dict(k=0), "null"), (dict(v_cache=0), "null"),
                                          (dict(D=4096), "size")])
def test_append(lib_built, change, match):
    c = _cabi(lib_built)
    assert c.lib.i4tc_kv_append(struct.pack("@8P16q", *{**APPEND, **change}.values()), 0, None) < 0 and match in c.last_error()
    assert c.lib.i4tc_kv_append(None, 0, None) < 0
    assert c.lib.i4tc_kv_append(struct.pack("@8P16q", *{**APPEND, "batch": 0}.values()), 0, None) == 0


def test_ops_refuse_cpu_tensors(lib_built):
    import torch

    from fp8_inference_toolkit_b200 import ops

    x = torch.zeros(2, 4, 16, 64, dtype=torch.bfloat16)
    index = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.w4a16_linear(x[0, 0], index, index, 1), lambda: ops.w4a16_gated_linear(x[0, 0], index, index, 1),
                 lambda: ops.rope(x[0], index, index), lambda: ops.rope_(x[0], index, index), lambda: ops.tree_attention(x, x, x, x, x, index, index),
                 lambda: ops.kv_cache_append_(x, x, x, x, index, index)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
