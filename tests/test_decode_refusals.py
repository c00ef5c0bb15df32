"""CPU: the C entry points of the decoding operators refuse what they cannot serve before any CUDA call."""
import struct

import pytest


def _cabi(lib_built):
    from fp8_inference_toolkit_b200 import _cabi

    return _cabi


def test_linear(lib_built):
    c = _cabi(lib_built)
    call = lambda *a: c.lib.i4tc_w4a16_linear(*a, 0, None)  # noqa: E731
    x = w = s = o = 4096                                    # addresses that nothing reads
    for args, match in [((x, c.FP32, 1, 128, 128, w, s, 0, 0, o, 8), "bfloat16"), ((x, c.BF16, -1, 128, 128, w, s, 0, 0, o, 8), "size"),
                        ((x, c.BF16, 1, 0, 0, w, s, 0, 0, o, 8), "size"), ((x, c.BF16, 1, 192, 192, w, s, 0, 0, o, 8), "divisible"),
                        ((x, c.BF16, 1, 96, 96, w, s, 1, 0, o, 8), "multiple of 64"), ((x, c.BF16, 1, 1 << 21, 1 << 21, w, s, 0, 0, o, 8), "too large"),
                        ((x + 2, c.BF16, 1, 128, 128, w, s, 0, 0, o, 8), "aligned"), ((x, c.BF16, 1, 128, 130, w, s, 0, 0, o, 8), "aligned"),
                        ((None, c.BF16, 1, 128, 128, w, s, 0, 0, o, 8), "null")]:
        assert call(*args) < 0 and match in c.last_error()
    assert call(None, c.BF16, 0, 128, 128, None, None, 0, 0, None, 8) == 0


def test_rope(lib_built):
    c = _cabi(lib_built)
    call = lambda *a: c.lib.i4tc_rope(*a, 0, None)  # noqa: E731
    x, at, f, o = 4096, 8192, 16384, 1 << 20
    for args, match in [((x, c.FP32, 1, 1, 8, 8, 8, 8, at, 0, f, 0, 1.0, 0, o, 8, 8), "bfloat16"), ((x, c.BF16, 1, 1, 8, 7, 8, 8, at, 0, f, 0, 1.0, 0, o, 8, 8), "even"),
                        ((x, c.BF16, 1, 1, 8, 10, 8, 8, at, 0, f, 0, 1.0, 0, o, 8, 8), "even"), ((x, c.BF16, 1, 1, 8, 8, 8, 8, None, 0, f, 0, 1.0, 0, o, 8, 8), "null"),
                        ((x, c.BF16, 1, 1, 8, 8, 8, 8, at, 0, f, 0, 1.0, 0, x, 16, 8), "strides"), ((x + 1, c.BF16, 1, 1, 8, 8, 8, 8, at, 0, f, 0, 1.0, 0, o, 8, 8), "aligned"),
                        ((x, c.BF16, 1, 1, 4096, 8, 8, 8, at, 0, f, 0, 1.0, 0, o, 8, 8), "size")]:
        assert call(*args) < 0 and match in c.last_error()
    assert call(None, c.BF16, 0, 1, 8, 8, 8, 8, None, 0, None, 0, 1.0, 0, None, 8, 8) == 0


ATTENTION = ("q k v k_cache v_cache table lengths mask out scratch bytes dtype batch tokens heads kv_heads D pages page width "
             "qb qt qh nb nt nh ps ss hs ts mb").split()
GOOD = dict(q=4096, k=4096, v=4096, k_cache=4096, v_cache=4096, table=4096, lengths=4096, mask=0, out=4096, scratch=4096, bytes=0, dtype=0, batch=1, tokens=1,
            heads=2, kv_heads=1, D=64, pages=4, page=16, width=4, qb=128, qt=128, qh=64, nb=64, nt=64, nh=64, ps=1024, ss=64, hs=64, ts=4, mb=0)


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
