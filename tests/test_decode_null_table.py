"""CPU: a block table is read wherever a token's place is looked up, so it has to be there even for a cache without pages."""
import struct

import pytest

ATTENTION = dict(q=4096, k=4096, v=4096, k_cache=4096, v_cache=4096, table=4096, lengths=4096, mask=0, out=4096, scratch=4096, bytes=0, dtype=0, batch=1, tokens=1,
                 heads=2, kv_heads=1, D=64, pages=4, page=16, width=4, qb=128, qt=128, qh=64, nb=64, nt=64, nh=64, ps=1024, ss=64, hs=64, ts=4, mb=0)
APPEND = dict(k=4096, v=4096, k_cache=4096, v_cache=4096, table=4096, lengths=4096, counts=0, select=0, element=2, batch=1, tokens=1, kv_heads=1, D=64, pages=4, page=16,
              width=4, nb=64, nt=64, nh=64, ps=1024, ss=64, hs=64, ts=4, sel=0)


@pytest.mark.parametrize("change", [dict(table=0), dict(table=0, pages=0), dict(table=0, pages=0, k_cache=0, v_cache=0), dict(k_cache=0), dict(v_cache=0)])
def test_null_pointers(lib_built, change):
    from fp8_inference_toolkit_b200 import _cabi as c

    for entry, args in ((c.lib.i4tc_tree_attention, struct.pack("@10P21qd", *{**ATTENTION, **change}.values(), 0.125)),
                        (c.lib.i4tc_kv_append, struct.pack("@8P16q", *{**APPEND, **change}.values()))):
        assert entry(args, 0, None) < 0 and "null" in c.last_error()
