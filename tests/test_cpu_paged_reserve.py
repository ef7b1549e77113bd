"""The sizes that ``PagedCache.reserve`` asks for cover every smaller call."""
import ctypes as C

import pytest

from voxgen_b200 import api

A = 0x1000


def need(queries, heads, kv_heads, budget):
    table = api.PagedTableDesc(A, A, A, A, A, 4096, 64, 4096, 16)
    cache = api.PagedCacheDesc(C.pointer(table), A, A, 1, kv_heads, 64)
    n = C.c_uint64()
    assert api.lib().vg_k_paged_attention_bytes(C.byref(cache), queries, heads, budget, C.byref(n)) == 0
    return n.value


def reserved(queries, *shape):
    """What reserve makes room for: the sizes that voxgen_b200/paged.py asks for."""
    from pathlib import Path
    text = (Path(api.__file__).parent / "paged.py").read_text()
    assert "while queries:" in text and "queries //= 2" in text
    most = 0
    while queries:
        most = max(most, need(queries, *shape))
        queries //= 2
    return most


@pytest.mark.parametrize("heads,kv_heads,budget", [(8, 1, 0), (16, 2, 0), (16, 2, 7), (24, 1, 0), (72, 1, 0), (512, 1, 5), (24, 3, 1), (64, 64, 0)])
def test_a_reserved_workspace_serves_every_smaller_batch(heads, kv_heads, budget):
    shape = heads, kv_heads, budget
    marks = {1, 2, 3, 100, 148, 222, 443, 444, 445, 888, 889, 1183, 2000, 16383, 16384, 16385, 20000, 40000}
    sizes = {}
    for n in sorted(marks | {max(1, m // k) for m in marks for k in (2, 3, 64, 128)}):
        sizes[n] = need(n, *shape)
        room = reserved(n, *shape)
        assert all(x <= room for m, x in sizes.items()), n
        if budget:      # and of shorter lists
            assert need(n, heads, kv_heads, 1) <= room
