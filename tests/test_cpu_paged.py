"""The paged cache's entry points without a GPU: sizes, and every refusal that the host makes before it enqueues anything
(addresses are made up; nothing is read)."""
import ctypes as C
import re

import pytest

from voxgen_b200 import api

OK, EINVAL, EUNSUPPORTED, ERANGE = 0, -1, -4, -5
A = 0x1000   # stands for a device address
TABLE = dict(table=A, rows=A, status=A, free=A, pool=A, seqs=4, seq_pages=32, pages=64, page_rows=64)
CACHE = dict(data=A, summaries=A, dtype=1, kv_heads=2, head_dim=128)
STEP = dict(starts=A, slots=A, positions=A, sequences=A, runs=A, tokens=8)


def table(**over):
    d = {**TABLE, **over}
    return api.PagedTableDesc(*[d[n] for n, _ in api.PagedTableDesc._fields_])


def cache(of=None, **over):
    d = {**CACHE, **over}
    return C.byref(api.PagedCacheDesc(C.pointer(of or table()), *[d[n] for n, _ in api.PagedCacheDesc._fields_[1:]]))


def step_of(**over):
    d = {**STEP, **over}
    return C.byref(api.PagedStepDesc(*[d[n] for n, _ in api.PagedStepDesc._fields_]))


def step(t=None, counts=A, keep=A, step=None):
    return api.lib().vg_k_paged_step(C.byref(t or table()), counts, keep, step or step_of(), None)


def append(c=None, s=None, k=A, v=A, dtype=0):
    return api.lib().vg_k_paged_append(c or cache(), s or step_of(), k, v, dtype, None, None, None)


def select(c=None, q=A, dtype=0, queries=4, heads=16, sequences=None, positions=None, budget=8, sinks=1, recent=2, chosen=A):
    return api.lib().vg_k_paged_select(c or cache(), q, dtype, queries, heads, None, sequences, positions, budget, sinks, recent,
                                       chosen, None)


def attention(c=None, q=A, dtype=0, queries=4, heads=16, sequences=None, positions=None, chosen=None, budget=0, scale=0.1,
              out=2 * A, ws=A, ws_bytes=1 << 40):
    return api.lib().vg_k_paged_attention(c or cache(), q, dtype, queries, heads, None, sequences, positions, chosen, budget,
                                          scale, out, ws, ws_bytes, None)


def attention_bytes(c=None, queries=4, heads=16, budget=0):
    n = C.c_uint64()
    return api.lib().vg_k_paged_attention_bytes(c or cache(), queries, heads, budget, C.byref(n)), n.value


@pytest.mark.parametrize("shape,want", [((1, 16, 1, 64), (4096, 256)), ((5, 64, 2, 128), (327680, 5120)),
                                        ((1 << 20, 256, 8, 128), ((1 << 20) * 8 * 2 * 256 * 256, (1 << 20) * 8 * 512))])
def test_bytes(shape, want):
    a, b = C.c_uint64(), C.c_uint64()
    assert api.lib().vg_k_paged_bytes(*shape, C.byref(a), C.byref(b)) == OK and (a.value, b.value) == want


@pytest.mark.parametrize("shape,want", [
    ((0, 16, 1, 64), EINVAL), ((1, 16, 0, 64), EINVAL), ((1, 8, 1, 64), EUNSUPPORTED), ((1, 24, 1, 64), EUNSUPPORTED),
    ((1, 512, 1, 64), EUNSUPPORTED), ((1, 16, 1, 96), EUNSUPPORTED), ((1 << 28, 16, 1, 64), ERANGE), ((1 << 26, 16, 64, 64), ERANGE)])
def test_bytes_refuses(shape, want):
    a, b = C.c_uint64(), C.c_uint64()
    assert api.lib().vg_k_paged_bytes(*shape, C.byref(a), C.byref(b)) == want


@pytest.mark.parametrize("tokens,page,seqs,want", [(0, 16, 4, 0), (1, 16, 4, 1), (100, 16, 4, 14), (9, 16, 4, 8), (7, 256, 4, 7)])
def test_runs(tokens, page, seqs, want):
    n = C.c_uint32()
    assert api.lib().vg_k_paged_runs(C.byref(table(page_rows=page, seqs=seqs)), tokens, C.byref(n)) == OK and n.value == want
    assert api.lib().vg_k_paged_runs(C.byref(table()), (1 << 30) + 1, C.byref(n)) == ERANGE
    assert api.lib().vg_k_paged_runs(C.byref(table()), 1, None) == EINVAL


TABLE_FAULTS = [({n: None}, EINVAL) for n in ("table", "rows", "status", "free", "pool")] + \
    [({n: A + 2}, EINVAL) for n in ("table", "rows", "status", "free", "pool")] + \
    [({n: 0}, EINVAL) for n in ("seqs", "seq_pages", "pages")] + \
    [({"page_rows": n}, EUNSUPPORTED) for n in (0, 8, 48, 512)] + \
    [({"seqs": 4097}, ERANGE), ({"pages": 1 << 25}, ERANGE), ({"seq_pages": (1 << 24) + 1}, ERANGE)]


@pytest.mark.parametrize("over,want", TABLE_FAULTS)
def test_a_bad_table_is_refused(over, want):
    assert step(table(**over)) == want
    for call in (append, select, attention):
        assert call(cache(table(**over))) == want


def test_no_table():
    assert api.lib().vg_k_paged_step(None, A, A, step_of(), None) == EINVAL
    none = C.byref(api.PagedCacheDesc(None, A, A, 1, 2, 128))
    for call in (append, select, attention):
        assert call(none) == EINVAL
    assert api.lib().vg_k_paged_append(None, step_of(), A, A, 0, None, None, None) == EINVAL


@pytest.mark.parametrize("over,want", [
    ({"data": None}, EINVAL), ({"data": A + 8}, EINVAL), ({"summaries": A + 16}, EINVAL), ({"kv_heads": 0}, EINVAL),
    ({"dtype": 0}, EUNSUPPORTED), ({"dtype": 8}, EUNSUPPORTED), ({"head_dim": 32}, EUNSUPPORTED), ({"head_dim": 256}, EUNSUPPORTED),
    ({"kv_heads": 1 << 26}, ERANGE)])
def test_a_bad_cache_is_refused(over, want):
    for call in (append, select, attention):
        assert call(cache(**over)) == want
    assert attention_bytes(cache(**over))[0] == want


@pytest.mark.parametrize("over", [{n: None} for n in ("starts", "slots", "positions", "sequences", "runs")] +
                         [{n: A + 4} for n in ("starts", "slots", "positions", "sequences", "runs")])
def test_a_bad_step_is_refused(over):
    assert step(step=step_of(**over)) == EINVAL
    assert append(s=step_of(**over)) == EINVAL


def test_step_refuses():
    assert step(counts=None) == EINVAL and step(counts=A + 2) == EINVAL and step(keep=A + 1) == EINVAL
    assert step(step=step_of(tokens=(1 << 30) + 1)) == ERANGE


@pytest.mark.parametrize("over,want", [({"k": None}, EINVAL), ({"v": None}, EINVAL), ({"k": A + 2}, EINVAL), ({"dtype": 8}, EUNSUPPORTED)])
def test_append_refuses(over, want):
    assert append(**over) == want


def test_an_append_of_no_tokens_needs_no_rows():
    assert append(s=step_of(tokens=0), k=None, v=None) == OK


QUERY_FAULTS = [({"q": None}, EINVAL), ({"q": A + 2}, EINVAL), ({"dtype": 2}, EUNSUPPORTED), ({"queries": 0}, EINVAL),
                ({"queries": 5}, EINVAL), ({"heads": 0}, EINVAL), ({"heads": 15}, EINVAL), ({"sequences": A + 2}, EINVAL),
                ({"positions": A + 1}, EINVAL)]


@pytest.mark.parametrize("over,want", QUERY_FAULTS + [
    ({"chosen": None}, EINVAL), ({"chosen": A + 2}, EINVAL), ({"budget": 0}, EINVAL), ({"sinks": 6, "recent": 3}, ERANGE),
    ({"sinks": 0xFFFFFFFF, "recent": 2}, ERANGE), ({"c": cache(summaries=None)}, EINVAL),
    ({"c": cache(table(seq_pages=24577))}, ERANGE), ({"budget": 1 << 31, "sinks": 0}, ERANGE)])
def test_select_refuses(over, want):
    assert select(**over) == want


@pytest.mark.parametrize("over,want", QUERY_FAULTS + [
    ({"out": None}, EINVAL), ({"out": 2 * A + 8}, EINVAL), ({"out": A}, EINVAL), ({"ws": None}, EINVAL), ({"ws": A + 8}, EINVAL),
    ({"ws_bytes": 16}, EINVAL), ({"scale": 0.0}, EINVAL), ({"scale": -1.0}, EINVAL), ({"scale": float("nan")}, EINVAL),
    ({"scale": float("inf")}, EINVAL), ({"chosen": A}, EINVAL), ({"budget": 8}, EINVAL), ({"chosen": A + 2, "budget": 8}, EINVAL),
    ({"queries": 1 << 31, "sequences": A}, ERANGE)])
def test_attention_refuses(over, want):
    assert attention(**over) == want


def test_attention_bytes():
    rc, few = attention_bytes()
    assert rc == OK and few == 4 * (1 << 14) + 2 * 148 * 4 * 8 * 130 * 4
    # many segments: as many partial results, however many they are; none where no segment is cut
    big = table(seqs=4096)
    assert attention_bytes(cache(big), queries=500)[1] == attention_bytes(cache(big), queries=4000)[1] > few
    assert attention_bytes(cache(big), queries=100000)[1] == 4 * (1 << 14)
    assert attention_bytes(queries=0)[0] == EINVAL and attention_bytes(heads=15)[0] == EINVAL
    assert attention_bytes(cache(table(seqs=4096, seq_pages=1 << 24)), queries=4096)[0] == ERANGE
    assert attention_bytes(budget=1 << 29)[0] == ERANGE


def test_ring_stages_are_whole_rounds_of_the_warps():
    """A stage of the attention's ring is always the same team's: the property that its waits need."""
    from voxgen_b200._build import CSRC
    text = (CSRC / "paged_attention.cuh").read_text()
    assert "kPagedWarps = 12, kPagedFew = 4;" in text and "kStages % W == 0" in text
    for warps, rounds in ((12, 2), (4, 1)):
        for dim in (64, 128):
            stages, team_of = rounds * warps * 128 // dim, {}
            for tiles in (1, 2, 4):
                teams = warps // tiles
                for block in range(10 * stages):
                    assert team_of.setdefault((tiles, block % stages), block % teams) == block % teams


def test_dynamic_shared_memory_is_declared_with_the_alignment_of_its_widest_access():
    from voxgen_b200._build import CSRC
    found = {}
    for path in CSRC.glob("paged*.cuh"):
        for align, name in re.findall(r"extern __shared__ (?:__align__\((\d+)\) )?\w+ (\w+)\[\]", path.read_text()):
            found[name] = int(align or 0)
    assert len(found) == 3 and all(a >= 16 for a in found.values()), found
