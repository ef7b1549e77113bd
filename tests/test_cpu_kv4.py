"""The 4-bit cache's entry points without a GPU: sizes, and every refusal that the host makes before
it enqueues anything (addresses are made up; nothing is read)."""
import ctypes as C
import re

import pytest

from voxgen_b200 import api

EINVAL, EUNSUPPORTED, ERANGE, EFULL = -1, -4, -5, -6
A = 0x1000   # stands for a device address


def desc(**over):
    d = dict(data=A, state=A, weights=A, positions=A, seqs=2, kv_heads=2, head_dim=128, capacity=256)
    d.update(over)
    return api.Kv4CacheDesc(*[d[n] for n, _ in api.Kv4CacheDesc._fields_])


@pytest.mark.parametrize("seqs,kv_heads,dim,capacity,want", [
    (1, 1, 128, 1, 9216), (1, 1, 128, 64, 9216), (1, 1, 128, 65, 2 * 9216), (3, 2, 64, 100, 6 * 2 * 4608),
    (28, 2, 128, 32768, 56 * 512 * 9216),
])
def test_bytes(seqs, kv_heads, dim, capacity, want):
    n = C.c_uint64()
    assert api.lib().vg_k_kv4_bytes(seqs, kv_heads, dim, capacity, C.byref(n)) == 0
    assert n.value == want


@pytest.mark.parametrize("shape,want", [
    ((0, 1, 128, 64), EINVAL), ((1, 0, 128, 64), EINVAL), ((1, 1, 128, 0), EINVAL), ((1, 1, 96, 64), EUNSUPPORTED),
    ((1, 1, 256, 64), EUNSUPPORTED), ((1, 1, 128, 1 << 31), ERANGE), ((1 << 20, 1 << 20, 128, 64), ERANGE),
])
def test_bytes_refuses(shape, want):
    n = C.c_uint64()
    assert api.lib().vg_k_kv4_bytes(*shape, C.byref(n)) == want
    assert api.lib().vg_k_kv4_bytes(1, 1, 128, 64, None) == EINVAL


CACHE_FAULTS = [({"data": None}, EINVAL), ({"state": None}, EINVAL), ({"data": A + 8}, EINVAL), ({"state": A + 4}, EINVAL),
                ({"weights": A + 2}, EINVAL), ({"seqs": 0}, EINVAL), ({"kv_heads": 0}, EINVAL), ({"capacity": 0}, EINVAL),
                ({"head_dim": 32}, EUNSUPPORTED), ({"capacity": 1 << 31}, ERANGE)]


def append(c, k=A, v=A, dtype=0, tokens=4, at=None, counts=None):
    return api.lib().vg_k_kv4_append(c, k, v, dtype, tokens, None, None, at, counts, None)


def read(c, first=None, tokens=4, dtype=1, k=A, v=A):
    return api.lib().vg_k_kv4_read(c, first, tokens, dtype, k, v, None)


def attention(c, q=A, dtype=0, heads=16, tokens=1, counts=None, scale=0.1, track=0, out=A, ws=A, ws_bytes=1 << 40):
    return api.lib().vg_k_kv4_attention(c, q, dtype, heads, tokens, None, counts, scale, track, out, ws, ws_bytes, None)


def evict(c, budget=128, recent=16, sinks=4, into=None):
    return api.lib().vg_k_kv4_evict(c, budget, recent, sinks, into, None)


@pytest.mark.parametrize("call", [append, read, attention, evict])
def test_a_bad_cache_is_refused(call):
    assert call(None) == EINVAL
    for over, want in CACHE_FAULTS:
        assert call(C.byref(desc(**over))) == want, over


@pytest.mark.parametrize("over,want", [
    ({"k": None}, EINVAL), ({"v": None}, EINVAL), ({"dtype": 8}, EUNSUPPORTED), ({"tokens": 0}, EINVAL),
    ({"tokens": 257}, EFULL), ({"k": A + 2}, EINVAL), ({"at": A + 1}, EINVAL), ({"counts": A + 2}, EINVAL),
])
def test_append_refuses(over, want):
    assert append(C.byref(desc()), **over) == want


@pytest.mark.parametrize("over,want", [
    ({"k": None}, EINVAL), ({"v": None}, EINVAL), ({"dtype": 2}, EUNSUPPORTED), ({"tokens": 0}, EINVAL),
    ({"k": A + 8}, EINVAL), ({"v": A + 4}, EINVAL), ({"first": A + 2}, EINVAL),
])
def test_read_refuses(over, want):
    assert read(C.byref(desc()), **over) == want


@pytest.mark.parametrize("over,want", [
    ({"q": None}, EINVAL), ({"out": None}, EINVAL), ({"ws": None}, EINVAL), ({"ws_bytes": 16}, EINVAL),
    ({"heads": 0}, EINVAL), ({"heads": 15}, EINVAL), ({"tokens": 0}, EINVAL), ({"dtype": 8}, EUNSUPPORTED),
    ({"scale": 0.0}, EINVAL), ({"scale": -1.0}, EINVAL), ({"scale": float("nan")}, EINVAL),
    ({"scale": float("inf")}, EINVAL), ({"q": A + 2}, EINVAL), ({"out": A + 8}, EINVAL), ({"ws": A + 8}, EINVAL),
    ({"counts": A + 1}, EINVAL), ({"tokens": 1 << 30}, ERANGE),
])
def test_attention_refuses(over, want):
    assert attention(C.byref(desc()), **over) == want


def test_attention_refuses_to_track_in_place():
    assert attention(C.byref(desc()), q=A, out=A, track=1) == EINVAL


def test_attention_refuses_to_track_without_weights():
    assert attention(C.byref(desc(weights=None)), track=1) == EINVAL


@pytest.mark.parametrize("cache,over,want", [
    ({"weights": None}, {}, EINVAL), ({"positions": None}, {}, EINVAL), ({}, {"budget": 0}, EINVAL),
    ({}, {"budget": 257}, ERANGE), ({}, {"budget": 16, "recent": 14, "sinks": 3}, ERANGE),
    ({}, {"recent": 0xFFFFFFFF, "sinks": 2}, ERANGE), ({"capacity": 65537}, {}, ERANGE),
])
def test_evict_refuses(cache, over, want):
    assert evict(C.byref(desc(**cache)), **over) == want


@pytest.mark.parametrize("over", [{"data": 2 * A}, {"seqs": 3}, {"kv_heads": 1}, {"head_dim": 64}, {"capacity": 128},
                                  {"weights": None}, {"positions": None}, {"state": 2 * A},
                                  {"state": 2 * A, "weights": 2 * A}])
def test_evict_refuses_another_cache(over):
    assert evict(C.byref(desc()), into=C.byref(desc(**over))) == EINVAL


def test_verify_refuses():
    good = dict(tokens=A, draft=A, target=A, u_accept=A, u_sample=A, counts=None, seqs=1, drafted=4, vocab=96, accepted=A,
                next=A, stream=None)
    for name in ("tokens", "draft", "target", "u_accept", "u_sample", "accepted", "next"):
        assert api.lib().vg_k_verify_draft(*{**good, name: None}.values()) == EINVAL, name
        assert api.lib().vg_k_verify_draft(*{**good, name: A + 2}.values()) == EINVAL, name
    for name in ("seqs", "drafted", "vocab"):
        assert api.lib().vg_k_verify_draft(*{**good, name: 0}.values()) == EINVAL, name
    assert api.lib().vg_k_verify_draft(*{**good, "vocab": 1 << 25}.values()) == ERANGE
    assert api.lib().vg_k_verify_draft(*{**good, "counts": A + 1}.values()) == EINVAL


def test_dynamic_shared_memory_is_declared_with_the_alignment_of_its_widest_access():
    """The kernels read and write it 16 bytes at a time; an element type of 1 or 4 bytes promises less."""
    from voxgen_b200._build import CSRC
    found = {}
    for path in CSRC.glob("kv4*.cuh"):
        for align, name in re.findall(r"extern __shared__ (?:__align__\((\d+)\) )?\w+ (\w+)\[\]", path.read_text()):
            found[name] = int(align or 0)
    assert len(found) == 4 and all(a >= 16 for a in found.values()), found
