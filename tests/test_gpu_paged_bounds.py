"""The paged attention's outputs one by one: each (query, head, channel) within a bound of its own, tight enough that a block of 16
rows left out of 20,000 shows. Helpers are test_gpu_paged.py's.

Bound, with p a query head's weights in 64 bits, S its largest sum of a score's magnitudes and A = sum(p |v|) of the channel:
half a step of the output's type at the exact value; S 2^-17 A, as scores are off by S 2^-18 at most (derived in
test_gpu_paged.py) and weights twice, above and below the line; and 2^-14 A for sums: at most 512 products are added to one
before it is added to another with rounding to nearest, each cut by 2^-23 of it at most, and P's terms, the exponential and the
joins (2^-18 in all) are well below what is left of that."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from test_gpu_paged import TYPES, filled, ints, normal, rows_of  # noqa: E402


def half_step(x, dtype):
    f = torch.finfo(TYPES[dtype])
    return (x.abs() * f.eps / 2).clamp_min(f.smallest_normal * f.eps / 2)


def exact(q, k, v, rows, scale):
    """Of one query's heads of one KV head: output and bound without the rounding of the output."""
    e = q @ k[rows].T * scale
    p = e.softmax(1)
    size = (q.abs() @ k[rows].abs().T).amax(1, keepdim=True) * scale
    return p @ v[rows], (size * 2.0 ** -17 + 2.0 ** -14) * (p @ v[rows].abs())


def check(cache, q, out, dtype, sequences=None, positions=None, chosen=None, teeth=0):
    """Every output; and of the first `teeth` queries that a block of 16 rows left out of the exact one would be found."""
    page, group = cache.table.page_rows, q.shape[1] // cache.kv_heads
    held = {}
    for i in range(len(q)):
        s = i if sequences is None else sequences[i]
        held[s] = held[s] if s in held else rows_of(cache, s)
        n = held[s][0].shape[1] if positions is None else positions[i] + 1
        for h in range(cache.kv_heads):
            k, v = held[s][0][h], held[s][1][h]
            rows = torch.arange(n, device="cuda")
            if chosen is not None:
                rows = torch.cat([rows[p * page:(p + 1) * page] for p in chosen[i][h] if p >= 0])
            mine = slice(h * group, (h + 1) * group)
            x, got = q[i, mine].double(), out[i, mine].double()
            want, bound = exact(x, k, v, rows, q.shape[2] ** -0.5)
            bound = bound + half_step(want, dtype)
            assert ((got - want).abs() <= bound).all(), (i, h, float(((got - want).abs() / bound).max()))
            if i < teeth:
                for at in (0, len(rows) // 32 * 16, (len(rows) - 1) // 16 * 16 - 16):
                    less = torch.cat((rows[:at], rows[at + 16:]))
                    assert ((exact(x, k, v, less, q.shape[2] ** -0.5)[0] - want).abs() > bound).any(), "the bound is too wide"


PAIRS = [(d, k) for d in TYPES for k in ("f16", "bf16")]


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 128), (8, 2, 64), (24, 1, 64)])
@pytest.mark.parametrize("dtype,kind", PAIRS)
def test_long_contexts(heads, kv_heads, dim, dtype, kind):
    """Segments cut into many pieces, with 1 and 4 tiles, and lists of chosen pages."""
    rows = [20000, 300, 9001]
    cache = filled(3, rows, 64, kv_heads, dim, kind)
    q = normal(4, 3, heads, dim, dtype=TYPES[dtype])
    check(cache, q, cache.attention(q), dtype, teeth=3)
    chosen = cache.select(q, 60, sinks=1, recent=2)
    check(cache, q, cache.attention(q, chosen=chosen), dtype, chosen=chosen.tolist())
    sequences, last = [0] * 5 + [2] * 2, [19995, 19996, 19997, 19998, 19999, 8999, 9000]
    q = normal(5, 7, heads, dim, dtype=TYPES[dtype])
    check(cache, q, cache.attention(q, sequences=ints(sequences), positions=ints(last)), dtype, sequences, last, teeth=1)


@pytest.mark.parametrize("dtype,kind", PAIRS)
def test_hundreds_of_segments(dtype, kind):
    """CTAs of 4 warps: whole segments and long ones that are cut, over all rows and over chosen pages, and drafts."""
    rng = np.random.default_rng(5)
    rows = rng.integers(1, 70, 230)
    rows[[3, 100]] = 20000, 1300
    cache = filled(1, rows.tolist(), 16, 2, 64, kind)
    q = normal(2, 230, 16, 64, dtype=TYPES[dtype])
    check(cache, q, cache.attention(q), dtype, teeth=0)
    check(cache, q[3:4], cache.attention(q)[3:4], dtype, [3], teeth=1)
    chosen = cache.select(q, 7, sinks=1, recent=2)
    check(cache, q, cache.attention(q, chosen=chosen), dtype, chosen=chosen.tolist())
    sequences = [s for s in (3, 100) for _ in range(130)]
    last = [int(x) for s in (3, 100) for x in rng.integers(rows[s] // 2, rows[s], 130)]
    q = normal(6, 260, 16, 64, dtype=TYPES[dtype])
    check(cache, q, cache.attention(q, sequences=ints(sequences), positions=ints(last)), dtype, sequences, last, teeth=1)
