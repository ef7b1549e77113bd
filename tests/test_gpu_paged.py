"""The paged cache on the GPU (step, append, select, attention), through ``voxgen_b200.paged``, against references
on the CPU (paged_reference.py).

Tolerances. An attention output is a mean of V weighted by exp(score). Scores: operands are held to at least 2^-22, and
up to 24 products of 16 channels are added with rounding towards zero, each within 2^-23 of S, the largest sum of the
magnitudes of a score's terms: S * 2^-18 with what is left over. That is a weight's relative error, and an output is off
by twice it times max|v|. Sums of P V: 24 such additions before fp32 output is rounded to nearest, then fp32 sums, the
exponential's 2^-22 and the joins: 2^-17 of max|v|. 16-bit output: its rounding (fp16 2^-11, bf16 2^-8), P's rounding
over an fp16 cache (2^-11, twice: above and below the line), and up to 2^9 additions of 2^-23 towards zero.
"""
import numpy as np
import pytest

import paged_reference as R

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from voxgen_b200 import paged  # noqa: E402
from voxgen_b200.api import VoxGenError  # noqa: E402

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EXTRA = {"f32": 0.0, "f16": 2.0 ** -11 + 2.0 ** -10, "bf16": 2.0 ** -8 + 2.0 ** -10}


def normal(seed, *shape, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).cuda()


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def host(x):
    return x.double().cpu().numpy()


# ---------------------------------------------------------------------------------------------
# step
# ---------------------------------------------------------------------------------------------
def check_step(table, ref, step, want):
    starts, slots, positions, sequences, runs = want
    assert step.starts.tolist() == starts
    assert step.slots.tolist() == slots
    assert step.positions.tolist() == positions
    assert step.sequences.tolist() == sequences
    assert step.runs.tolist() == runs
    assert table.table.tolist() == ref.table()
    assert table.rows.tolist() == ref.rows and table.status.tolist() == ref.status
    assert table.pool.tolist() == [len(ref.free), 0]
    assert table.free[:len(ref.free)].tolist() == ref.free


@pytest.mark.parametrize("seqs,pages,page,most,tokens", [
    (1, 1, 16, 1, 1), (1, 9, 16, 8, 130), (3, 5, 32, 8, 64), (33, 90, 16, 12, 300), (7, 14, 64, 20, 500),
    (40, 60, 128, 3, 5000), (300, 900, 16, 7, 9001), (1025, 700, 16, 2, 2050), (4096, 2500, 16, 3, 8197), (5, 5, 256, 9, 1001)])
def test_steps_follow_the_reference(seqs, pages, page, most, tokens):
    """Rounds of growing, cutting and finishing, with pools and sequences that run out, and counts out of range."""
    rng = np.random.default_rng(seqs + tokens)
    ref = R.Table(seqs, pages, page, most)
    table = paged.PageTable(seqs, pages, page, most)
    seen = set()
    for turn in range(12):
        mean = max(1, int(tokens / seqs * rng.choice([0.2, 0.9, 1.2])))
        counts = rng.integers(0, 2 * mean + 1, seqs)
        counts[rng.random(seqs) < 0.1] = 0
        if turn % 3 == 2:
            counts[rng.integers(0, seqs)] = rng.choice([-1, tokens + 1, -2 ** 31, 2 ** 31 - 1])
        if turn % 4 == 3 or seqs == 1:
            counts[rng.integers(0, seqs)] = min(tokens, most * page + rng.integers(-1, 2))
        keep = rng.integers(0, most * page + 3, seqs)
        keep[rng.random(seqs) < 0.5] = -1
        keep[rng.random(seqs) < 0.2] = 0
        use = None if turn % 5 == 4 else keep
        step = table.step(ints(counts), tokens, keep=None if use is None else ints(use))
        check_step(table, ref, step, ref.step(counts.tolist(), tokens, None if use is None else use.tolist()))
        seen |= set(ref.status)
    assert seqs < 5 or seen >= {0, R.NO_PAGES}


def test_a_step_that_only_gives_back():
    table, ref = paged.PageTable(3, 8, 16, 4), R.Table(3, 8, 16, 4)
    check_step(table, ref, table.step(ints([40, 0, 16]), 56), ref.step([40, 0, 16], 56))
    step = table.step(ints([0, 0, 0]), 0, keep=ints([17, 0, 0]))
    assert step.slots.numel() == 0 and step.runs.numel() == 0
    ref.step([0, 0, 0], 0, [17, 0, 0])
    assert table.table.tolist() == ref.table() and table.rows.tolist() == [17, 0, 0] and table.pool.tolist() == [6, 0]
    assert table.free[:6].tolist() == ref.free
    step = table.step(ints([1, 0, 0]), 0)      # no token fits no place
    assert table.status.tolist() == [paged.STATUS_BAD_COUNT, 0, 0] and table.rows.tolist() == [17, 0, 0]


def test_a_step_taken_back_gives_the_same_pages_again():
    table = paged.PageTable(6, 100, 16, 30)
    table.step(ints([5, 100, 0, 33, 17, 64]), 300)
    rows = table.rows.clone()
    counts = ints([20, 1, 90, 3, 0, 30])
    first = table.step(counts, 144)
    state = [x.clone() for x in (table.table, table.rows, table.pool, first.slots, first.runs)]
    for _ in range(3):
        again = table.step(counts, 144, keep=rows)
        for a, b in zip(state, (table.table, table.rows, table.pool, again.slots, again.runs)):
            assert torch.equal(a, b)


def test_a_step_writes_over_an_earlier_one():
    table = paged.PageTable(2, 10, 16, 5)
    step = table.step(ints([3, 2]), 6)
    assert step.positions.tolist() == [0, 1, 2, 0, 1, -1]
    assert table.step(ints([1, 2]), 6, into=step) is step
    assert step.positions.tolist() == [3, 2, 3, -1, -1, -1]
    with pytest.raises(VoxGenError, match="VG_EINVAL"):
        table.step(ints([1, 2]), 5, into=step)
    table.reset()
    assert table.rows.tolist() == [0, 0] and table.pool.tolist() == [10, 0] and (table.table == -1).all()
    assert table.free.tolist() == list(range(10))


# ---------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------
def shuffled(seqs, pages, page, most, seed=0):
    """A table whose pages come in a mixed order."""
    g = torch.Generator().manual_seed(seed)
    return paged.PageTable(seqs, pages, page, most, free=torch.randperm(pages, generator=g).int().cuda())


def extremes(k, dtype):
    """Smallest and largest of rows [rows, dim] per channel, as summaries hold them."""
    top = torch.finfo(dtype).max
    low = k.masked_fill(k.isnan(), float("inf")).amin(0)
    high = k.masked_fill(k.isnan(), -float("inf")).amax(0)
    none = k.isnan().all(0)
    return torch.stack((low, high)).clamp(-top, top).masked_fill(none, 0.0)


def expect_append(cache, layer, before, step, k, v, old_summaries):
    """The pool after an append, by torch on the host."""
    page = cache.table.page_rows
    data = before.clone()
    summaries = None if old_summaries is None else old_summaries.clone()
    filled = {}
    for t, slot in enumerate(step.slots.tolist()):
        if slot >= 0:
            data[slot // page, :, 0, slot % page] = k[t].cpu().to(cache.dtype)
            data[slot // page, :, 1, slot % page] = v[t].cpu().to(cache.dtype)
            filled[slot // page] = slot % page + 1
    if summaries is not None:
        for p, n in filled.items():
            for h in range(cache.kv_heads):
                summaries[p, h] = extremes(data[p, h, 0, :n], cache.dtype)
    return data, summaries


def same_bits(a, b):
    return torch.equal(a.cpu().view(torch.int16), b.cpu().view(torch.int16))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("page,kv_heads,dim,counts", [
    (16, 1, 64, [1]), (16, 2, 128, [15, 0, 17, 16]), (64, 3, 64, [130, 1, 63]), (32, 8, 128, [1, 1, 1, 1, 1]),
    (256, 1, 128, [300, 7])])
def test_append_holds_the_rounded_rows(dtype, kind, page, kv_heads, dim, counts):
    """Three appends one after the other, the second to the second layer; whatever no slot names stays as it was."""
    n = len(counts)
    table = shuffled(n, 3 * sum(-(-c // page) + 1 for c in counts), page, 4 + 3 * max(counts) // page)
    cache = paged.PagedCache(table, kv_heads, dim, dtype=TYPES[kind], layers=2, summaries=True)
    cache.data.copy_(normal(9, *cache.data.shape))
    for turn in range(3):
        layer = turn % 2
        tokens = sum(counts) + 3
        step = table.step(ints(counts), tokens)
        k, v = (normal(2 * turn + i, tokens, kv_heads, dim, dtype=TYPES[dtype]) for i in (0, 1))
        before = cache.data.cpu().clone()
        want, ends = expect_append(cache, layer, before[layer], step, k, v, cache.summaries[layer].cpu())
        cache.append(step, k, v, layer=layer)
        assert same_bits(cache.data[layer], want) and same_bits(cache.data[1 - layer], before[1 - layer])
        # equal numbers: a summary's zero may have either sign
        assert torch.equal(cache.summaries[layer].cpu(), ends)
        assert torch.equal(cache.k(layer), cache.data[layer, :, :, 0]) and torch.equal(cache.v(layer), cache.data[layer, :, :, 1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_append_special_values(kind, dtype):
    """What is past the cache's largest number is held as that one and reported, as is NaN; NaN is passed over by
    summaries, and a channel of NaN alone counts as 0."""
    t = TYPES[kind]
    inf, nan = float("inf"), float("nan")
    top = torch.finfo(t).max
    past = inf if dtype == "f16" else torch.finfo(TYPES[dtype]).max     # past fp16, and for fp32 past bf16
    k = torch.zeros(5, 1, 64, device="cuda")
    k[:, 0, 0] = torch.tensor([nan, 1.0, -2.0, nan, 0.5])
    k[:, 0, 1] = inf
    k[:, 0, 2] = -inf
    k[:, 0, 3] = nan
    k[:, 0, 4] = torch.tensor([inf, -inf, 0.0, nan, 1.0])
    k[:, 0, 5] = past
    k = k.to(TYPES[dtype])
    held = top if kind == "f16" or dtype == "f16" else past if dtype == "bf16" else top
    table = shuffled(1, 4, 16, 4)
    cache = paged.PagedCache(table, 1, 64, dtype=t, summaries=True)
    cache.append(table.step(ints([5]), 5), k, k)
    assert table.pool[1] == paged.STATUS_NONFINITE
    page = table.table[0, 0]
    low, high = cache.summaries[0, page, 0].double().cpu()
    assert low[:6].tolist() == [-2.0, top, -top, 0.0, -top, held]
    assert high[:6].tolist() == [1.0, top, -top, 0.0, top, held]
    assert not low[6:].any() and not high[6:].any()
    for row in (cache.k()[page, 0, 0], cache.v()[page, 0, 0]):
        row = row.double().cpu()
        assert row[0].isnan() and row[3].isnan() and row[[1, 2, 4, 5]].tolist() == [top, -top, top, held]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_append_reports_what_it_clamps(kind, dtype):
    """One value in K or V, at either end of a row, with and without summaries; the largest number itself does not count."""
    top = min(torch.finfo(TYPES[kind]).max, torch.finfo(TYPES[dtype]).max)
    if (kind, dtype) == ("f16", "bf16"):
        top = 65280.0       # bf16's largest below 65504, which it rounds to 65536
    for value, bit in ((top, 0), (-top, 0), (float("inf"), 16), (-float("inf"), 16), (float("nan"), 16)):
        for place in (0, 127):
            for summaries in (False, True):
                x = normal(3, 5, 2, 128, dtype=TYPES[dtype])
                y = x.clone()
                x[3, 1, place] = value
                for k, v in ((x, y), (y, x)):
                    table = shuffled(1, 4, 16, 4)
                    cache = paged.PagedCache(table, 2, 128, dtype=TYPES[kind], summaries=summaries)
                    cache.append(table.step(ints([5]), 5), k, v)
                    assert table.pool[1] == bit, (value, place)


@pytest.mark.parametrize("summaries", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_append_takes_any_strides(dtype, summaries):
    table = shuffled(2, 12, 16, 6)
    tokens, heads, dim = 45, 2, 128
    step = table.step(ints([20, 25]), tokens)
    wide = normal(1, tokens + 1, 3 * heads * dim + 1, dtype=TYPES[dtype])
    views = [wide[1:, :2 * heads * dim].unflatten(1, (2 * heads, dim)).split(heads, 1),            # odd base, odd rows
             wide.flatten()[:heads * tokens * dim * 2].view(heads * 2, tokens, dim).transpose(0, 1).split(heads, 1),   # head first
             (wide[:1, None, :dim].expand(tokens, heads, dim), wide[1:2, None, 1:dim + 1].expand(tokens, heads, dim))]  # strides of 0
    for k, v in views:
        plain, strided = (paged.PagedCache(table, heads, dim, summaries=summaries) for _ in range(2))
        plain.append(step, k.contiguous(), v.contiguous())
        strided.append(step, k, v)
        assert same_bits(plain.data, strided.data)
        assert not summaries or same_bits(plain.summaries, strided.summaries)


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
def filled(seed, rows, page, kv_heads, dim, kind="f16", spare=2, layers=1, garbage=True, most=0, layer=0):
    """A cache whose sequences hold rows[s] normal rows; every other place of its pool would read as NaN."""
    table = shuffled(len(rows), sum(-(-r // page) for r in rows) + spare, page, max(1, most, -(-max(rows) // page)), seed)
    cache = paged.PagedCache(table, kv_heads, dim, dtype=TYPES[kind], layers=layers, summaries=True)
    if garbage:
        cache.data.fill_(float("nan"))
    if sum(rows):
        step = table.step(ints(list(rows)), sum(rows))
        k, v = (normal(seed + i, sum(rows), kv_heads, dim) for i in (1, 2))
        cache.append(step, k, v, layer=layer)
    assert table.rows.tolist() == list(rows) and not table.status.any()
    return cache


def rows_of(cache, seq, layer=0):
    """K and V [kv_heads, rows, dim] that a sequence holds, in 64 bits."""
    n, page = int(cache.table.rows[seq]), cache.table.page_rows
    pages = cache.table.table[seq, :-(-n // page)].long()
    x = cache.data[layer][pages].double().permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :n]
    return x[:, 0], x[:, 1]


def check_attention(cache, q, out, dtype, sequences=None, positions=None, chosen=None, scale=None, layer=0):
    page = cache.table.page_rows
    held = {}
    top, most = 0.0, 1e-30
    want = torch.zeros(out.shape, dtype=torch.float64, device="cuda")
    group = q.shape[1] // cache.kv_heads
    for i in range(len(q)):
        s = i if sequences is None else sequences[i]
        if not 0 <= s < cache.table.seqs:
            continue
        if s not in held:
            held[s] = rows_of(cache, s, layer)
        k, v = held[s]
        n = k.shape[1] if positions is None else max(0, min(k.shape[1], positions[i] + 1))
        if chosen is None:
            mine = [torch.arange(n, device="cuda")] * cache.kv_heads
        else:
            mine = [torch.tensor([r for p in chosen[i][h] if p >= 0 for r in range(p * page, (p + 1) * page) if r < n],
                                 dtype=torch.long, device="cuda") for h in range(cache.kv_heads)]
        want[i] = R.attention(q[i], k, v, mine, scale)
        if n > 0:
            size = (q[i].double().abs().unflatten(0, (-1, group)) @ k[:, :n].abs().transpose(1, 2)).max()
            top = max(top, float(size) * (q.shape[2] ** -0.5 if scale is None else scale))
            most = max(most, float(v[:, :n].abs().max()))
    tol = (top * 2.0 ** -17 + 2.0 ** -17 + EXTRA[dtype]) * most
    worst = float((out.double() - want).abs().max())
    assert worst <= tol, (worst, tol)


SHAPES = [
    # heads, kv_heads, dim, page, rows of each sequence
    (16, 2, 128, 64, [513]), (16, 2, 64, 16, [1, 0, 17, 16, 15, 400]), (2, 1, 128, 32, [31, 32, 33, 1000, 2]),
    (8, 8, 64, 128, [129, 127, 5]), (12, 2, 128, 16, [700, 3, 64]), (32, 2, 128, 16, [90, 600]), (1, 1, 64, 256, [300, 255, 257]),
    (40, 2, 64, 32, [100, 1]), (6, 3, 128, 64, [1500] + [20] * 11), (16, 1, 128, 16, [2500, 1]),
]


@pytest.mark.parametrize("heads,kv_heads,dim,page,rows", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_attention_of_every_sequence(heads, kv_heads, dim, page, rows, dtype, kind):
    cache = filled(3, rows, page, kv_heads, dim, kind)
    q = normal(4, len(rows), heads, dim, dtype=TYPES[dtype])
    out = cache.attention(q)
    check_attention(cache, q, out, dtype)
    for s, n in enumerate(rows):
        assert n or not out[s].any()
    assert torch.equal(out, cache.attention(q))         # the same order of sums every time
    assert cache.table.pool[1] == 0


@pytest.mark.parametrize("dtype,kind", [("f32", "f16"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16")])
def test_attention_of_drafts_and_prompts(dtype, kind):
    """Several tokens of a sequence attend causally; padding, refused and unknown sequences give zeros."""
    cache = filled(5, [40, 300, 7], 16, 2, 128, kind, spare=10, most=30)
    table = cache.table
    step = table.step(ints([3, 4, 70]), 80)
    k, v = (normal(i, 80, 2, 128, dtype=TYPES[dtype]) for i in (7, 8))
    cache.append(step, k, v)
    q = normal(9, 80, 16, 128, dtype=TYPES[dtype])
    out = cache.attention(q, sequences=step.sequences, positions=step.positions)
    check_attention(cache, q, out, dtype, step.sequences.tolist(), step.positions.tolist())
    assert not out[77:].any()
    sequences, positions = [2, 0, 3, -1, 2 ** 31 - 1, -2 ** 31, 1, 1, 0], [5, 10 ** 9, 3, 3, 3, 3, -1, 0, -2 ** 31]
    out = cache.attention(q[:9], sequences=ints(sequences), positions=ints(positions))
    check_attention(cache, q[:9], out, dtype, sequences, positions)
    assert not out[2:7].any() and not out[8].any() and out[7].any()
    # either alone
    check_attention(cache, q[:4], cache.attention(q[:4], sequences=ints([1, 1, 0, 2])), dtype, [1, 1, 0, 2])
    check_attention(cache, q[:3], cache.attention(q[:3], positions=ints([4, -1, 16])), dtype, None, [4, -1, 16])


@pytest.mark.parametrize("seqs", [60, 150, 700])
def test_attention_of_many_sequences(seqs):
    """Segments in one, a few and no pieces each, with one long sequence among short ones."""
    rng = np.random.default_rng(seqs)
    rows = rng.integers(0, 120, seqs)
    rows[seqs // 3] = 5000
    cache = filled(1, rows.tolist(), 16, 2, 64, "f16")
    q = normal(2, seqs, 8, 64)
    check_attention(cache, q, cache.attention(q), "f32")


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 128), (8, 2, 64), (24, 1, 64), (72, 1, 128)])
@pytest.mark.parametrize("dtype,kind", [("f32", "f16"), ("f32", "bf16"), ("bf16", "bf16")])
def test_attention_of_long_contexts(heads, kv_heads, dim, dtype, kind):
    """The ring of copies goes round many times, with teams of 1 to 8 warps in a CTA one after the other."""
    rows = [20000, 7, 9001, 300]
    cache = filled(3, rows, 64, kv_heads, dim, kind)
    q = normal(4, 4, heads, dim, dtype=TYPES[dtype])
    check_attention(cache, q, cache.attention(q), dtype)
    rng = np.random.default_rng(heads)
    sequences = [s for s in rng.integers(0, 4, 14) for _ in range(rng.integers(1, 10))]
    positions = [int(max(0, rows[s] - 1 - rng.integers(0, 40))) for s in sequences]
    q = normal(5, len(sequences), heads, dim, dtype=TYPES[dtype])
    out = cache.attention(q, sequences=ints(sequences), positions=ints(positions))
    check_attention(cache, q, out, dtype, sequences, positions)
    again = cache.attention(q, sequences=ints(sequences), positions=ints(positions))
    assert torch.equal(out, again)


@pytest.mark.parametrize("heads,dim", [(16, 128), (40, 64), (48, 128)])
@pytest.mark.parametrize("dtype,kind", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("f16", "bf16"), ("bf16", "bf16")])
def test_attention_of_hundreds_of_segments(heads, dim, dtype, kind):
    """Enough of them for CTAs of 4 warps, with long ones that are cut, over all rows and over chosen pages."""
    rng = np.random.default_rng(heads)
    rows = rng.integers(0, 70, 230)
    rows[[3, 100]] = 2500, 1300
    cache = filled(1, rows.tolist(), 16, 2, dim, kind)
    q = normal(2, 230, heads, dim, dtype=TYPES[dtype])
    out = cache.attention(q)
    check_attention(cache, q, out, dtype)
    assert torch.equal(out, cache.attention(q))
    chosen = cache.select(q, 7, sinks=1, recent=2)
    check_attention(cache, q, cache.attention(q, chosen=chosen), dtype, chosen=chosen.tolist())


@pytest.mark.parametrize("kv_heads", [1, 3])
def test_attention_of_more_queries_than_are_planned_ahead(kv_heads):
    """Tokens of a few sequences, in runs, past what a CTA keeps in shared memory, with and without cut segments."""
    rng = np.random.default_rng(kv_heads)
    rows = [4000, 10, 700]
    cache = filled(1, rows, 32, kv_heads, 64, "f16")
    sequences = [s for s in rng.integers(-1, 4, 400) for _ in range(rng.integers(1, 9))]
    positions = [int(rng.integers(0, rows[s])) if 0 <= s < 3 else 5 for s in sequences]
    assert len(sequences) > 1100
    q = normal(3, len(sequences), 8 * kv_heads, 64, dtype=torch.float16)
    out = cache.attention(q, sequences=ints(sequences), positions=ints(positions))
    check_attention(cache, q, out, "f16", sequences, positions)
    some = [i for i, s in enumerate(sequences) if s == 0][:300]     # between the two: 300 queries, CTAs of 12 warps for 1 KV head
    at = torch.tensor(some, device="cuda")
    out = cache.attention(q[at], sequences=ints(sequences)[at], positions=ints(positions)[at])
    check_attention(cache, q[at], out, "f16", [sequences[i] for i in some], [positions[i] for i in some])


def test_attention_of_many_drafts():
    """More segments than CTAs, so that a CTA's pieces differ in their tiles."""
    rng = np.random.default_rng(1)
    rows = rng.integers(1, 900, 40).tolist()
    cache = filled(3, rows, 16, 2, 64, "f16")
    sequences = [s for s in range(40) for _ in range(rng.integers(1, 12))]
    positions = [int(rng.integers(0, rows[s])) for s in sequences]
    q = normal(5, len(sequences), 16, 64)
    out = cache.attention(q, sequences=ints(sequences), positions=ints(positions))
    check_attention(cache, q, out, "f32", sequences, positions)


def test_a_row_that_only_later_tokens_see_may_hold_anything():
    """NaN in the row of a draft's second token leaves its first token's output alone."""
    cache = filled(3, [40, 33], 16, 1, 64, "f16")
    table = cache.table
    q = normal(5, 4, 8, 64)
    sequences, positions = ints([0, 0, 0, 1]), ints([37, 38, 39, 32])
    want = cache.attention(q, sequences=sequences, positions=positions)
    for part in (cache.k(), cache.v()):
        place = int(table.table[0, 38 // 16]), 0, 38 % 16
        kept = part[place].clone()
        part[place] = float("nan")
        out = cache.attention(q, sequences=sequences, positions=positions)
        assert torch.equal(out[[0, 3]], want[[0, 3]]) and out[1:3].isnan().all()
        part[place] = kept


def test_attention_of_more_segments_than_are_cut():
    cache = filled(1, [70, 20], 16, 1, 64, "f16")
    n = (1 << 14) + 5
    q = normal(2, n, 1, 64)
    sequences, positions = [i % 2 for i in range(n)], [i % 75 for i in range(n)]
    out = cache.attention(q, sequences=ints(sequences), positions=ints(positions))
    check_attention(cache, q, out, "f32", sequences, positions)


def test_attention_takes_strides_scale_and_out():
    cache = filled(2, [100, 33], 32, 2, 64, "bf16")
    wide = normal(3, 3, 9 * 64 + 1)
    q = wide[1:, 1:8 * 64 + 1].unflatten(1, (8, 64))
    out = torch.full((2, 8, 64), 7.0, device="cuda")
    assert cache.attention(q, scale=0.3, out=out) is out
    check_attention(cache, q, out, "f32", scale=0.3)
    t = wide.flatten()[:8 * 2 * 64].view(8, 2, 64).transpose(0, 1)
    check_attention(cache, t, cache.attention(t), "f32")
    one = normal(4, 1, 1, 64).expand(2, 8, 64)
    check_attention(cache, one, cache.attention(one), "f32")


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_large_and_special_values(kind, dtype):
    """Scores far apart, a head of zeros, and NaN among the rows that are held: it reaches the outputs of its sequence (in K)
    or its channel (in V), and no others."""
    cache = filled(6, [200, 200, 200, 200, 40], 16, 1, 64, kind)
    table = cache.table
    where = [(int(table.table[s, 3]), 5) for s in range(4)]           # row 53 of each
    for s, x in enumerate([100.0, -60000.0, float("nan")]):
        cache.k()[where[s][0], 0, 5] = x
    cache.v()[where[3][0], 0, 5, 7] = float("nan")
    q = normal(1, 5, 4, 64, dtype=TYPES[dtype]).abs() + 0.5
    q[0, 1] = 0
    out = cache.attention(q)
    assert out[2].isnan().all() and out[3, :, 7].isnan().all()
    cache.v()[where[3][0], 0, 5, 7] = 0.0
    clean = [0, 1, 4]
    check_attention(cache, q[clean], out[clean], dtype, clean)
    rest = [c for c in range(64) if c != 7]
    assert torch.equal(out[3][:, rest], cache.attention(q)[3][:, rest])
    # a query of NaN, and one of infinities
    q[0, 0, 3], q[1, 2, 5] = float("nan"), float("inf")
    bad = cache.attention(q)
    assert bad[0, 0].isnan().all() and bad[1, 2].isnan().all()
    assert torch.equal(bad[0, 1:], out[0, 1:]) and torch.equal(bad[4], out[4])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_attention_of_scores_of_minus_infinity(kind):
    """Every score -infinity: NaN, as the formula's 0 / 0. (16-bit queries: their terms are not split.)"""
    cache = filled(6, [200, 40], 16, 1, 64, kind)
    cache.k().fill_(float("-inf"))
    q = normal(1, 2, 4, 64, dtype=TYPES[kind]).abs() + 0.5
    assert cache.attention(q).isnan().all()


def test_attention_of_scores_past_two_to_the_24():
    """A softmax of scores that far apart is the mean of V over the rows of the largest one."""
    for kind in ("f16", "bf16"):
        cache = filled(6, [300], 16, 1, 64, kind)
        cache.k().mul_(200)
        q = normal(1, 1, 2, 64) * 1e4
        out = host(cache.attention(q))[0]
        k, v = rows_of(cache, 0)
        best = (k[0] @ q[0].double().T).argmax(0)
        np.testing.assert_allclose(out, host(v[0, best]), rtol=2.0 ** -20, atol=2.0 ** -20)


def test_damaged_tables_read_no_bad_page():
    cache = filled(6, [100, 50], 16, 2, 64, "f16", spare=0)
    table = cache.table.table
    good = table[0].clone()
    q = normal(1, 2, 4, 64)
    alone = cache.attention(q)[1]
    for bad in (-1, 10 ** 9, cache.table.pages, -2 ** 31):
        table[0, 2] = bad
        out = cache.attention(q)          # rows of the page are passed over
        assert torch.isfinite(out).all() and torch.equal(out[1], alone)
        cache.select(q, 3)
    table[0] = good
    cache.table.rows[0] = 2 ** 31 - 1     # no more rows than the table has room for
    assert cache.attention(q).shape == q.shape


def test_offsets_past_32_bits():
    """A pool of 5 GB whose sequence lies at both ends."""
    page, heads, dim = 64, 8, 128
    pages = 5 * (1 << 30) // (2 * heads * page * dim * 2)
    table = paged.PageTable(1, pages, page, 4)
    table.free[:] = torch.arange(pages, device="cuda").roll(2)     # ... the last pages first
    cache = paged.PagedCache(table, heads, dim, summaries=True)
    table.free[pages - 4:] = ints([0, pages - 1, 1, pages - 2])
    step = table.step(ints([200]), 200)
    assert table.table[0].tolist() == [0, pages - 1, 1, pages - 2]
    k, v = (normal(i, 200, heads, dim) for i in (1, 2))
    cache.append(step, k, v)
    assert torch.equal(cache.k()[pages - 1, :, 0], k[64].half())
    q = normal(3, 1, heads, dim)
    check_attention(cache, q, cache.attention(q), "f32")
    chosen = cache.select(q, 2, recent=1)
    for h in range(heads):
        low, high = (host(cache.summaries[0, table.table[0].long(), h, i]) for i in (0, 1))
        assert chosen[0, h].tolist() == R.choose(host(q)[0, h:h + 1], low, high, 2, 0, 1)


# ---------------------------------------------------------------------------------------------
# select, and attention of what it chose
# ---------------------------------------------------------------------------------------------
def check_select(cache, q, chosen, budget, sinks, recent, sequences=None, positions=None):
    group, page = q.shape[1] // cache.kv_heads, cache.table.page_rows
    x, got = host(q), chosen.tolist()
    ends = host(cache.summaries[0])
    table, rows = cache.table.table.tolist(), cache.table.rows.tolist()
    for i in range(len(x)):
        s = i if sequences is None else sequences[i]
        n = rows[s] if positions is None else min(rows[s], positions[i] + 1)
        pages = table[s][:-(-n // page)]
        for h in range(cache.kv_heads):
            want = R.choose(x[i, h * group:(h + 1) * group], ends[pages, h, 0], ends[pages, h, 1], budget, sinks, recent)
            assert got[i][h] == want, (i, h)


@pytest.mark.parametrize("heads,kv_heads,dim,page,rows", SHAPES)
@pytest.mark.parametrize("dtype,kind", [("f32", "f16"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f16")])
def test_select_and_attention(heads, kv_heads, dim, page, rows, dtype, kind):
    cache = filled(3, rows, page, kv_heads, dim, kind)
    q = normal(4, len(rows), heads, dim, dtype=TYPES[dtype])
    for budget, sinks, recent in ((1, 0, 1), (1, 0, 0), (2, 1, 1), (5, 1, 2), (9, 0, 0), (200, 3, 4)):
        chosen = cache.select(q, budget, sinks=sinks, recent=recent)
        check_select(cache, q, chosen, budget, sinks, recent)
        out = cache.attention(q, chosen=chosen)
        check_attention(cache, q, out, dtype, chosen=chosen.tolist())
    # all pages: the same rows as without a list
    check_attention(cache, q, cache.attention(q, chosen=cache.select(q, 200)), dtype)


def test_select_of_drafts():
    cache = filled(5, [400, 900], 16, 2, 64, "f16")
    sequences, positions = [0, 1, 1, 0, 1], [399, 899, 500, 16, -1]
    q = normal(9, 5, 8, 64)
    chosen = cache.select(q, 6, sinks=1, recent=2, sequences=ints(sequences), positions=ints(positions))
    check_select(cache, q, chosen, 6, 1, 2, sequences, positions)
    assert chosen[4].eq(-1).all()
    out = cache.attention(q, sequences=ints(sequences), positions=ints(positions), chosen=chosen)
    check_attention(cache, q, out, "f32", sequences, positions, chosen.tolist())


@pytest.mark.parametrize("pages", [300, 2048, 8192, 24576])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_select_among_many_pages(pages, kind):
    """Summaries alone: scores of every spread, crowded ones and ties among them."""
    for style in ("normal", "ties", "crowded", "wild"):
        table = shuffled(2, pages * 2, 16, pages)
        cache = paged.PagedCache(table, 1, 64, dtype=TYPES[kind], summaries=True)
        table.step(ints([pages * 16 - 3, pages * 8]), pages * 24)
        g = torch.Generator().manual_seed(pages)
        ends = torch.randn(2 * pages, 1, 2, 64, generator=g)
        if style == "ties":
            ends = torch.randint(-1, 2, ends.shape, generator=g).float() * (torch.rand(2 * pages, 1, 1, 1, generator=g) < 0.01)
        elif style == "crowded":
            ends = 1000 + ends.round() / 8 * (torch.rand(2 * pages, 1, 1, 1, generator=g) < 0.5)
        elif style == "wild":
            ends = ends * torch.exp2(torch.randint(-14, 14, (2 * pages, 1, 1, 1), generator=g).float())
        ends = ends.sort(2).values
        cache.summaries[0].copy_(ends)
        q = torch.randint(-3, 4, (2, 2, 64), generator=g).float().cuda() if style in ("ties", "crowded") else normal(3, 2, 2, 64)
        for budget, sinks, recent in ((64, 1, 2), (pages - 1, 0, 1), (17, 0, 0)):
            check_select(cache, q, cache.select(q, budget, sinks=sinks, recent=recent), budget, sinks, recent)


def test_select_of_special_queries():
    cache = filled(5, [400, 400, 400, 400], 16, 1, 64, "f16")
    q = normal(9, 4, 2, 64)
    q[0, 0, 3] = float("nan")
    q[1, 1, 5] = float("inf")
    q[2, 0, 7] = float("-inf")
    q[3] = 0
    check_select(cache, q, cache.select(q, 5, recent=1), 5, 0, 1)
    assert cache.select(q, 5, recent=1)[3, 0].tolist() == [0, 1, 2, 3, 24]      # all equal: the lowest pages
    for power in (-140, 120):
        big = normal(9, 4, 2, 64) * 2.0 ** power
        check_select(cache, big, cache.select(big, 5, recent=1), 5, 0, 1)


def test_attention_of_any_list():
    """Lists that no selection made: in any order, with gaps, pages past the rows, and a page named twice."""
    cache = filled(5, [100, 33], 16, 2, 64, "f16", most=9)
    q = normal(9, 2, 8, 64)
    lists = [[[6, -1, 0, 3], [-1, -1, -1, -1]], [[2, 1, 8, 2], [100, -5, 2 ** 31 - 1, 0]]]
    out = cache.attention(q, chosen=ints(lists))
    check_attention(cache, q, out, "f32", chosen=[[[p if p < 9 else -1 for p in x] for x in y] for y in lists])
    assert not out[0, 4:].any()


# ---------------------------------------------------------------------------------------------
# together, and in a program
# ---------------------------------------------------------------------------------------------
def test_a_serving_loop():
    """Requests come, grow, have drafts rejected and finish; every layer's attention is that of the rows they were given."""
    rng = np.random.default_rng(5)
    seqs, page, kv_heads, dim, layers = 6, 16, 2, 64, 2
    table = shuffled(seqs, 28, page, 20)
    cache = paged.PagedCache(table, kv_heads, dim, dtype=torch.float16, layers=layers, summaries=True)
    ref = R.Table(seqs, 0, page, 20, free=table.free.tolist())
    held = [[(np.zeros((0, kv_heads, dim)),) * 2 for _ in range(layers)] for _ in range(seqs)]
    refused = 0
    for turn in range(25):
        keep = np.full(seqs, -1)
        for s in range(seqs):
            if rng.random() < 0.12:
                keep[s] = 0                                   # finished
            elif rng.random() < 0.4:
                keep[s] = max(0, ref.rows[s] - rng.integers(0, 4))   # rejected drafts
        counts = np.where(keep == 0, rng.integers(1, 200, seqs), rng.integers(0, 5, seqs))
        tokens = int(counts.sum()) + 2
        step = table.step(ints(counts), tokens, keep=ints(keep))
        check_step(table, ref, step, ref.step(counts.tolist(), tokens, keep.tolist()))
        refused += sum(x != 0 for x in ref.status)
        starts = step.starts.tolist()
        for layer in range(layers):
            k, v = (normal(100 * turn + 2 * layer + i, tokens, kv_heads, dim) for i in (0, 1))
            cache.append(step, k, v, layer=layer)
            q = normal(turn, tokens, 8, dim)
            out = cache.attention(q, sequences=step.sequences, positions=step.positions, layer=layer)
            check_attention(cache, q, out, "f32", step.sequences.tolist(), step.positions.tolist(), layer=layer)
            for s in range(seqs):
                cut = ref.rows[s] - (counts[s] if ref.status[s] == 0 else 0)
                new = [host(x[starts[s]:starts[s + 1]].half()) if ref.status[s] == 0 else x[:0].cpu().numpy() for x in (k, v)]
                held[s][layer] = tuple(np.concatenate((a[:cut], b)) for a, b in zip(held[s][layer], new))
                for mine, theirs in zip(held[s][layer], rows_of(cache, s, layer)):
                    np.testing.assert_array_equal(mine.transpose(1, 0, 2), host(theirs))
            chosen = cache.select(q, 4, sinks=1, recent=1, sequences=step.sequences, positions=step.positions, layer=layer)
            out = cache.attention(q, sequences=step.sequences, positions=step.positions, chosen=chosen, layer=layer)
            check_attention(cache, q, out, "f32", step.sequences.tolist(), step.positions.tolist(), chosen.tolist(), layer=layer)
    assert refused


@pytest.mark.parametrize("budget", [None, 2])
@pytest.mark.parametrize("pages", [64, 9])
def test_the_serving_example(budget, pages):
    """Every request gets its tokens and all pages come back, also where requests have to wait for pages; with all pages
    attended, a request's tokens do not depend on what else is served."""
    import sys
    from pathlib import Path
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
    import paged_serving
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, 500, n).tolist() for n in (3, 40, 17, 60, 1, 33, 90)]
    answers, table = paged_serving.serve(prompts, new=9, pages=pages, budget=budget)
    assert [len(x) for x in answers] == [9] * 7 and table.pool.tolist() == [pages, 0] and not table.rows.any()
    if budget is None:
        for i in (0, 3, 6):
            alone, _ = paged_serving.serve(prompts[i:i + 1], new=9)
            assert alone[0][:4] == answers[i][:4]      # greedy choices between near scores may part later


def test_a_captured_loop_replays():
    """A decode step captured once and replayed gives what eager calls give, bit for bit."""
    def build():
        cache = filled(5, [100, 40, 7], 16, 2, 64, "f16", spare=30, most=20)
        return cache, ints([1, 1, 1]), normal(1, 3, 2, 64), normal(2, 3, 2, 64), normal(3, 3, 8, 64)

    def once(cache, counts, k, v, q, step=None):
        step = cache.table.step(counts, 3, into=step)
        cache.append(step, k, v)
        out = cache.attention(q, sequences=step.sequences, positions=step.positions)
        chosen = cache.select(q, 3, recent=1)
        return step, out, cache.attention(q, chosen=chosen), chosen

    eager, captured = build(), build()
    captured[0].reserve(3, 8)
    captured[0].reserve(3, 8, 3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = once(*captured)
    for turn in range(20):
        for a, b in zip(eager[2:], captured[2:]):
            x = normal(10 + turn, *a.shape)
            a.copy_(x)
            b.copy_(x)
        want = once(*eager)
        graph.replay()
        torch.cuda.synchronize()
        assert want[0].slots.tolist() == kept[0].slots.tolist()
        for a, b in zip(want[1:], kept[1:]):
            assert torch.equal(a, b)
        assert same_bits(eager[0].data, captured[0].data) and same_bits(eager[0].summaries, captured[0].summaries)
    assert eager[0].table.rows.tolist() == [120, 60, 27] == captured[0].table.rows.tolist()


def test_a_graph_replays_after_its_workspace_was_outgrown():
    cache = filled(5, [600, 40], 16, 2, 64, "f16")
    q = normal(1, 2, 8, 64)
    want = cache.attention(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attention(q)
    size = cache._workspace.numel()
    many = normal(2, 2000, 8, 64)
    cache.attention(many, sequences=ints([0, 1] * 1000))
    assert cache._workspace.numel() > size
    junk = torch.full((size,), 255, dtype=torch.uint8, device="cuda")   # would land where a freed workspace was
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    assert junk.numel() == size and torch.equal(cache.attention(q), want)


def test_a_graph_without_a_reserved_workspace():
    cache = filled(5, [600, 40], 16, 2, 64, "f16")
    q = normal(1, 2, 8, 64)
    paged.PagedCache(cache.table, 2, 64).attention(q)      # loads the kernels
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attention(q)
        with pytest.raises(VoxGenError, match="VG_EINVAL"):
            cache.reserve(2, 8)
    assert cache._workspace is None
    for _ in range(2):
        graph.replay()
        check_attention(cache, q, out, "f32")


def test_calls_on_another_stream():
    table = shuffled(2, 20, 16, 10)
    cache = paged.PagedCache(table, 2, 64, summaries=True)
    k, v, q = normal(1, 100, 2, 64), normal(2, 100, 2, 64), normal(3, 2, 8, 64)
    counts = ints([60, 40])
    for stream in (torch.cuda.Stream(), torch.cuda.Stream()):
        table.reset()
        cache.data.zero_()
        torch.cuda.synchronize()
        raw = stream.cuda_stream if stream is not None else 0
        torch.cuda._sleep(10 ** 6)                         # the default stream is busy meanwhile
        step = table.step(counts, 100, stream=stream)
        cache.append(step, k, v, stream=raw)
        out = cache.attention(q, stream=stream)
        chosen = cache.select(q, 2, stream=stream)
        sparse = cache.attention(q, chosen=chosen, stream=raw)
        torch.cuda.synchronize()
        check_attention(cache, q, out, "f32")
        check_select(cache, q, chosen, 2, 0, 1)
        check_attention(cache, q, sparse, "f32", chosen=chosen.tolist())


def test_one_workspace_serves_calls_of_any_shape():
    cache = filled(5, [3000, 40, 900], 16, 2, 64, "f16")
    table = cache.table
    calls = [(1, 8), (3, 16), (2, 2), (3, 40), (1, 16)]
    cache.reserve(3, 40)
    for n, heads in calls * 2:
        q = normal(n + heads, n, heads, 64)
        fresh = paged.PagedCache(table, 2, 64, data=cache.data[0], summaries=cache.summaries[0])
        assert torch.equal(cache.attention(q), fresh.attention(q))
        chosen = cache.select(q, 20)
        assert torch.equal(cache.attention(q, chosen=chosen), fresh.attention(q, chosen=chosen))


def test_a_step_of_arrays_in_hand():
    table = shuffled(2, 20, 16, 10)
    step = table.step(ints([30, 11]), 50)
    copy = paged.Step.of(table, *(x.clone() for x in (step.starts, step.slots, step.positions, step.sequences, step.runs)))
    k, v = normal(1, 50, 2, 64), normal(2, 50, 2, 64)
    a, b = (paged.PagedCache(table, 2, 64, summaries=True) for _ in range(2))
    a.append(step, k, v)
    b.append(copy, k, v)
    assert same_bits(a.data, b.data) and same_bits(a.summaries, b.summaries)


def test_calls_without_queries_or_tokens():
    cache = filled(5, [60, 40], 16, 2, 64, "f16")
    q = normal(1, 0, 8, 64)
    assert cache.attention(q).shape == (0, 8, 64)
    assert cache.select(q, 3).shape == (0, 2, 3)
    step = cache.table.step(ints([0, 0]), 0)
    before = cache.data.clone()
    cache.append(step, normal(1, 0, 2, 64), normal(1, 0, 2, 64))
    assert same_bits(before, cache.data) and cache.table.rows.tolist() == [60, 40]


def test_refusals():
    cache = filled(5, [60, 40], 16, 2, 64, "f16")
    table = cache.table
    q = normal(1, 2, 8, 64)
    step = table.step(ints([1, 1]), 2)
    k = normal(2, 2, 2, 64)

    def refused(call, code="VG_EINVAL"):
        with pytest.raises(VoxGenError, match=code):
            call()

    refused(lambda: table.step(ints([1]), 2))
    refused(lambda: table.step(ints([1, 1]).long(), 2))
    refused(lambda: table.step(ints([1, 1]).cpu(), 2))
    refused(lambda: table.step(ints([1, 1]), -1))
    refused(lambda: table.step(ints([1, 1]), 1 << 31), "VG_ERANGE")
    refused(lambda: table.step(ints([1, 1]), 2, keep=ints([1, 1, 1])))
    refused(lambda: cache.append(step, k, k[:1]))
    refused(lambda: cache.append(step, k[:1], k[:1]))
    refused(lambda: cache.append(step, k, k.half()))
    refused(lambda: cache.append(step, k.double(), k.double()), "VG_EUNSUPPORTED")
    refused(lambda: cache.append(paged.PageTable(2, 10, 16, 5).step(ints([1, 1]), 2), k, k))     # another table's
    refused(lambda: table.step(ints([1, 1]), 2, into=paged.PageTable(2, 10, 16, 5).step(ints([1, 1]), 2)))
    refused(lambda: cache.append(step, k, k, layer=1))
    refused(lambda: cache.append(step, k, k, layer=-1))
    refused(lambda: cache.append(step, k.transpose(1, 2).contiguous().transpose(1, 2), k))
    refused(lambda: cache.attention(q[0]))
    refused(lambda: cache.attention(q[:, :7]))
    refused(lambda: cache.attention(normal(1, 3, 8, 64)))                 # no sequence 2
    refused(lambda: cache.attention(q, sequences=ints([0])))
    refused(lambda: cache.attention(q, positions=ints([0, 1]).long()))
    refused(lambda: cache.attention(q, scale=0.0))
    refused(lambda: cache.attention(q, scale=float("nan")))
    refused(lambda: cache.attention(q, out=q))
    refused(lambda: cache.attention(q, out=torch.empty(2, 8, 64, dtype=torch.float16, device="cuda")))
    refused(lambda: cache.attention(q, chosen=ints([[0], [1]])))
    refused(lambda: cache.attention(q, chosen=torch.empty(2, 2, 0, dtype=torch.int32, device="cuda")))
    refused(lambda: cache.attention(q, chosen=ints([[[0], [1]]])))
    refused(lambda: cache.attention(q.double()), "VG_EUNSUPPORTED")
    refused(lambda: cache.select(q, 0))
    refused(lambda: cache.select(q, 2, sinks=2, recent=1), "VG_ERANGE")
    refused(lambda: cache.select(q, 2, sinks=-1))
    refused(lambda: paged.PagedCache(table, 2, 64).select(q, 2))          # keeps no summaries
    refused(lambda: paged.PagedCache(table, 2, 64, dtype=torch.float32), "VG_EUNSUPPORTED")
    refused(lambda: paged.PagedCache(table, 2, 96), "VG_EUNSUPPORTED")
    refused(lambda: paged.PagedCache(table, 2, 64, layers=0))
    refused(lambda: paged.PagedCache(table, 2, 64, data=cache.data[0, :-1]))
    refused(lambda: paged.PageTable(2, 10, 24, 5), "VG_EUNSUPPORTED")
    refused(lambda: paged.PageTable(5000, 10, 16, 5), "VG_ERANGE")
    refused(lambda: paged.PageTable(2, 10, 16, 5, rows=ints([0])))
    refused(lambda: paged.PageTable(2, 10, 16, 5, device="cpu"))
    refused(lambda: paged.Step.of(table, step.starts, step.slots, step.positions, step.sequences, step.runs[:-1]))
    assert table.rows.tolist() == [61, 41]
