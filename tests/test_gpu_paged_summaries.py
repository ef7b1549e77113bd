"""Summaries of a paged cache's pages, and what selection makes of them, as rows come and go. Helpers are test_gpu_paged.py's."""
import numpy as np
import pytest

import paged_reference as R

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from test_gpu_paged import check_attention, check_select, extremes, filled, ints, normal, rows_of, shuffled  # noqa: E402
from voxgen_b200 import paged  # noqa: E402


def test_a_cut_page_keeps_its_summary_until_its_next_append():
    """A page whose rows are cut counts as it did at its last append; the next one takes the rows that it then holds."""
    cache = filled(5, [400, 300], 16, 2, 64, "f16", spare=4)
    table = cache.table
    page = int(table.table[0, 9])                                     # rows 144 .. 159 of sequence 0
    cache.k()[page, :, 8] = 9.0                                       # row 152 is dropped and had been the largest
    cache.summaries[0, page, :, 1] = 9.0
    kept = cache.summaries.clone()
    step = table.step(ints([0, 0]), 0, keep=ints([150, -1]))
    cache.append(step, normal(1, 0, 2, 64), normal(1, 0, 2, 64))
    assert torch.equal(cache.summaries, kept) and table.rows.tolist() == [150, 300]
    q = normal(9, 2, 8, 64)
    for budget, sinks, recent in ((3, 0, 0), (4, 1, 1)):
        chosen = cache.select(q, budget, sinks=sinks, recent=recent)
        check_select(cache, q, chosen, budget, sinks, recent)         # by the summaries as they are
        out = cache.attention(q, chosen=chosen)
        check_attention(cache, q, out, "f32", chosen=chosen.tolist())
        assert 9 in chosen[0, 0].tolist()
    step = table.step(ints([1, 0]), 1)
    k = normal(2, 1, 2, 64)
    cache.append(step, k, k)
    held = rows_of(cache, 0)[0][:, 144:]
    assert held.shape[1] == 7
    for h in range(2):
        assert torch.equal(cache.summaries[0, page, h].double(), extremes(held[h], torch.float16))
    check_select(cache, q, cache.select(q, 3), 3, 0, 1)


def test_selection_in_a_serving_loop():
    """Requests come, grow, have rows rejected and finish: summaries are those of the rows at each page's last append, and
    every choice is the definition's."""
    rng = np.random.default_rng(7)
    seqs, page, kv_heads, dim = 5, 16, 2, 64
    table = shuffled(seqs, 40, page, 14)
    cache = paged.PagedCache(table, kv_heads, dim, dtype=torch.bfloat16, summaries=True)
    ref = R.Table(seqs, 0, page, 14, free=table.free.tolist())
    want = torch.zeros_like(cache.summaries[0])
    cut = 0
    for turn in range(30):
        keep, counts = np.full(seqs, -1), rng.integers(0, 4, seqs)
        for s in range(seqs):
            if rng.random() < 0.1:
                keep[s], counts[s] = 0, rng.integers(1, 200)
            elif rng.random() < 0.4:
                keep[s] = max(0, ref.rows[s] - rng.integers(1, 30))
                counts[s] *= rng.random() < 0.5                       # often none: the cut page gets no append
                cut += counts[s] == 0 and keep[s] % page != 0
        tokens = int(counts.sum()) + 1
        step = table.step(ints(counts), tokens, keep=ints(keep))
        runs = ref.step(counts.tolist(), tokens, keep.tolist())[4]
        assert table.rows.tolist() == ref.rows and table.table.tolist() == ref.table()
        k, v = (normal(2 * turn + i, tokens, kv_heads, dim) * rng.choice([0.2, 1, 3]) for i in (0, 1))
        cache.append(step, k, v)
        for _, at, row, n in runs:
            for h in range(kv_heads if n else 0):
                want[at, h] = extremes(cache.k()[at, h, :row + n].double(), torch.bfloat16).to(want.dtype)
        assert torch.equal(cache.summaries[0], want)                  # pages without new rows are left alone
        q = normal(turn, tokens, 8, dim)
        which = step.sequences.tolist(), step.positions.tolist()
        chosen = cache.select(q, 4, sinks=1, recent=1, sequences=step.sequences, positions=step.positions)
        live = [i for i, s in enumerate(which[0]) if s >= 0]
        at = torch.tensor(live, dtype=torch.long, device="cuda")
        check_select(cache, q[at], chosen[at], 4, 1, 1, [which[0][i] for i in live], [which[1][i] for i in live])
        assert (chosen[[i for i in range(tokens) if i not in live]] == -1).all()
        out = cache.attention(q, sequences=step.sequences, positions=step.positions, chosen=chosen)
        check_attention(cache, q, out, "f32", *which, chosen.tolist())
    assert cut > 5
