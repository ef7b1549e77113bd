"""Steps of a paged cache's table that are not its last one, and steps of no tokens. Helpers are test_gpu_paged.py's."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from test_gpu_paged import ints, normal, same_bits, shuffled  # noqa: E402
from voxgen_b200 import paged  # noqa: E402
from voxgen_b200.api import VoxGenError  # noqa: E402


def refused(call):
    with pytest.raises(VoxGenError, match="VG_EINVAL"):
        call()


def test_an_older_step_is_refused():
    """Its rows would go into pages that are another sequence's by now."""
    table = shuffled(2, 4, 16, 4)
    cache = paged.PagedCache(table, 1, 64, layers=2, summaries=True)
    k = normal(1, 20, 1, 64)
    first = table.step(ints([20, 0]), 20)
    cache.append(first, k, k)
    second = table.step(ints([0, 20]), 20, keep=ints([0, 0]))       # the same pages, for the other sequence
    assert first.slots.tolist() == second.slots.tolist()
    cache.append(second, 2 * k, 2 * k, layer=0)
    before = cache.data.clone()
    refused(lambda: cache.append(first, k, k, layer=1))
    assert same_bits(cache.data, before)
    cache.append(second, 2 * k, 2 * k, layer=1)                     # every layer's append is of the last step
    with pytest.raises(VoxGenError):
        table.step(ints([1, 1, 1]), 2)                              # a refused call is no step
    cache.append(second, k, k, layer=1)
    third = table.step(ints([1, 1]), 20, into=first)
    assert third is first
    cache.append(first, k, k)
    refused(lambda: cache.append(second, k, k))
    table.reset()
    refused(lambda: cache.append(first, k, k))


def test_arrays_in_hand_and_captured_steps_are_not_asked_for_their_age():
    table = shuffled(2, 8, 16, 4)
    cache = paged.PagedCache(table, 1, 64)
    k = normal(1, 4, 1, 64)
    step = table.step(ints([2, 2]), 4)
    parts = [x.clone() for x in (step.starts, step.slots, step.positions, step.sequences, step.runs)]
    mine = paged.Step.of(table, *parts)
    step = table.step(ints([2, 2]), 4)
    for x, y in zip(parts, (step.starts, step.slots, step.positions, step.sequences, step.runs)):
        x.copy_(y)
    cache.append(mine, k, k)                                        # the last step's, copied into the same arrays
    counts = ints([1, 1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = table.step(counts, 4)
        cache.append(captured, k, k)
    cache.append(step, k, k)                                        # no replay yet: still the last step
    graph.replay()
    cache.append(captured, k, k)                                    # outside of the graph, after its replay
    assert table.rows.tolist() == [5, 5] and captured.positions.tolist()[:2] == [4, 4]


def test_a_reserved_workspace_is_not_outgrown_by_a_smaller_batch():
    """Of 20,000 queries nothing is cut and nothing needs room; of 600 something does."""
    table = shuffled(2, 40, 16, 20)
    cache = paged.PagedCache(table, 1, 64)
    k = normal(1, 300, 1, 64)
    cache.append(table.step(ints([300, 0]), 300), k, k)
    cache.reserve(20000, 8)
    ready = cache._workspace
    q = normal(2, 600, 8, 64)
    sequences = ints([0, 1] * 300)
    want = cache.attention(q, sequences=sequences)
    assert cache._workspace is ready
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attention(q, sequences=sequences)
    graph.replay()
    assert cache._workspace is ready and torch.equal(out, want)


def test_arrays_in_hand_of_no_tokens():
    table = shuffled(2, 10, 16, 5)
    cache = paged.PagedCache(table, 1, 64)
    table.step(ints([30, 20]), 50)
    step = table.step(ints([0, 0]), 0)
    copy = paged.Step.of(table, *(x.clone() for x in (step.starts, step.slots, step.positions, step.sequences, step.runs)))
    none = normal(1, 0, 1, 64)
    before = cache.data.clone()
    cache.append(copy, none, none)
    assert same_bits(cache.data, before)
    assert table.step(ints([0, 0]), 0, keep=ints([17, 0]), into=copy) is copy
    cache.append(copy, none, none)
    assert table.rows.tolist() == [17, 0] and copy.starts.tolist() == [0, 0, 0]
