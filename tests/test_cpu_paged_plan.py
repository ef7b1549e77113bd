"""The paged attention's plan in 32-bit arithmetic on the CPU: however long the contexts that the entry point takes, pieces have
blocks, and those of cut segments no more partial results than the workspace has room for."""
import numpy as np
import pytest

from voxgen_b200._build import CSRC

TICKETS, MOST, WHOLE, UNCUT, M = 1 << 14, 1 << 26, 48, 0xFFFFFFFF, 0xFFFFFFFF
WEIGHT = (4, 6, 10)            # of a block of a segment of 1, 2 or 4 tiles
f32 = np.float32


def over(a, b):
    return (min(int(f32(a) * (f32(1) + f32(2.0 ** -20)) / f32(b)), M) + 1) & M     # the GPU's conversion saturates


def size_of(tiles, size):
    if size == UNCUT:
        return MOST
    return min(size, MOST) if tiles == 0 else ((2 * size + 2) & M) // 3 if tiles == 1 else ((2 * size + 4) & M) // 5


def parts(blocks, tiles, size):
    """Pieces of a segment; raises where the kernel's loop would not end."""
    if blocks * WEIGHT[tiles] <= WHOLE * 4:
        return 1
    each = size_of(tiles, size)
    if each == 0:
        raise AssertionError("pieces of no blocks")
    return -(-blocks // each)


def target_of(segments, ctas):
    return ctas * min(max((segments * 4 + ctas * 3 - 1) // (ctas * 3), 1), 4)


def plan(entries, lanes, ctas, warps):
    """entries: (blocks, log2 tiles) of each segment's lead. Size, pieces, the partial results of cut segments, and the target."""
    total = sum((b * WEIGHT[t] + 3) // 4 for b, t in entries) * lanes
    assert total < 1 << 31
    segments = len(entries) * lanes
    target = target_of(segments, ctas)
    least = max(warps, over(total, target))
    more = max(least, over(total, target - segments)) - least if target > segments else 0
    for k in range(8):
        size = (least + (more if k == 7 else (more * k * k & M) // 49)) & M
        n = [parts(b, t, size) for b, t in entries]
        if sum(n) * lanes <= target:
            break
    return size, sum(n) * lanes, sum(x for x in n if x > 1) * lanes, target


def longest(tiles, lanes):
    """Blocks of the longest context that the entry point takes: it counts every query's, and a segment of T tiles as T."""
    return min(MOST, ((1 << 31) - 1) // (lanes * int(sum(2 ** t for t in tiles))))


def cases():
    rng = np.random.default_rng(1)
    # one free piece a call: the largest sizes that a plan can ask for
    for tiles, lanes in (([0] * 1182 + [1], 1), ([0] * 1183, 1), ([1] * 591, 1), ([0] * 590 + [1], 2), ([2] * 1183, 1), ([0] * 33, 1)):
        yield [(longest(tiles, lanes), t) for t in tiles], lanes
    for _ in range(400):
        lanes = int(rng.choice([1, 1, 2, 3, 8]))
        count = int(2 ** rng.uniform(0, np.log2(16384 // lanes)))
        tiles = rng.choice([0, 0, 1, 2], count)
        high = longest(tiles, lanes)
        low = 2 ** rng.uniform(0, np.log2(high))
        yield [(max(1, int(b)), int(t)) for b, t in zip(rng.uniform(low, high, count), tiles)], lanes


def test_pieces_stay_within_the_workspace():
    for entries, lanes in cases():
        segments = len(entries) * lanes
        warps = 12 if segments < 444 else 4
        size, pieces, cut, target = plan(entries, lanes, 148 if warps == 12 else 296, warps)
        assert cut <= 2 * target, (len(entries), lanes, size, pieces, cut, target)


@pytest.mark.parametrize("text", [
    "constexpr uint32_t kPagedWhole = 48;", "constexpr uint32_t kPagedTickets = 1u << 14;", "constexpr uint32_t kPagedMost = 1u << 26;",
    "return (entry & 3) == 0 ? min(size, kPagedMost) : (entry & 3) == 1 ? (2 * size + 2) / 3 : (2 * size + 4) / 5;",
    "return (entry & 3) == 0 ? 4 : (entry & 3) == 1 ? 6 : 10;", "size = least + (k == 7 ? more : more * k * k / 49);",
    "return segments > kPagedTickets ? 0 : 2 * paged_target((uint32_t)segments, ctas);"])
def test_the_kernel_computes_what_is_computed_here(text):
    assert text in (CSRC / "paged_attention.cuh").read_text()
