"""The 4-bit cache's operators in 64 bits (numpy), for the tests: written from their definitions,
apart from the kernels and from the forms that the benchmark compares with."""
from fractions import Fraction

import numpy as np

LARGEST, SMALLEST = 7168.0, 2.0 ** -18


def scales_of(x):
    """The scale of each block of 32 channels of x [..., head_dim], as exact float64 numbers."""
    x = np.nan_to_num(np.asarray(x, np.float64), nan=0.0, posinf=LARGEST, neginf=-LARGEST).clip(-LARGEST, LARGEST)
    b = x.reshape(*x.shape[:-1], -1, 32)
    high, low = b.max(-1), b.min(-1)
    d = np.where(high >= -low, high, low) / -8
    m, e = np.frexp(d)
    d = np.ldexp(np.rint(m * 128), e - 7)   # np.rint: ties to even, as the definition
    return np.where(np.abs(d) < SMALLEST, 0.0, d)


def unpack(data, seqs, kv_heads, head_dim, capacity):
    """K and V values [seqs, kv_heads, capacity, head_dim] of a cache's bytes (from the layout alone)."""
    tiles = -(-capacity // 64)
    raw = np.asarray(data, np.uint8).reshape(seqs, kv_heads, tiles, 72 * head_dim)
    out = []
    for v in (0, 1):
        codes = raw[..., v * 32 * head_dim:(v + 1) * 32 * head_dim].reshape(seqs, kv_heads, tiles * 64, head_dim // 2)
        start = 64 * head_dim + v * 4 * head_dim
        scale = np.ascontiguousarray(raw[..., start:start + 4 * head_dim]).view(np.float16)
        scale = scale.reshape(seqs, kv_heads, tiles * 64, head_dim // 32).astype(np.float64)
        n = np.stack((codes & 15, codes >> 4), -1).reshape(seqs, kv_heads, tiles * 64, head_dim).astype(np.float64) - 8
        with np.errstate(invalid="ignore"):
            out.append((n * np.repeat(scale, 32, -1))[:, :, :capacity])
    return out


def attention(q, k, v, rows, counts=None, scale=None):
    """out [seqs, tokens, heads, head_dim] and, per cache row, the attention it drew
    [seqs, kv_heads, capacity], both float64."""
    q = np.asarray(q, np.float64)
    seqs, tokens, heads, dim = q.shape
    kv_heads = k.shape[1]
    group = heads // kv_heads
    scale = dim ** -0.5 if scale is None else scale
    out = np.zeros_like(q)
    drawn = np.zeros(k.shape[:3])
    for s in range(seqs):
        c = tokens if counts is None else counts[s]
        for t in range(c):
            seen = rows[s] - c + t + 1
            if seen <= 0:
                continue
            for h in range(heads):
                e = k[s, h // group, :seen] @ q[s, t, h] * scale
                p = np.exp(e - e.max())
                p /= p.sum()
                out[s, t, h] = p @ v[s, h // group, :seen]
                drawn[s, h // group, :seen] += p
    return out, drawn


def evict(weights, positions, rows, nxt, budget, recent, sinks):
    """For one sequence and head: the source row of each of the first `budget` rows, or None when nothing goes."""
    if rows <= budget:
        return None

    def rank(r):
        pos, w = int(positions[r]), float(weights[r])
        if pos >= nxt - recent or pos < sinks:
            return (0, 0.0, r)
        return (1, np.inf if w != w else -w, r) if w == w else (2, 0.0, r)

    kept = sorted(range(rows), key=rank)[:budget]
    late = iter(sorted(r for r in kept if r >= budget))
    early = set(r for r in kept if r < budget)
    return [r if r in early else next(late) for r in range(budget)]


def verify(tokens, draft, target, u_accept, u_sample):
    """(accepted, next) of one sequence in exact arithmetic."""
    drafted, vocab = draft.shape
    n = 0
    while n < drafted:
        x = int(tokens[n])
        if not 0 <= x < vocab or not np.float32(u_accept[n]) * np.float32(draft[n, x]) < np.float32(target[n, x]):
            break
        n += 1
    rest = target[n].astype(np.float32)
    if n < drafted:
        less = (target[n] - draft[n]).astype(np.float32)
        if (less > 0).any():
            rest = less
    whole = [int(Fraction(float(min(max(w, 0.0), 1.0))) * 2 ** 38) if w == w else 0 for w in rest]
    point = (int(Fraction(float(u_sample)) * 2 ** 24) * sum(whole)) >> 24
    total = 0
    for i, w in enumerate(whole):
        total += w
        if total > point:
            return n, i
    return n, vocab - 1
