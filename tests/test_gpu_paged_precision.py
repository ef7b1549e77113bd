"""The paged attention's precision for 16-bit queries, where the rounding of an output does not cover that of its weights and
sums: outputs that nearly cancel, against 64 bits. Helpers and the cache's checks are test_gpu_paged.py's."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from test_gpu_paged import TYPES, ints, shuffled  # noqa: E402
from voxgen_b200 import paged  # noqa: E402


def uniform(seed, *shape):
    return torch.rand(*shape, generator=torch.Generator().manual_seed(seed)).double()


def half_step(x, dtype):
    """The most that rounding x to a type may move it."""
    f = torch.finfo(TYPES[dtype])
    return (x.abs() * f.eps / 2).clamp_min(f.smallest_normal * f.eps / 2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_weights_are_held_to_32_bits(kind, dtype):
    """Three rows a sequence whose weighted values cancel to 2^-17 of their size and below, so that an error of a weight
    shows in the output. Scores are exact: one channel of q and K, 8 bits each.

    Bound, in terms of A = sum(p |v|): the weight of row 1 is off by the rounding of its exponent (2^-22 for the range that
    P is held in, times ln 2), the constant's 2^-25 of it and the exponential's 2^-22, and half of A at most is its; P's terms
    leave 2^-24; three products (a term each) cut four numbers aligned to the largest at 2^-24, 2^-22 each. In all
    1.1 * 2^-20; 2^-19 is allowed, and half a step of the output. (P in two bf16 terms is off by up to 2^-17 of row 1's
    part, in one fp16 term by 2^-12.)"""
    n, heads, dim = 64, 8, 64
    t = TYPES[kind]
    a = 1 + (uniform(1, n, heads) * 128).floor() / 128                    # in [1, 2)
    b = (1 + (uniform(2, n) * 128).floor() / 128) / 2
    w = (-a * b[:, None]).exp()                                           # of row 1; rows 0 and 2 have 1
    u = 1 + (uniform(3, n, dim) * 128).floor() / 128
    mine = w[:, torch.arange(dim) % heads]                                # channel c cancels for head c % heads
    v1 = -(u / mine).to(t).double()
    v2 = -(u + mine * v1).to(t).double()
    k, v = torch.zeros(2, n, 3, 1, dim, dtype=torch.float64)
    k[:, 1, 0, 0] = -b
    v[:, 0, 0], v[:, 1, 0], v[:, 2, 0] = u, v1, v2
    table = shuffled(n, n, 16, 1)
    cache = paged.PagedCache(table, 1, dim, dtype=t)
    cache.append(table.step(ints([3] * n), 3 * n), *(x.flatten(0, 1).float().cuda() for x in (k, v)))
    q = torch.zeros(n, heads, dim, dtype=TYPES[dtype])
    q[:, :, 0] = a.to(q.dtype)
    out = cache.attention(q.cuda(), scale=1.0).double().cpu()
    total = 2 + w[:, :, None]
    want = (u[:, None] + w[:, :, None] * v1[:, None] + v2[:, None]) / total
    size = (u[:, None] + w[:, :, None] * v1[:, None].abs() + v2[:, None].abs()) / total
    worst = (((out - want).abs() - half_step(want, dtype)) / size).max()
    assert worst <= 2.0 ** -19, float(worst.log2())


@pytest.mark.parametrize("dtype,kind", [("f16", "f16"), ("bf16", "bf16"), ("bf16", "f16"), ("f16", "bf16"), ("f32", "f16")])
def test_sums_of_long_pieces_have_no_bias(dtype, kind):
    """More segments than are cut, 4 tokens each, over 131072 rows: one warp adds all of them. The second half of the rows
    holds the first half's K and its V with the other sign, so outputs are 0, and sums that are cut towards zero on their way up
    and down again are not.

    Bound, in terms of A = sum(p |v|): a sum is taken afresh after at most 96 products (32 steps of up to three terms), each
    cut at 2^-22 of what that sum has seen, 2^-15.4 A in all; the 256 sums of an output are added with roundings of 2^-24, 2^-16 A;
    weights of equal rows are equal. 2^-14.5 is allowed. (Summed in one, the 16384 products of two terms leave 2^-13.7.)"""
    half, n, heads, dim = 1 << 16, (1 << 14) + 4, 8, 64
    t = TYPES[kind]
    b = (uniform(1, half) * 256).floor() / 256
    u = (1 + uniform(2, half, dim)).to(t).double()
    k = torch.zeros(2 * half, 1, dim, dtype=torch.float64)
    k[:, 0, 0] = torch.cat((b, b))
    v = torch.cat((u, -u))[:, None]
    table = shuffled(1, 2 * half // 256, 256, 2 * half // 256)
    cache = paged.PagedCache(table, 1, dim, dtype=t)
    cache.append(table.step(ints([2 * half]), 2 * half), k.float().cuda(), v.float().cuda())
    a = 1 + torch.arange(heads).double() / heads
    q = torch.zeros(n, heads, dim, dtype=TYPES[dtype])
    q[:, :, 0] = a.to(q.dtype)
    out = cache.attention(q.cuda(), sequences=ints([0] * n), scale=1.0).double().cpu()
    p = (a[:, None] * b).exp()
    size = p @ u / p.sum(1, keepdim=True)
    worst = (out.abs() / size).max()
    assert worst <= 2.0 ** -14.5, float(worst.log2())


def small_cache(kind, rows, heads=1, dim=64, seed=3, hook=None):
    """A cache of sequences of rows[s] normal rows, after ``hook(k, v, start)`` has changed them; K and V as they are held, in 64
    bits (an infinity as the largest number)."""
    t = TYPES[kind]
    table = shuffled(len(rows), sum(-(-r // 16) for r in rows), 16, -(-max(rows) // 16))
    cache = paged.PagedCache(table, heads, dim, dtype=t)
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(sum(rows), heads, dim, generator=g) for _ in "kv")
    starts = [sum(rows[:s]) for s in range(len(rows))]
    hook(k, v, starts)
    cache.append(table.step(ints(list(rows)), sum(rows)), k.cuda(), v.cuda())
    top = torch.finfo(t).max
    held = [x.clamp(-top, top).to(t).double() for x in (k, v)]
    return cache, [[x[a:a + n, 0] for x in held] for a, n in zip(starts, rows)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_values_at_the_largest_number(kind, dtype):
    """Infinities in V, held as the largest number: a mean with some of them in it is finite. Bound: test_gpu_paged.py's for scores
    (S 2^-17) and sums (2^-15) on sum(p |v|) of the output itself, and half a step of it."""
    def hook(k, v, starts):
        for s, places in enumerate(((3, 17, 18, 39), (20, 2000, 2001, 4500))):
            for r in places:
                v[starts[s] + r, 0, 5] = float("inf")
                v[starts[s] + r, 0, 6] = -float("inf")
    cache, held = small_cache(kind, (40, 5000), hook=hook)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(5)).to(TYPES[dtype])
    q[:, 0] = 0
    out = cache.attention(q.cuda()).double().cpu()
    most = torch.finfo(TYPES[dtype]).max
    for s, (k, v) in enumerate(held):
        p = (q[s].double() @ k.T / 8).softmax(1)
        want, size = p @ v, p @ v.abs()
        top = float((q[s].double().abs() @ k.T.abs()).max()) / 8
        near = want.abs() < most
        assert (out[s][want > most * 1.01] == float("inf")).all() and (out[s][want < -most * 1.01] == -float("inf")).all()
        good = (out[s] - want).abs() <= half_step(want, dtype) + (top * 2.0 ** -17 + 2.0 ** -15) * size
        assert (good | ~near).all()
        assert near.all() or (kind, dtype) == ("bf16", "f16")


@pytest.mark.parametrize("dtype", TYPES)
def test_keys_at_the_largest_number(dtype):
    """Infinities in K of a bf16 cache, held as the largest number: rows with it take all of the weight, or none. Ties (the rest of
    a score is far below the largest number's last bit) are means of V: bound 2^-20 of it, and half a step."""
    def hook(k, v, starts):
        for s, places in enumerate(((3, 17, 30), (20, 2000, 4500))):
            for r, x in zip(places, (float("inf"), float("inf"), -float("inf"))):
                k[starts[s] + r, 0, 5] = x
    cache, held = small_cache("bf16", (40, 5000), hook=hook)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(5)).to(TYPES[dtype])
    q[:, 0, 5], q[:, 1, 5], q[:, 2, 5], q[:, 3, 5] = 1.5, -1.5, 0.0, 100.0
    out = cache.attention(q.cuda()).double().cpu()
    for s, (k, v) in enumerate(held):
        e = q[s].double() @ k.T / 8
        p = (e - e.amax(1, keepdim=True)).exp()
        want = p @ v / p.sum(1, keepdim=True)
        # where its channel counts for nothing, such a row is like any other
        slack = torch.full((4, 64), 2.0 ** -20 * float(v.abs().max()), dtype=torch.float64)
        top = float((q[s, 2].double().abs() @ k.abs().T).max()) / 8
        slack[2] = (top * 2.0 ** -17 + 2.0 ** -15) * (p[2] @ v.abs()) / p[2].sum()
        assert ((out[s] - want).abs() <= half_step(want, dtype) + slack).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("power", [-100, -110])
def test_values_near_the_smallest_number(power, dtype):
    """Weights are held scaled, so products of a bf16 cache's smallest values are subnormal: each of the up to three products of a
    block, and each of 48 joined warps and pieces, is off by 2^-149 at most, which the weights' sum (2^-20 at least) makes 2^-129 in
    the output: 2^-120 for the 160 of them here. To it test_gpu_paged.py's bound for scores and sums."""
    def hook(k, v, starts):
        v.copy_((1 + v.abs()) * 2.0 ** power)
    cache, held = small_cache("bf16", (40, 100), hook=hook)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(5)).to(TYPES[dtype])
    out = cache.attention(q.cuda()).double().cpu()
    for s, (k, v) in enumerate(held):
        want = (q[s].double() @ k.T / 8).softmax(1) @ v
        top = float((q[s].double().abs() @ k.T.abs()).max()) / 8
        bound = half_step(want, dtype) + (top * 2.0 ** -17 + 2.0 ** -15) * want + 2.0 ** -120
        assert ((out[s] - want).abs() <= bound).all()
