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
