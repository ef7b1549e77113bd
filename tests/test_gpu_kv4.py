"""The 4-bit cache on the GPU (append, read, attention, evict) and draft verification, through
``voxgen_b200.kv4``, against 64-bit references (kv4_reference.py).

Tolerances. An attention output is a mean of cache values weighted by exp(score). Operands carry at
least 22 bits and sums are fp32, so a score of terms whose magnitudes add up to S is off by at most
about S * 2^-20, a weight by that relative to itself, and an output by twice that times the largest
value: (S * 2^-19 + 2^-17) * max|v|. With 16-bit queries the weights may be rounded to 11 bits, and the
output is: 2^-10 (fp16) or 2^-8 (bf16) of max|v| more.
"""
import numpy as np
import pytest

import kv4_reference as R

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from voxgen_b200 import kv4  # noqa: E402
from voxgen_b200.api import VoxGenError  # noqa: E402

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def normal(seed, *shape, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).cuda()


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def filled(seed, rows, kv_heads, dim, capacity, track=False, garbage=True):
    """A cache whose sequences hold rows[s] normal rows, and bytes that would read as NaN past them."""
    cache = kv4.Kv4Cache(len(rows), kv_heads, dim, capacity, track=track)
    cache.data.fill_(0xFF if garbage else 0)
    if max(rows):
        k, v = (normal(seed + i, len(rows), max(rows), kv_heads, dim) for i in (0, 1))
        cache.append(k, v, counts=ints(*rows))
    assert cache.rows().tolist() == list(rows) and not any(cache.status())
    return cache


def held(cache):
    return R.unpack(cache.data.cpu().numpy(), cache.seqs, cache.kv_heads, cache.head_dim, cache.capacity)


def tolerance(q, k, v, rows, dtype, scale=None):
    n = max(max(rows), 1)
    k, v = (np.stack([np.pad(x[s, :, :r], ((0, 0), (0, n - r), (0, 0))) for s, r in enumerate(rows)]) for x in (k, v))
    group = q.shape[2] // k.shape[1]
    s = np.einsum("sthd,shnd->sthn", np.abs(q), np.repeat(np.abs(k), group, 1)).max()
    s *= q.shape[3] ** -0.5 if scale is None else scale
    extra = {"f32": 0, "f16": 2.0 ** -10, "bf16": 2.0 ** -8}[dtype]
    return s, (s * 2.0 ** -19 + 2.0 ** -17 + extra) * np.abs(v).max()


# ---------------------------------------------------------------------------------------------
# append and read
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("seqs,tokens,kv_heads,dim,capacity", [
    (1, 1, 1, 64, 1), (3, 1, 2, 128, 65), (2, 63, 3, 64, 64), (1, 200, 8, 128, 300), (5, 130, 1, 128, 131)])
def test_append_holds_the_nearest_codes(dtype, seqs, tokens, kv_heads, dim, capacity):
    k, v = (normal(i, seqs, tokens, kv_heads, dim, dtype=TYPES[dtype]) * (3.0 ** i) for i in (0, 1))
    cache = kv4.Kv4Cache(seqs, kv_heads, dim, capacity)
    cache.append(k, v)
    got = cache.read(tokens, dtype=torch.float32)
    raw = held(cache)
    for x, y, bits in zip((k, v), got, raw):
        x = x.double().cpu().numpy()
        y = y.double().cpu().numpy()
        np.testing.assert_array_equal(y, bits[:, :, :tokens].transpose(0, 2, 1, 3))   # read is exact
        d = np.repeat(R.scales_of(x), 32, -1)
        n = np.divide(y, d, out=np.zeros_like(y), where=d != 0)
        np.testing.assert_array_equal(n, np.rint(n))     # every value is a whole multiple of the exact scale,
        assert n.min() >= -8 and n.max() <= 7            # within the codes' range,
        near = np.clip(x / np.where(d == 0, 1, d), -8, 7)
        assert (np.abs(n - near) <= 0.5 + 8 * 2.0 ** -22).all()   # and the nearest one, but for fp32's rounding of x/d
    assert cache.rows().tolist() == [tokens] * seqs
    assert cache.state[:, 1].tolist() == [tokens] * seqs and not any(cache.status())
    assert not cache.state[:, 3].any()


def test_append_special_values():
    """Zero and tiny blocks, ties between +b and -b, infinities, NaN, values past the range."""
    x = torch.zeros(1, 8, 1, 64)
    x[0, 1, 0, :32] = 2.0 ** -17           # below the smallest scale: held as zeros
    x[0, 2, 0, :2] = torch.tensor([3.0, -3.0])
    x[0, 3, 0, :2] = torch.tensor([-8.0, 1.0])
    x[0, 4, 0, :2] = torch.tensor([float("inf"), 1.0])
    x[0, 5, 0, :2] = torch.tensor([float("nan"), 1.0])
    x[0, 6, 0, :2] = torch.tensor([-1e30, 7168.0])
    x[0, 7, 0, :2] = torch.tensor([2.0 ** -14, 2.0 ** -15])
    cache = kv4.Kv4Cache(1, 1, 64, 64)
    cache.append(x[:, :4].cuda(), x[:, :4].cuda())
    assert cache.status() == [0]
    cache.append(x[:, 4:].cuda(), x[:, 4:].cuda())
    assert cache.status() == [kv4.STATUS_NONFINITE]
    k, v = cache.read(8, dtype=torch.float32)
    assert torch.equal(k, v)
    y = k[0, :, 0].cpu()
    assert not y[:2].any() and not y[:, 32:].any()
    assert y[2, :2].tolist() == [3.0, -2.625]            # +3 is the extreme (code -8 of -3/8), -3 is 7 steps
    assert y[3, :2].tolist() == [-8.0, 1.0]
    assert y[4, :2].tolist() == [7168.0, 0.0]
    assert y[5, :2].tolist() == [0.0, 1.0]
    assert y[6, :2].tolist() == [-6272.0, 7168.0]        # 7 steps of 896 the other way
    assert y[7, :2].tolist() == [2.0 ** -14, 2.0 ** -15]
    assert torch.isfinite(y).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_append_reports_what_it_clamps(dtype, dim):
    """A finite value past 7168 in K or V, at either end of a row, sets its own sequence's status; 7168 does not."""
    step = {"f32": 0.0625, "f16": 4.0, "bf16": 32.0}[dtype]       # 7168 + step is the type's next number, or near it
    for value, bit in ((7168.0, 0), (7168.0 + step, kv4.STATUS_NONFINITE), (-7168.0 - step, kv4.STATUS_NONFINITE),
                       (65024.0, kv4.STATUS_NONFINITE)):
        for place in (0, dim - 1):
            x = normal(3, 2, 5, 2, dim, dtype=TYPES[dtype])
            y = x.clone()
            x[1, 3, 1, place] = value
            for k, v in ((x, y), (y, x)):
                cache = kv4.Kv4Cache(2, 2, dim, 64)
                cache.append(k, v)
                assert cache.status() == [0, bit], (value, place)


@pytest.mark.parametrize("dtype", TYPES)
def test_append_and_read_of_strided_rows(dtype):
    """K and V as parts of a fused projection, on and off 16-byte boundaries, and transposed heads."""
    fused = normal(5, 2, 40, 1 + 2 * 3 * 64, dtype=TYPES[dtype])
    for shift in (0, 1):
        k, v = (fused[:, :, shift + i * 192:shift + (i + 1) * 192].unflatten(2, (3, 64)) for i in (0, 1))
        a, b, c = (kv4.Kv4Cache(2, 3, 64, 64) for _ in range(3))
        a.append(k, v)
        b.append(k.contiguous(), v.contiguous())
        c.append(k.transpose(1, 2).contiguous().transpose(1, 2), v)
        for x, y, z in zip(a.read(40), b.read(40), c.read(40)):
            assert torch.equal(x, y) and torch.equal(x, z)


def test_append_at_and_counts():
    cache = filled(3, [10, 64, 0], 2, 64, 80, track=True)
    before = cache.read(80)
    k, v = (normal(i, 3, 5, 2, 64) for i in (7, 8))
    cache.append(k, v, at=ints(8, 64, 0), counts=ints(5, 0, 3))
    assert cache.rows().tolist() == [13, 64, 3]
    assert cache.state[:, 1].tolist() == [13, 64, 3]
    after = cache.read(80)
    other = kv4.Kv4Cache(3, 2, 64, 80)
    other.append(k, v)
    new = other.read(5)
    for b, a, n in zip(before, after, new):
        assert torch.equal(a[0, :8], b[0, :8]) and torch.equal(a[0, 8:13], n[0]) and torch.equal(a[2, :3], n[2, :3])
        assert torch.equal(a[1], b[1]) and not a[2, 3:].any() and not a[0, 13:].any()
    assert cache.positions[0, 1, :13].tolist() == list(range(13)) and not cache.weights.any()
    got = cache.read(4, first=ints(9, -2, 200))
    assert torch.equal(got[0][0], after[0][0, 9:13])
    assert not got[0][1, :2].any() and torch.equal(got[0][1, 2:], after[0][1, :2])   # rows before 0 read as 0
    assert not got[0][2].any()


@pytest.mark.parametrize("at,counts,bit", [
    ([61, 10], [4, 4], kv4.STATUS_FULL), ([65, 10], [4, 4], kv4.STATUS_BAD_ROW), ([-1, 10], [4, 4], kv4.STATUS_BAD_ROW),
    ([3, 10], [5, 4], kv4.STATUS_BAD_ROW), ([3, 10], [-1, 4], kv4.STATUS_BAD_ROW)])
def test_append_that_does_not_fit_leaves_its_sequence(at, counts, bit):
    cache = filled(4, [64, 40], 1, 128, 64)
    before = [x.clone() for x in cache.read(64)]
    k, v = (normal(i, 2, 4, 1, 128) for i in (1, 2))
    cache.append(k, v, at=ints(*at), counts=ints(*counts))
    assert cache.rows().tolist() == [64, 14] and cache.status() == [bit, 0]
    for b, a in zip(before, cache.read(64)):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1, :10], b[1, :10])


def test_rows_past_4_gigabytes():
    """The last sequence of a cache whose bytes need more than 32 bits to address."""
    seqs, capacity = 130, 131072
    cache = kv4.Kv4Cache(seqs, 2, 128, capacity)
    assert cache.data.numel() > 1 << 32
    last = seqs - 1
    k, v = (normal(i, 1, 70, 2, 128) for i in (1, 2))
    small = kv4.Kv4Cache(1, 2, 128, 128)
    small.append(k, v)
    want = small.read(70)
    # rows [capacity - 70, capacity) of the last sequence
    cache.state[last, :2] = capacity - 70
    wide = [x.expand(seqs, 70, 2, 128) for x in (k, v)]
    counts = torch.zeros(seqs, dtype=torch.int32, device="cuda")
    counts[last] = 70
    cache.append(*wide, counts=counts)
    assert cache.rows()[last].item() == capacity and cache.status()[last] == 0
    first = torch.zeros(seqs, dtype=torch.int32, device="cuda")
    first[last] = capacity - 70
    got = cache.read(70, first=first)
    for a, b in zip(got, want):
        assert torch.equal(a[last], b[0])
    # attention over that sequence alone: every other row has a value of 0 and a score of 0
    view = cache.data.view(seqs, -1)
    view[last, :view.shape[1] // 2].zero_()
    view[last, view.shape[1] // 2:].zero_()
    cache.state[last, :2] = capacity - 70
    cache.append(*wide, counts=counts)
    q = normal(9, 1, 1, 16, 128).expand(seqs, 1, 16, 128).contiguous()
    cache.state[:last].zero_()
    out = cache.attention(q)[last, 0].double().cpu()
    e = torch.einsum("hd,nhd->hn", q[0, 0].double().cpu(), want[0][0].double().cpu().repeat_interleave(8, 1)) / 128 ** 0.5
    p = e.exp()
    p = p / (p.sum(-1, keepdim=True) + capacity - 70)
    ref = torch.einsum("hn,nhd->hd", p, want[1][0].double().cpu().repeat_interleave(8, 1))
    assert (out - ref).abs().max() <= (40 * 2.0 ** -19 + 2.0 ** -17) * want[1].abs().max().item()
    assert not cache.attention(q)[:last].any()


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
SHAPES = [
    # rows of each sequence, tokens, heads, KV heads, head_dim
    ([1], 1, 16, 2, 64), ([63, 64, 65], 1, 16, 2, 128), ([1000, 3, 517, 128, 129], 1, 8, 2, 128),
    ([700], 1, 12, 2, 64), ([333, 40], 1, 8, 8, 128), ([257, 300], 1, 32, 1, 64), ([2100], 1, 2, 2, 128),
    ([300, 17, 64], 2, 16, 2, 128), ([130, 500], 5, 16, 2, 128), ([90, 700], 3, 6, 3, 64), ([400], 16, 8, 1, 128),
    ([600, 33], 17, 16, 2, 128), ([300], 33, 12, 2, 64), ([129, 450], 100, 4, 2, 128), ([300], 300, 2, 1, 128),
    ([511], 257, 8, 2, 64),
    # many segments, whole or cut; one long sequence among short ones; pieces of one segment on every SM
    ([5000] + [3] * 59, 1, 4, 2, 64), ([33] * 70 + [900], 1, 8, 8, 64), ([20000], 1, 1, 1, 64), ([20000], 40, 1, 1, 64),
    # blocks of 256 query rows (16-bit), the last of them with few; units dealt out over many short segments
    ([310, 350, 300, 333, 420, 301], 300, 8, 8, 64), ([60, 200, 41] * 10, 40, 8, 8, 64), ([700, 650], 640, 12, 2, 128),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,tokens,heads,kv_heads,dim", SHAPES)
def test_attention(dtype, rows, tokens, heads, kv_heads, dim):
    cache = filled(len(rows) + tokens, rows, kv_heads, dim, max(rows) + 3)
    q = (normal(77, len(rows), tokens, heads, dim) * 1.5).to(TYPES[dtype])
    out = cache.attention(q)
    assert out.dtype == q.dtype
    again = cache.attention(q)
    assert torch.equal(out, again)   # sums have a fixed order
    k, v = held(cache)
    qn = q.double().cpu().numpy()
    want, _ = R.attention(qn, k, v, rows)
    _, tol = tolerance(qn, k, v, rows, dtype)
    assert np.abs(out.double().cpu().numpy() - want).max() <= tol


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,tokens,heads,kv_heads,dim", [
    # cut into pieces, about two a CTA; the last block has 128 query rows
    ([2048], 2000, 16, 2, 64),
    # dealt out unit by unit, several segments a CTA
    ([512, 600, 515, 700, 640, 512, 777, 530], 512, 16, 2, 64), ([530, 400, 777], 400, 24, 2, 128)])
def test_prompts_whose_blocks_follow_one_another(dtype, rows, tokens, heads, kv_heads, dim):
    """256 query rows at a time, more blocks than SMs: a CTA's results leave while the next block's cache rows
    are being unpacked."""
    cache = filled(len(rows) + tokens, rows, kv_heads, dim, max(rows) + 3)
    q = (normal(78, len(rows), tokens, heads, dim) * 1.5).to(TYPES[dtype])
    out = cache.attention(q)
    assert torch.equal(out, cache.attention(q))
    k, v = held(cache)
    qn = q.double().cpu().numpy()
    want, _ = R.attention(qn, k, v, rows)
    _, tol = tolerance(qn, k, v, rows, dtype)
    assert np.abs(out.double().cpu().numpy() - want).max() <= tol


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,tokens,counts", [
    ([0, 5, 3, 64, 200], 1, None), ([2, 0, 70], 5, None), ([10, 10, 90, 0], 6, [0, 3, 6, 2]), ([20, 150], 64, [64, 1]),
    ([0, 0], 40, [40, 0])])
def test_queries_that_see_nothing_give_zeros(dtype, rows, tokens, counts):
    """Empty sequences, tokens before the first row, tokens past a sequence's count."""
    cache = filled(11, rows, 2, 128, 256, track=True)
    cache.weights.fill_(0.5)
    q = normal(5, len(rows), tokens, 16, 128, dtype=TYPES[dtype])
    out = torch.full_like(q, float("nan"))
    cache.attention(q, counts=None if counts is None else ints(*counts), out=out)
    k, v = held(cache)
    qn = q.double().cpu().numpy()
    want, drawn = R.attention(qn, k, v, rows, counts)
    s, tol = tolerance(qn, k, v, rows, dtype)
    got = out.double().cpu().numpy()
    assert np.abs(got - want).max() <= tol
    empty = np.abs(want).max((2, 3)) == 0
    assert not got[empty].any()
    assert np.abs(cache.weights.cpu().numpy() - 0.5 - drawn).max() <= (s * 2.0 ** -19 + 2.0 ** -20) * drawn.max() + 2.0 ** -22


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,tokens,heads,kv_heads,dim", [
    ([1, 130, 700], 1, 16, 2, 128), ([500, 77], 5, 16, 2, 128), ([300], 40, 12, 2, 64), ([260], 200, 4, 4, 128)])
def test_tracked_attention(dtype, rows, tokens, heads, kv_heads, dim):
    cache = filled(21, rows, kv_heads, dim, max(rows) + 1, track=True)
    cache.weights.fill_(0.25)
    q = normal(6, len(rows), tokens, heads, dim, dtype=TYPES[dtype]) * 2
    plain = cache.attention(q, track=False)
    assert (cache.weights == 0.25).all()
    assert torch.equal(cache.attention(q), plain)
    first = cache.weights.clone()
    cache.weights.fill_(0.25)
    cache.attention(q)
    assert torch.equal(cache.weights, first)
    k, v = held(cache)
    qn = q.double().cpu().numpy()
    _, drawn = R.attention(qn, k, v, rows)
    s, _ = tolerance(qn, k, v, rows, dtype)
    got = first.double().cpu().numpy() - 0.25
    assert (np.abs(got - drawn) <= (s * 2.0 ** -19 + 2.0 ** -18) * drawn + 2.0 ** -23 * (drawn + 1)).all()
    for i, n in enumerate(rows):
        assert (first[i, :, n:] == 0.25).all()   # rows that are not held


@pytest.mark.parametrize("tokens", [1, 4, 40])
@pytest.mark.parametrize("dtype", TYPES)
def test_queries_of_extreme_values(dtype, tokens):
    """A NaN or an infinity reaches its own head and token only; zeros and large magnitudes are exact cases."""
    cache = filled(31, [150], 2, 128, 150)
    q = normal(8, 1, tokens, 16, 128, dtype=TYPES[dtype])
    q[0, 0, 3, 5] = float("nan")
    q[0, 0, 9, 1] = float("inf")
    q[0, 0, 4] = 0
    q[0, 0, 5] *= 2000       # scores in the thousands: one row takes all
    q[0, 0, 6] *= 2.0 ** -14   # scores near 0
    out = cache.attention(q).double().cpu().numpy()
    assert np.isnan(out[0, 0, 3]).all() and np.isnan(out[0, 0, 9]).all()
    k, v = held(cache)
    clean = q.clone()
    clean[0, 0, 3] = clean[0, 0, 9] = 0
    qn = clean.double().cpu().numpy()
    want, _ = R.attention(qn, k, v, [150])
    _, tol = tolerance(qn[:, :, [h for h in range(16) if h != 5]][:, :, :14], k, v, [150], dtype)
    keep = np.ones(out.shape[:3], bool)
    keep[0, 0, [3, 5, 9]] = False
    assert np.abs(out - want)[keep].max() <= tol
    # the head of large scores: its largest score leads by far more than the scores are off by
    order = np.sort(k[0, 0] @ qn[0, 0, 5] * 128 ** -0.5)
    assert order[-1] - order[-2] > 40
    best = np.argmax(k[0, 0] @ qn[0, 0, 5])
    assert np.abs(out[0, 0, 5] - v[0, 0, best]).max() <= (2.0 ** -17 + 2.0 ** -8) * np.abs(v).max()


@pytest.mark.parametrize("rows,tokens,counts", [([1, 700], 1, None), ([5, 700], 5, [5, 3]), ([6000], 2, None), ([40, 900], 40, None),
                                                ([900], 600, [500])])
@pytest.mark.parametrize("dtype", TYPES)
def test_scores_that_are_all_minus_infinity(dtype, rows, tokens, counts):
    """An infinite query whose every score is -infinity has no softmax: NaN, and not the zeros of a query that sees no
    row. Other heads and tokens, and those past the count, are as they would be."""
    cache = kv4.Kv4Cache(len(rows), 2, 64, max(rows), track=True)
    k, v = (normal(i, len(rows), max(rows), 2, 64) for i in (1, 2))
    k[..., 5] = k[..., 5].abs() + 0.5
    cache.append(k, v, counts=ints(*rows))
    q = normal(3, len(rows), tokens, 16, 64, dtype=TYPES[dtype])
    q[:, 0, 3, 5] = q[:, -1, 9, 5] = -float("inf")
    clean = q.clone()
    clean[:, 0, 3] = clean[:, -1, 9] = 0
    limits = None if counts is None else ints(*counts)
    out, want = cache.attention(q, counts=limits), cache.attention(clean, counts=limits, track=False)
    for s, n in enumerate(rows):
        c = tokens if counts is None else counts[s]
        for t, h in ((0, 3), (tokens - 1, 9)):
            sees = t < c and n - c + t + 1 > 0
            assert out[s, t, h].isnan().all() if sees else not out[s, t, h].any()
            out[s, t, h] = want[s, t, h] = 0
        assert cache.weights[s, 0, 0].isnan() and not cache.weights[s, :, n:].any()
    assert torch.equal(out, want)


@pytest.mark.parametrize("tokens", [1, 4, 40, 300])
@pytest.mark.parametrize("dtype", TYPES)
def test_scores_past_2_to_the_24(dtype, tokens):
    """Scores of 2^25 to 2^40, where fp32 has no fractions left: a row that leads by more than the scores are off by
    takes all, and every output stays a mean of values."""
    n, dim = 400, 128
    for size, scale in ((1e4, 1.0), (1e4, 40.0), (-1e4, 1.0)) if dtype == "f16" else ((1e6, 0.1), (1e7, 1.0), (-1e6, 1.0)):
        cache = kv4.Kv4Cache(1, 2, dim, n, track=True)
        k, v = normal(1, 1, n, 2, dim) * 1000, normal(2, 1, n, 2, dim)
        if size < 0:
            k, size = k.abs(), -size   # one sign: no score is near 0
        cache.append(k, v)
        q = normal(3, 1, tokens, 16, dim, dtype=torch.float32)
        if (k > 0).all():
            q = -q.abs()
        q = (q * size).to(TYPES[dtype])
        out = cache.attention(q, scale=scale).double().cpu().numpy()[0]
        assert np.isfinite(out).all()
        hk, hv = (x[0] for x in held(cache))
        qn = q[0].double().cpu().numpy()
        top = np.abs(hv).max()
        assert np.abs(out).max() <= top * (1 + 2.0 ** -7)
        off = scale * 2.0 ** -19 * np.einsum("thd,hnd->thn", np.abs(qn), np.repeat(np.abs(hk), 8, 0)).max()
        score = scale * np.einsum("thd,hnd->thn", qn, np.repeat(hk, 8, 0))
        seen = n - tokens + 1 + np.arange(tokens)
        score[np.arange(n) >= np.broadcast_to(seen[:, None, None], score.shape)] = -np.inf
        order = np.sort(score, -1)
        clear = order[..., -1] - order[..., -2] > 2 * off + 40
        assert clear.mean() > 0.9
        t, h = np.nonzero(clear)
        best = hv[h // 8, score.argmax(-1)[t, h]]
        extra = {"f32": 2.0 ** -17, "f16": 2.0 ** -10, "bf16": 2.0 ** -8}[dtype]
        assert np.abs(out[t, h] - best).max() <= extra * top
        drawn = cache.weights.cpu().numpy()
        assert (drawn >= 0).all() and drawn.max() <= 8 * tokens


def test_one_row_takes_all_and_the_rest_still_counts():
    """One row of weight 1 against 30000 of weight 2^-20 each: the small ones add up to 3% of the output."""
    n = 30001
    cache = kv4.Kv4Cache(1, 1, 64, n)
    k, v = torch.zeros(1, n, 1, 64), torch.zeros(1, n, 1, 64)
    k[0, 777, 0, 0] = 8.0
    v[0, :, 0, 1] = 1.0
    v[0, 777, 0, 1] = 0.0
    cache.append(k.cuda(), v.cuda())
    for dtype in TYPES.values():
        q = torch.zeros(1, 1, 2, 64, dtype=dtype, device="cuda")
        q[..., 0] = 20 * 0.6931471805599453 / 8 * 8
        out = cache.attention(q)[0, 0].double().cpu()
        x = q[0, 0, 0, 0].double().item()
        small = np.exp(-x * 8 / 8)
        want = 30000 * small / (1 + 30000 * small)
        tol = {torch.float32: 2.0 ** -16, torch.float16: 2.0 ** -9, torch.bfloat16: 2.0 ** -7}[dtype]
        assert (out[:, 1] - want).abs().max() <= tol * want


@pytest.mark.parametrize("tokens", [1, 4, 40])
def test_strided_queries_scale_and_out(tokens):
    cache = filled(41, [200, 90], 2, 128, 256)
    fused = normal(9, 2, tokens, 4 + 16 * 128)
    q = fused[:, :, 1:1 + 16 * 128].unflatten(2, (16, 128))
    assert not q.is_contiguous()
    out = torch.empty(2, tokens, 16, 128, device="cuda")
    assert cache.attention(q, scale=0.03, out=out) is out
    assert torch.equal(out, cache.attention(q.contiguous(), scale=0.03))
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(out, cache.attention(turned, scale=0.03))
    k, v = held(cache)
    qn = q.double().cpu().numpy()
    want, _ = R.attention(qn, k, v, [200, 90], scale=0.03)
    _, tol = tolerance(qn, k, v, [200, 90], "f32", 0.03)
    assert np.abs(out.double().cpu().numpy() - want).max() <= tol


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,tokens", [([5000, 90], 1), ([3000], 2), ([900, 700], 40), ([2000], 600)])
def test_queries_may_be_overwritten(dtype, rows, tokens):
    """out = q where nothing is tracked, with segments cut among CTAs; refused where something is."""
    cache = filled(43, rows, 2, 64, max(rows), track=True)
    q = normal(9, len(rows), tokens, 8, 64, dtype=TYPES[dtype])
    want = cache.attention(q, track=False)
    with pytest.raises(VoxGenError, match="out cannot be q"):
        cache.attention(q, out=q)
    assert torch.equal(cache.attention(q, track=False, out=q), want) and not cache.weights.any()


@pytest.mark.parametrize("tokens", [1, 4, 40])
def test_other_streams_and_graphs(tokens):
    """The calls run on the stream they are given, and a captured loop replays from the device's state."""
    rows = [300, 70]
    k, v = (normal(i, 2, tokens, 2, 128) for i in (1, 2))
    q = normal(3, 2, tokens, 16, 128)
    want = filled(51, rows, 2, 128, 512, track=True)
    got = filled(51, rows, 2, 128, 512, track=True)
    for _ in range(3):
        want.append(k, v)
        reference = want.attention(q)
    got.attention(q, track=False)        # the workspace exists before the capture
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got.append(k, v)
        got.attention(q)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(q)
    with torch.cuda.graph(graph):
        got.append(k, v)
        got.attention(q, out=out)
    for _ in range(2):
        graph.replay()
    assert torch.equal(out, reference) and torch.equal(got.weights, want.weights)
    assert torch.equal(got.state, want.state)


def test_a_graph_replays_after_its_workspace_was_outgrown():
    """A decode step is captured, then a prompt needs a larger workspace: the graph's stays its own. Buffers of the old
    one's size, allocated since, are not written to, and nothing that they hold is read."""
    q, prompt = normal(1, 2, 1, 16, 128), normal(2, 2, 64, 16, 128)
    cache = filled(55, [900, 700], 2, 128, 1024, track=True)
    cache.reserve(16, 1)
    size = cache._workspace.numel()
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(q)
    with torch.cuda.graph(graph):
        cache.attention(q, out=out)
    cache.weights.zero_()
    want = filled(55, [900, 700], 2, 128, 1024, track=True)
    for _ in range(2):
        reference = want.attention(q)
        cache.attention(prompt, track=False)
        fillers = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(8)]
        out.fill_(float("nan"))
        graph.replay()
        assert torch.equal(out, reference) and torch.equal(cache.weights, want.weights)
        assert all((x == 255).all() for x in fillers)


@pytest.mark.parametrize("tokens", [1, 64])
def test_a_first_call_in_a_capture(tokens):
    """Nothing was reserved: the calls of the graph, and those outside it before its first replay, find zeroed
    workspaces all the same."""
    q = normal(1, 2, tokens, 16, 128)
    cache = filled(56, [900, 700], 2, 128, 1024)
    reference = filled(56, [900, 700], 2, 128, 1024).attention(q)
    dirty = torch.full((64 << 20,), 255, dtype=torch.uint8, device="cuda")   # what an allocation may find
    torch.cuda.synchronize()
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(q)
    with torch.cuda.graph(graph):
        cache.attention(q, out=out)
        cache.attention(q, out=out)
        with pytest.raises(VoxGenError, match="captured"):
            cache.reserve(16, 128)
    del dirty
    assert torch.equal(cache.attention(q), reference)
    for _ in range(2):
        out.fill_(float("nan"))
        graph.replay()
        assert torch.equal(out, reference)
        assert torch.equal(cache.attention(q), reference)


def test_a_stream_as_an_argument():
    """Each call on a given stream, as a torch stream or its address, from another current stream."""
    k, v, q = normal(1, 2, 3, 2, 64), normal(2, 2, 3, 2, 64), normal(3, 2, 3, 8, 64)
    want = filled(91, [70, 20], 2, 64, 128, track=True)
    want.append(k, v)
    reference, rows = want.attention(q), want.read(80)
    want.evict(40, 8, 2)
    side = torch.cuda.Stream()
    for stream in (side, side.cuda_stream):
        got = filled(91, [70, 20], 2, 64, 128, track=True)
        side.wait_stream(torch.cuda.current_stream())
        got.append(k, v, stream=stream)
        out = got.attention(q, stream=stream)
        read = got.read(80, stream=stream)
        got.evict(40, 8, 2, stream=stream)
        p = torch.full((2, 3, 7), 1 / 7, device="cuda")
        side.wait_stream(torch.cuda.current_stream())
        accepted, token = kv4.verify_draft(ints(1, 2, 3, 4).view(2, 2), p[:, :2].contiguous(), p,
                                           torch.zeros(2, 2, device="cuda"), torch.zeros(2, device="cuda"), stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(out, reference) and torch.equal(got.state, want.state) and torch.equal(got.weights, want.weights)
        assert all(torch.equal(a, b) for a, b in zip(read, rows))
        assert accepted.tolist() == [2, 2] and token.tolist() == [0, 0]


def test_the_default_streams_address():
    """Address 0 is the default stream, from any current stream."""
    cache = filled(92, [70, 20], 2, 64, 128)
    seen = []
    cache._lib = type("Calls", (), {"vg_k_kv4_append": lambda *a: seen.append(a[-1]) or 0})()
    k = normal(1, 2, 3, 2, 64)
    assert torch.cuda.default_stream().cuda_stream == 0
    with torch.cuda.stream(torch.cuda.Stream()):
        current = torch.cuda.current_stream().cuda_stream
        cache.append(k, k, stream=0)
        cache.append(k, k)
    assert seen == [0, current]


def test_one_workspace_serves_calls_of_any_shape():
    cache = filled(61, [500, 90], 2, 128, 512, track=True)
    fresh = filled(61, [500, 90], 2, 128, 512, track=True)
    big = normal(1, 2, 64, 16, 128)
    cache.attention(big)
    for tokens in (1, 5, 64, 1, 17):
        q = normal(tokens, 2, tokens, 16, 128, dtype=torch.float16)
        fresh._workspace = None
        assert torch.equal(cache.attention(q, track=False), fresh.attention(q, track=False))


def test_refusals_name_the_fault():
    cache = filled(71, [10], 2, 64, 64)
    q = normal(1, 1, 1, 4, 64)
    with pytest.raises(VoxGenError, match="not supported"):
        cache.attention(q.double())
    with pytest.raises(VoxGenError, match="does not track"):
        cache.attention(q, track=True)
    with pytest.raises(VoxGenError, match="VG_EINVAL"):
        cache.attention(normal(1, 1, 1, 3, 64))
    with pytest.raises(VoxGenError, match="expected"):
        cache.attention(normal(1, 2, 1, 4, 64))
    with pytest.raises(VoxGenError, match="out must"):
        cache.attention(q, out=q.half())
    with pytest.raises(VoxGenError, match="agree"):
        cache.append(normal(1, 1, 1, 2, 64), normal(1, 1, 2, 2, 64))
    with pytest.raises(VoxGenError, match="VG_EFULL"):
        cache.append(*(normal(1, 1, 65, 2, 64),) * 2)
    with pytest.raises(VoxGenError, match="counts"):
        cache.append(*(normal(1, 1, 1, 2, 64),) * 2, counts=torch.ones(1, device="cuda"))
    with pytest.raises(VoxGenError, match="channels"):
        cache.append(*(normal(1, 1, 1, 64, 2).transpose(2, 3),) * 2)
    with pytest.raises(VoxGenError, match="VG_EINVAL"):
        cache.evict(10)
    with pytest.raises(VoxGenError, match="VG_EUNSUPPORTED"):
        kv4.Kv4Cache(1, 2, 32, 64)
    with pytest.raises(VoxGenError, match="state"):
        kv4.Kv4Cache(1, 2, 64, 64, state=torch.zeros(2, 4, dtype=torch.int32, device="cuda"))
    assert cache.rows().tolist() == [10]


def test_more_sequences_than_can_be_cut():
    """Past 16384 segments every one is a piece; a sample of them is checked."""
    seqs = 2100
    rows = [1 + i * 7 % 150 for i in range(seqs)]
    cache = filled(81, rows, 8, 64, 150)
    q = normal(82, seqs, 1, 8, 64)
    out = cache.attention(q)
    assert torch.equal(out, cache.attention(q))
    some = list(range(0, seqs, 97)) + [seqs - 1]
    run = 8 * -(-150 // 64) * 72 * 64
    raw = cache.data.view(seqs, run)[some].cpu().numpy()
    k, v = R.unpack(raw, len(some), 8, 64, 150)
    qn = q[some].double().cpu().numpy()
    want, _ = R.attention(qn, k, v, [rows[i] for i in some])
    _, tol = tolerance(qn, k, v, [rows[i] for i in some], "f32")
    assert np.abs(out[some].double().cpu().numpy() - want).max() <= tol


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_long_accumulation(dtype):
    """Dozens of cache tiles in one CTA, some tokens past their count. Tensor-core sums round towards zero, so a long
    fp32 accumulation would drift: 2^-22 of the result for a tile, of which a few (at most 4) are summed before a sum
    that rounds to nearest takes over (2^-20), fp32 sums and 22-bit operands beside it: 2^-18 of the result in the 2-norm. Rounding P
    and the output to fp16 adds 2^-11."""
    seqs, tokens = 30, 40
    counts = [(40, 5, 0)[i % 3] for i in range(seqs)]
    cache = filled(83, [4000] * seqs, 8, 64, 4000)
    q = normal(84, seqs, tokens, 8, 64, dtype=TYPES[dtype])
    out = cache.attention(q, counts=ints(*counts))
    assert torch.equal(out, cache.attention(q, counts=ints(*counts)))
    some = [0, 1, 2, 16, 28, 29]
    raw = cache.data.view(seqs, -1)[some].cpu().numpy()
    k, v = R.unpack(raw, len(some), 8, 64, 4000)
    want, _ = R.attention(q[some].double().cpu().numpy(), k, v, [4000] * len(some), [counts[i] for i in some])
    got = out[some].double().cpu().numpy()
    assert not got[want == 0].any()
    tol = 2.0 ** -18 + (2.0 ** -11 if dtype == "f16" else 0)
    assert np.linalg.norm(got - want) <= tol * np.linalg.norm(want)


# ---------------------------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------------------------
def evict_case(seed, seqs, kv_heads, dim, capacity, rows, ties):
    rng = np.random.default_rng(seed)
    cache = kv4.Kv4Cache(seqs, kv_heads, dim, capacity, track=True)
    cache.data.copy_(torch.from_numpy(rng.integers(0, 256, cache.data.numel(), dtype=np.uint8)))
    w = np.exp(rng.standard_normal((seqs, kv_heads, capacity)) * 2).astype(np.float32)
    if ties:
        w = np.round(w).astype(np.float32)
    pos = np.stack([[rng.permutation(2 * capacity)[:capacity] for _ in range(kv_heads)] for _ in range(seqs)])
    cache.weights.copy_(torch.from_numpy(w))
    cache.positions.copy_(torch.from_numpy(pos.astype(np.int32)))
    cache.state[:, 0] = ints(*rows)
    cache.state[:, 1] = 2 * capacity
    return cache


@pytest.mark.parametrize("separate", [False, True])
@pytest.mark.parametrize("seqs,kv_heads,dim,capacity,rows,budget,recent,sinks,ties", [
    (1, 1, 128, 2, [2], 1, 0, 0, False), (3, 2, 64, 130, [130, 64, 65], 64, 8, 4, True),
    (2, 3, 128, 700, [700, 0], 699, 100, 0, False), (2, 2, 128, 1500, [1500, 1027], 1, 1, 0, True),
    (1, 2, 64, 5000, [4999], 1300, 1300, 0, True), (2, 1, 128, 3000, [3000, 2000], 2000, 0, 0, True),
    (1, 1, 64, 600, [600], 600, 5, 5, False), (1, 8, 128, 1025, [1025], 513, 511, 2, False)])
def test_evict(separate, seqs, kv_heads, dim, capacity, rows, budget, recent, sinks, ties):
    cache = evict_case(seqs + capacity, seqs, kv_heads, dim, capacity, rows, ties)
    w, pos = cache.weights.cpu().numpy(), cache.positions.cpu().numpy()
    k, v = held(cache)
    bookkeeping = [x.clone() for x in (cache.state, cache.weights, cache.positions)]
    result = cache
    if separate:
        result = kv4.Kv4Cache(seqs, kv_heads, dim, capacity, data=cache.data, track=True)
        cache.evict(budget, recent, sinks, into=result)
        for a, b in zip((cache.state, cache.weights, cache.positions), bookkeeping):
            assert torch.equal(a, b)
    else:
        cache.evict(budget, recent, sinks)
    gk, gv = held(cache)
    gw, gp = result.weights.cpu().numpy(), result.positions.cpu().numpy()
    for s in range(seqs):
        assert result.state[s].tolist() == [min(rows[s], budget), 2 * capacity, 0, 0]
        for h in range(kv_heads):
            src = R.evict(w[s, h], pos[s, h], rows[s], 2 * capacity, budget, recent, sinks)
            n = budget if src is not None else rows[s]
            src = np.arange(n) if src is None else np.array(src)
            np.testing.assert_array_equal(gw[s, h, :n], w[s, h, src])
            np.testing.assert_array_equal(gp[s, h, :n], pos[s, h, src])
            np.testing.assert_array_equal(gk[s, h, :n], k[s, h, src])
            np.testing.assert_array_equal(gv[s, h, :n], v[s, h, src])
            np.testing.assert_array_equal(gk[s, h, budget:], k[s, h, budget:])   # rows past the budget are left


@pytest.mark.parametrize("separate", [False, True])
@pytest.mark.parametrize("seqs,kv_heads,dim,capacity,rows,budget,recent,sinks,ties", [
    (1, 1, 64, 32768, [32768], 16384, 100, 4, False),                  # the most rows whose keys fit beside the lists
    (1, 2, 64, 40000, [39999], 20000, 300, 4, True), (2, 1, 128, 65536, [65536, 50001], 32768, 0, 0, False),
    (1, 1, 64, 65536, [65536], 65535, 0, 1, True), (1, 1, 128, 65536, [65535], 1, 0, 0, True)])
def test_evict_of_long_caches(separate, seqs, kv_heads, dim, capacity, rows, budget, recent, sinks, ties):
    """Rows past 32768: 16-bit lists of up to 32768 rows, keys formed anew in every pass."""
    test_evict(separate, seqs, kv_heads, dim, capacity, rows, budget, recent, sinks, ties)


def test_evict_odd_weights():
    """NaN goes first, then -inf, then by value; -0 and +0 tie; +inf and protected rows stay."""
    nan, inf = float("nan"), float("inf")
    w = [0.0, nan, -0.0, inf, -inf, 1.0, nan, -1.0]
    for budget, want in ((7, {0, 2, 3, 4, 5, 6, 7}), (6, {0, 2, 3, 4, 5, 7}), (5, {0, 2, 3, 5, 7}), (4, {0, 2, 3, 5}),
                         (3, {0, 3, 5}), (2, {3, 5}), (1, {3})):
        cache = kv4.Kv4Cache(1, 1, 64, 8, track=True)
        cache.data.zero_()
        cache.weights[0, 0] = torch.tensor(w, device="cuda")
        cache.positions[0, 0] = torch.arange(8, dtype=torch.int32, device="cuda")
        cache.state[0, :2] = 8
        cache.evict(budget)
        got = set(cache.positions[0, 0, :budget].tolist())
        if budget == 7:   # of two NaN rows the lower one stays
            want = {0, 1, 2, 3, 4, 5, 7}
        assert got == want, (budget, got)


# ---------------------------------------------------------------------------------------------
# verification
# ---------------------------------------------------------------------------------------------
def check_verify(tokens, draft, target, ua, us, counts=None):
    dev = [torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in (tokens, draft, target, ua, us)]
    accepted, nxt = kv4.verify_draft(*dev, counts=None if counts is None else ints(*counts))
    for s in range(tokens.shape[0]):
        c = tokens.shape[1] if counts is None else counts[s]
        want = R.verify(tokens[s, :c], draft[s, :c], target[s, :c + 1], ua[s], us[s])
        assert (accepted[s].item(), nxt[s].item()) == want, s


def softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


@pytest.mark.parametrize("seqs,drafted,vocab,heat", [(1, 1, 1, 1.0), (4, 3, 2, 1.0), (9, 8, 96, 2.0), (5, 4, 1025, 0.0),
                                                     (3, 2, 5003, 3.0), (2, 20, 300, 6.0), (2, 3, 73448, 2.5)])
def test_verify(seqs, drafted, vocab, heat):
    rng = np.random.default_rng(vocab + seqs)
    logits = rng.standard_normal((seqs, drafted + 1, vocab)) * heat
    target = softmax(logits)
    draft = softmax(logits[:, :drafted] + rng.standard_normal((seqs, drafted, vocab)) * 0.5)
    tokens = np.array([[rng.choice(vocab, p=d.astype(np.float64) / d.sum(dtype=np.float64)) for d in row] for row in draft], np.int32)
    ua, us = (rng.random(n, dtype=np.float32) for n in ((seqs, drafted), seqs))
    check_verify(tokens, draft, target, ua, us)
    check_verify(tokens, draft, target, np.zeros_like(ua), us)     # accepts all
    counts = [int(c) for c in rng.integers(0, drafted + 1, seqs)]
    check_verify(tokens, draft, target, ua, us, counts)


def test_verify_edges():
    """Equal distributions, tokens outside the vocabulary, zero and odd probabilities, u at its ends."""
    v = 100
    even = np.full((1, 1, v), 1 / v, np.float32)
    two = np.concatenate([even, even], 1)
    last = np.float32(1 - 2.0 ** -24)
    for u in (0.0, 0.5, last):
        for us in (0.0, 0.25, last):
            check_verify(np.array([[7]], np.int32), even, two, np.array([[u]], np.float32), np.array([us], np.float32))
    for bad in (-1, v, 2 ** 31 - 1, -2 ** 31):
        check_verify(np.array([[bad]], np.int32), even, two, np.zeros((1, 1), np.float32), np.array([0.3], np.float32))
    more = two * np.float32(1.25)
    check_verify(np.array([[3]], np.int32), more[:, :1], two, np.array([[0.9]], np.float32), np.array([0.6], np.float32))
    odd = two.copy()
    odd[0, :, 10] = np.nan
    odd[0, :, 11] = -1.0
    odd[0, :, 12] = np.inf
    check_verify(np.array([[10]], np.int32), even, odd, np.array([[0.5]], np.float32), np.array([0.7], np.float32))
    zero = np.zeros_like(two)
    check_verify(np.array([[10]], np.int32), even, zero, np.array([[0.5]], np.float32), np.array([0.7], np.float32))


def test_verify_draws_from_the_target():
    """Over many random numbers the token after one draft follows the target's distribution: a draft is a way
    to draw, not a bias. 200000 draws over 5 tokens: each share is within 5 standard deviations."""
    n = 200000
    g = torch.Generator(device="cuda").manual_seed(3)
    p = torch.tensor([0.4, 0.3, 0.2, 0.07, 0.03], device="cuda")
    q = torch.tensor([0.1, 0.5, 0.05, 0.3, 0.05], device="cuda")
    drafted = torch.multinomial(q, n, replacement=True, generator=g).int().unsqueeze(1)
    ua, us = torch.rand(n, 1, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda")
    accepted, token = kv4.verify_draft(drafted, q.expand(n, 1, 5).contiguous(), p.expand(n, 2, 5).contiguous(), ua, us)
    first = torch.where(accepted == 1, drafted[:, 0], token)
    share = torch.bincount(first.long(), minlength=5).double().cpu() / n
    sd = (p * (1 - p) / n).sqrt().double().cpu()
    assert ((share - p.double().cpu()).abs() <= 5 * sd).all(), share


# ---------------------------------------------------------------------------------------------
# the operators together
# ---------------------------------------------------------------------------------------------
def example():
    import importlib.util
    from pathlib import Path
    path = Path(__file__).resolve().parents[1] / "examples" / "kv4_session.py"
    spec = importlib.util.spec_from_file_location("kv4_session", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_a_parked_session_goes_on(tmp_path):
    """A session's cache in 4 bits and back: the hidden states stay near those of the session that kept fp16.
    A block's step is 1/8 of its largest magnitude, so a cached value is off by at most 1/16 of it (1/8 for the one
    opposite the largest); after two layers and a norm the states (of order 1) may differ by a few tenths."""
    worst, (half, four) = example().park(tmp_path)
    assert 0 < worst < 1.0
    assert four * 3 < half * 64 / 48       # 48 rows take a whole tile of 64


def test_speculation_over_an_evicting_cache():
    """The loop against the same loop whose attention is plain torch over the values that the cache stands for."""
    module = example()

    def plain(cache, q):
        k, v = (x.permute(0, 2, 1, 3) for x in cache.read(cache.capacity, dtype=torch.float32))
        streams, n, heads, dim = q.shape
        group = heads // cache.kv_heads
        k, v = (x.repeat_interleave(group, 1) for x in (k, v))
        s = q.permute(0, 2, 1, 3) @ k.transpose(2, 3) / dim ** 0.5
        seen = cache.rows()[:, None] - n + 1 + torch.arange(n, device="cuda")
        hidden = torch.arange(cache.capacity, device="cuda") >= seen[..., None]
        p = s.masked_fill(hidden[:, None], float("-inf")).softmax(-1)
        cache.weights += p.sum(2).unflatten(1, (cache.kv_heads, group)).sum(2)
        return (p @ v).permute(0, 2, 1, 3)

    tokens, cache = module.speculate()
    want, other = module.speculate(attend=plain)
    assert torch.equal(tokens, want)
    assert torch.equal(cache.positions[:, :, :48], other.positions[:, :, :48])
    n = cache.rows().tolist()
    assert max(n) == 48 and not any(cache.status())
    # the rows that stay are distinct positions, the last 16 and the first 2 among them
    last = cache.state[:, 1].tolist()
    for i in range(4):
        for h in range(2):
            held = cache.positions[i, h, :n[i]].tolist()
            assert len(set(held)) == n[i] and {0, 1} <= set(held) and set(range(last[i] - 16, last[i])) <= set(held)
