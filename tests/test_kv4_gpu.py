"""The four-bit key/value cache on the GPU: append, read-out and attention against a plain restatement (tests/kv4_reference.py).

What the cache holds is compared bit for bit.  Attention is held to a bound per number: with u = 2^-8 (half a step of bf16), the result is rounded once
(u |y|); each softmax weight, and each value where the kernel rounds step * code + low, may be off by u (2 u sum p |v|); each key likewise,
which moves a score by at most e = u scale sum |q k| and a normalised weight by a factor within exp(2 e) (e over all the row sees); f32 sums add less than the
last place that is spared here (1e-5)."""
import ctypes as C

import numpy as np
import pytest

import kv4_reference as ref
from test_recorded_launches_gpu import Driver

pytestmark = pytest.mark.gpu


class Device:
    """Uploads that are given back together."""

    def __init__(self, rt):
        self.rt, self.bufs = rt, []

    def up(self, a):
        self.bufs.append(self.rt.upload(a))
        return self.bufs[-1]

    def free(self):
        for b in self.bufs:
            b.free()


@pytest.fixture()
def dev(rt):
    d = Device(rt)
    yield d
    rt.synchronize()
    d.free()


def make_batch(t0, dev, cache, pool, rows, uniform=False, n_rows=None, first=0):
    """The record of a batch whose sequence b has rows[b] rows; the buffers it names are kept on `dev`."""
    start = np.concatenate([[first], first + np.cumsum(rows)]).astype(np.int32)
    table, lens, starts = dev.up(cache.table), dev.up(np.array(cache.lens, np.int32)), dev.up(start)
    total = int(start[-1]) if n_rows is None else n_rows
    b = dev.rt.kv4_batch(pool.gpu_addr(), table.gpu_addr(), lens.gpu_addr(), n_pages=cache.n_pages, page_size=cache.page, n_kv_heads=cache.heads,
                         head_dim=cache.dim, n_seqs=len(rows), table_stride=cache.stride, n_rows=total, max_rows=max(max(rows), 1),
                         row_start=0 if uniform else starts.gpu_addr())
    b.buffers = (table, lens, starts)
    return b


def tokens_of(cache, rows):
    return [np.arange(n - r, n) for n, r in zip(cache.lens, rows)]


# --------------------------------------------------------------------------- append and read-out

def rope_table(rng, n, pairs):
    a = rng.uniform(-np.pi, np.pi, (n, pairs))
    return np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)


APPENDS = [
    # lens, rows, heads, group, dim, page, f32, rot, interleaved, axes
    ([1], [1], 1, 1, 64, 16, True, 64, False, None),
    ([300], [1], 8, 4, 128, 64, True, 128, False, None),
    ([17, 5, 64, 1], [1, 1, 1, 1], 2, 7, 128, 32, False, 64, True, None),
    ([40, 16, 33], [40, 3, 17], 3, 2, 64, 16, False, 32, False, None),
    ([65, 200], [64, 5], 2, 1, 128, 64, True, 16, True, None),
    ([70, 9], [70, 9], 1, 4, 128, 32, False, 128, False, [24, 20, 20]),
    ([70, 9], [70, 9], 2, 3, 64, 16, True, 64, True, [12, 0, 20]),
    ([31], [12], 4, 1, 64, 32, True, 48, False, [20, 4]),
    ([3, 0, 7], [1, 1, 1], 2, 2, 128, 16, True, 0, False, None),           # no rotation; an empty slot
    ([2, 8], [5, 5], 2, 2, 64, 16, False, 64, False, None),                # more rows than tokens
]


@pytest.mark.parametrize("lens, rows, heads, group, dim, page, f32, rot, interleaved, axes", APPENDS)
def test_append_holds_the_rows_and_rotates_the_queries(t0, rt, dev, lens, rows, heads, group, dim, page, f32, rot, interleaved, axes):
    rng = np.random.default_rng(sum(lens) + dim)
    cache = ref.Cache(rng, lens, heads, dim, page)
    before = rng.integers(0, 256, (cache.n_pages, heads, page * (dim + 8)), dtype=np.uint8)
    pool = dev.up(before)
    n, extra, hq = sum(rows), 2, group * heads
    total = n + extra                                                     # rows behind the last sequence
    b = make_batch(t0, dev, cache, pool, rows, n_rows=total)
    x = (rng.standard_normal((total, hq + 2 * heads, dim)) * 2).astype(np.float32)
    if not f32:
        x = ref.bf16_round(x)
    data = dev.up(x if f32 else ref.bf16_bits(x))
    size, wide = (4 if f32 else 2), (hq + 2 * heads) * dim
    out_stride = hq * dim + 16
    q_out = dev.up(np.full((total, out_stride), 0xABCD, np.uint16))
    n_positions = 400
    table = rope_table(rng, n_positions, max(rot, 16) // 2)
    positions = rng.integers(0, n_positions, (3, total)).astype(np.int32)
    kw = dict(rope=dev.up(table).gpu_addr(), n_positions=n_positions, rot_dim=rot, interleaved=interleaved) if rot else {}
    if axes:
        kw.update(axis_pairs=axes, positions=dev.up(positions[:len(axes)]).gpu_addr())
    at = data.gpu_addr()
    rt.kv4_append(b, rt.kv4_append_args(at + hq * dim * size, at + (hq + heads) * dim * size, k_stride=wide, v_stride=wide, in_f32=f32, q=at, q_stride=wide,
                                        q_out=q_out.gpu_addr(), q_out_stride=out_stride, n_q_heads=hq, **kw))
    rt.synchronize()
    token = np.concatenate(tokens_of(cache, rows))
    turned = x[:n].copy()
    if rot:
        pairs = rot // 2
        if axes:
            axis = np.repeat(np.arange(len(axes)), axes)
            cs = table[positions[axis][:, :n].T, np.arange(pairs)]
        else:
            cs = table[np.maximum(token, 0)]
        turned[:, :hq + heads] = ref.rotate(x[:n, :hq + heads], cs, interleaved)
    # queries
    got = q_out.read(total * out_stride * 2, np.uint16).reshape(total, out_stride)
    want = np.full((total, out_stride), 0xABCD, np.uint16)
    have = token >= 0
    want[:n, :hq * dim][have] = ref.bf16_bits(turned[:, :hq]).reshape(n, -1)[have]
    assert np.array_equal(got, want)
    # the pool: the rows' places hold them, every other byte is as it was
    k, v = turned[:, hq:hq + heads], turned[:, hq + heads:]
    want = before.copy()
    half = page * dim // 2
    seq = np.repeat(np.arange(len(rows)), rows)
    for r in np.flatnonzero(have):
        block, slot = want[cache.table[seq[r], token[r] // page]], token[r] % page
        new = ref.block_bytes(k[r][:, None], v[r][:, None])                # blocks of one token
        for start, row, piece in ((0, dim // 2, 0), (half, dim // 2, dim // 2), (2 * half, 4, dim), (2 * half + 4 * page, 4, dim + 4)):
            block[:, start + slot * row:start + (slot + 1) * row] = new[:, piece:piece + row]
    assert np.array_equal(pool.read(before.size).reshape(before.shape), want)
    # read back
    stride = heads * dim + 8
    ko, vo = (dev.up(np.full((total, stride), 0xABCD, np.uint16)) for _ in range(2))
    rt.kv4_dequant(b, rt.kv4_dequant_args(ko.gpu_addr(), vo.gpu_addr(), k_out_stride=stride, v_out_stride=stride))
    rt.synchronize()
    for buf, x64 in ((ko, ref.held(k)), (vo, ref.held(v))):
        want = np.full((total, stride), 0xABCD, np.uint16)
        want[:n, :heads * dim] = ref.bf16_bits(x64.astype(np.float32)).reshape(n, -1)
        want[:n, :heads * dim][~have] = 0
        assert np.array_equal(buf.read(total * stride * 2, np.uint16).reshape(total, stride), want)


@pytest.mark.parametrize("f32, interleaved", [(False, False), (True, False), (False, True)])
def test_a_long_append_is_exact(t0, rt, dev, f32, interleaved):
    # six million numbers: an operation that is not rounded by itself, or a quotient off by its last place, shows in some of them
    rng = np.random.default_rng(77)
    heads, dim, page, n = 8, 128, 64, 1024
    cache = ref.Cache(rng, [n], heads, dim, page, spare=0, extra_columns=0)
    pool = dev.up(np.zeros((cache.n_pages, heads, page * (dim + 8)), np.uint8))
    b = make_batch(t0, dev, cache, pool, [n], uniform=True)
    x = (rng.standard_normal((n, 6 * heads, dim)) * 2).astype(np.float32)
    if not f32:
        x = ref.bf16_round(x)
    data, table, q_out = dev.up(x if f32 else ref.bf16_bits(x)), rope_table(rng, n, dim // 2), dev.up(np.zeros((n, 4 * heads, dim), np.uint16))
    at, size, wide = data.gpu_addr(), (4 if f32 else 2), 6 * heads * dim
    rt.kv4_append(b, rt.kv4_append_args(at + 4 * heads * dim * size, at + 5 * heads * dim * size, k_stride=wide, v_stride=wide, in_f32=f32, q=at, q_stride=wide,
                                        q_out=q_out.gpu_addr(), n_q_heads=4 * heads, rope=dev.up(table).gpu_addr(), n_positions=n, rot_dim=dim, interleaved=interleaved))
    rt.synchronize()
    turned = ref.rotate(x[:, :5 * heads], table, interleaved)
    assert np.array_equal(q_out.read(n * 4 * heads * dim * 2, np.uint16), ref.bf16_bits(turned[:, :4 * heads]).ravel())
    k, x = turned[:, 4 * heads:], x[:, 4 * heads:]
    want = ref.block_bytes(*(a.reshape(-1, page, heads, dim).transpose(0, 2, 1, 3) for a in (k, x[:, heads:])))
    got = pool.read(want.size).reshape(want.shape[0], heads, -1)[cache.table[0]]
    assert np.array_equal(got, want)


def test_rows_that_four_bits_have_trouble_with(t0, rt, dev):
    # infinities, NaNs, ranges that overflow or vanish, constants, ties: the bytes are the restatement's, and what is read back its values
    rng = np.random.default_rng(5)
    dim, page = 64, 16
    x = rng.standard_normal((16, 1, dim)).astype(np.float32)
    x[0, 0, 7], x[1, 0, 8], x[2, 0, 63] = np.inf, -np.inf, np.nan
    x[3, 0, :2] = 3e38, -3e38                                               # the range overflows
    x[4] = 0.0
    x[5] = -0.0
    x[6] = 1.2345
    x[7] = np.float32(1e-40) * np.arange(dim)                               # subnormal range
    x[8] = np.float32(2.0**-120) * np.arange(dim)
    x[9] = np.arange(dim) % 31 / 2.0                                        # every second one a tie
    x[10] = 1000.0 + rng.uniform(0, 0.1, dim)                               # far from zero, close together
    x[11] *= 1e30
    x[12, 0, :] = np.float32(3.3e38)
    x[13, 0, :] = np.float32(-3.4e38)                                       # low rounds to minus infinity
    cache = ref.Cache(rng, [16], 1, dim, page, spare=0)
    pool = dev.up(np.zeros((1, 1, page * (dim + 8)), np.uint8))
    b = make_batch(t0, dev, cache, pool, [16], uniform=True)
    data = dev.up(x)
    rt.kv4_append(b, rt.kv4_append_args(data.gpu_addr(), data.gpu_addr(), in_f32=True))
    out = dev.up(np.zeros((2, 16, dim), np.uint16))
    rt.kv4_dequant(b, rt.kv4_dequant_args(out.gpu_addr(), 0))
    rt.kv4_dequant(b, rt.kv4_dequant_args(0, out.gpu_addr() + 16 * dim * 2))
    rt.synchronize()
    rows = x.transpose(1, 0, 2)
    got, want = pool.read(page * (dim + 8)).reshape(1, -1), ref.block_bytes(rows, rows)
    low = lambda a: a[:, page * dim:].copy().view(np.uint16) & 0x7FFF       # noqa: E731  (a zero may carry either sign)
    zero = low(want) == 0
    assert np.array_equal(got[:, :page * dim], want[:, :page * dim])
    assert np.array_equal(np.where(zero, low(got), got[:, page * dim:].copy().view(np.uint16)), np.where(zero, 0, want[:, page * dim:].copy().view(np.uint16)))
    k = ref.from_bits(out.read(2 * 16 * dim * 2, np.uint16)).reshape(2, 16, dim)
    with np.errstate(all="ignore"):
        expect = ref.bf16_round(ref.held(x)[:, 0].astype(np.float32))
    assert np.array_equal(np.isnan(k[0]), np.isnan(expect)) and np.array_equal(k[0][~np.isnan(k[0])], expect[~np.isnan(expect)])
    assert np.array_equal(out.read(2 * 16 * dim * 2, np.uint16).reshape(2, -1)[0], out.read(2 * 16 * dim * 2, np.uint16).reshape(2, -1)[1])
    assert sorted(set(np.flatnonzero(np.isnan(k[0]).any(1)))) == [0, 1, 2, 3, 13]


# --------------------------------------------------------------------------- attention

def check_attention(t0, rt, dev, lens, rows, heads, group, dim, page, window=0, uniform=False, stride=0, seed=0, scale=None, sharp=1.5, before=None, first=0, behind=0):
    rng = np.random.default_rng(seed + sum(lens))
    cache = ref.Cache(rng, lens, heads, dim, page)
    if before:
        before(cache, rng)
    pool = dev.up(cache.pool())
    hq, n = heads * group, sum(rows)
    total = first + n + behind
    scale = scale or dim**-0.5
    q = ref.bf16_round((rng.standard_normal((total, hq, dim)) * sharp).astype(np.float32))
    width = stride or hq * dim
    q_rows = np.zeros((total, width), np.uint16)
    q_rows[:, :hq * dim] = ref.bf16_bits(q).reshape(total, -1)
    qb, yb = dev.up(q_rows), dev.up(np.full((total, width), 0xABCD, np.uint16))
    b = make_batch(t0, dev, cache, pool, rows, uniform, n_rows=total, first=first)
    args = rt.kv4_attention_args(qb.gpu_addr(), yb.gpu_addr(), n_q_heads=hq, scale=scale, window=window, q_stride=stride, y_stride=stride)
    rt.kv4_attention(b, args)
    rt.synchronize()
    bits = yb.read(total * width * 2, np.uint16).reshape(total, width)
    y = ref.from_bits(bits[:, :hq * dim].copy()).reshape(total, hq, dim).astype(np.float64)
    assert np.all(bits[:, hq * dim:] == 0xABCD) and np.all(bits[:first] == 0xABCD) and np.all(bits[first + n:] == 0xABCD)
    at = first
    for s, (r, t) in enumerate(zip(rows, tokens_of(cache, rows))):
        if r == 0:
            continue
        k, v = ref.held(cache.k[s]), ref.held(cache.v[s])
        want, weight, reach = ref.attention(q[at:at + r].astype(np.float64), k, v, t, np.float64(np.float32(scale)), window)
        got = y[at:at + r]
        bound = ref.U * np.abs(want) + (2 * ref.U + np.expm1(2 * ref.U * reach))[..., None] * weight + 1e-5 * weight
        assert np.array_equal(np.isnan(got), np.isnan(want)), f"sequence {s}: NaN where there is none, or none where there is"
        fine = ~np.isnan(want)
        over = (np.abs(got - want) - bound)[fine]
        assert over.size == 0 or over.max() <= 0, f"sequence {s}: {over.max()} over the bound at {np.unravel_index(np.argmax(np.where(fine, np.abs(got - want) - bound, -1)), got.shape)}"
        at += r
    # the call repeats bit for bit
    again = dev.up(np.full((total, width), 0xABCD, np.uint16))
    args.y = again.gpu_addr()
    rt.kv4_attention(b, args)
    rt.synchronize()
    assert np.array_equal(again.read(total * width * 2, np.uint16).reshape(total, width), bits)
    return y


DECODE = [
    # lens, heads, group, dim, page, window
    ([1], 1, 1, 64, 16, 0), ([1], 1, 1, 128, 64, 0), ([2], 2, 4, 128, 32, 0), ([15, 16, 17], 2, 1, 64, 16, 0),
    ([63, 64, 65, 1], 2, 8, 128, 64, 0), ([77], 8, 4, 128, 16, 0), ([129, 400, 5], 3, 7, 64, 32, 0), ([700], 1, 16, 128, 32, 0),
    ([513, 1000], 2, 3, 128, 64, 0), ([300, 20, 64, 65], 2, 2, 64, 16, 64), ([300, 200], 1, 5, 128, 32, 1), ([200, 129], 2, 1, 128, 64, 100),
    ([2000], 1, 8, 128, 16, 0), ([1999, 3], 4, 1, 64, 64, 777), ([90, 33], 1, 17, 64, 16, 0), ([150], 1, 64, 128, 32, 0),
]


@pytest.mark.parametrize("lens, heads, group, dim, page, window", DECODE)
def test_attention_of_single_tokens(t0, rt, dev, lens, heads, group, dim, page, window):
    check_attention(t0, rt, dev, lens, [1] * len(lens), heads, group, dim, page, window, uniform=True)


ROWS = [
    # lens, rows, heads, group, dim, page, window
    ([2, 40], [2, 2], 2, 4, 128, 16, 0), ([100, 64, 9], [5, 3, 1], 2, 1, 64, 32, 0), ([70, 300], [8, 8], 1, 2, 128, 64, 0), ([130], [8], 2, 8, 64, 16, 50),
    ([17], [17], 2, 1, 128, 16, 0), ([50, 128], [33, 128], 1, 2, 64, 32, 0), ([260], [130], 2, 1, 128, 64, 0), ([127, 129, 128], [127, 129, 128], 1, 1, 64, 64, 0),
    ([300, 1, 90, 40], [60, 1, 1, 40], 2, 7, 64, 16, 0), ([200, 333], [200, 100], 1, 4, 128, 32, 64), ([400], [257], 1, 3, 128, 16, 0),
    ([513], [40], 2, 5, 128, 64, 0), ([90], [90], 1, 16, 64, 32, 7), ([520, 385], [300, 1], 1, 1, 128, 64, 129),
    ([64, 640], [20, 20], 1, 64, 64, 64, 0), ([1000], [3], 1, 6, 128, 64, 0),
]


@pytest.mark.parametrize("lens, rows, heads, group, dim, page, window", ROWS)
def test_attention_of_several_rows(t0, rt, dev, lens, rows, heads, group, dim, page, window):
    check_attention(t0, rt, dev, lens, rows, heads, group, dim, page, window)


@pytest.mark.parametrize("dim, rows", [(64, [1, 1, 1]), (128, [1, 1, 1]), (128, [40, 30, 1]), (64, [30, 40, 20])])
def test_attention_with_strides_and_rows_of_no_sequence(t0, rt, dev, dim, rows):
    check_attention(t0, rt, dev, [70, 41, 90], rows, 2, 2, dim, 16, stride=4 * dim + 24, first=3, behind=4)


@pytest.mark.parametrize("rows", [[1, 0, 1, 1], [3, 2, 0, 5], [40, 50, 0, 60]])
@pytest.mark.parametrize("dim", [64, 128])
def test_sequences_without_tokens_or_rows(t0, rt, dev, rows, dim):
    # empty slots give zeros, rows before the first token too
    y = check_attention(t0, rt, dev, [0, 5, 0, 33], rows, 2, 4, dim, 16)
    assert np.all(y[:rows[0]] == 0)


@pytest.mark.parametrize("rows, group", [([1], 4), ([6], 1), ([50], 4)])
def test_sharp_and_flat_softmax(t0, rt, dev, rows, group):
    check_attention(t0, rt, dev, [150], rows, 1, group, 128, 32, sharp=40.0)
    check_attention(t0, rt, dev, [150], rows, 1, group, 64, 32, scale=1e-6)
    check_attention(t0, rt, dev, [150], rows, 1, group, 64, 32, scale=3.0)


@pytest.mark.parametrize("rows, group", [([1, 1], 4), ([30, 30], 4), ([4, 30], 2)])
@pytest.mark.parametrize("what", ["k", "v"])
def test_a_nan_reaches_the_rows_that_see_it_and_no_others(t0, rt, dev, rows, group, what):
    # rows at tokens before it, and rows whose window has passed it, keep their numbers
    def spoil(cache, rng):
        getattr(cache, what)[0][80, 1, 3] = np.nan
        getattr(cache, what)[1][60, 0, 3] = np.inf
    y = check_attention(t0, rt, dev, [90, 100], rows, 2, group, 64, 16, window=32, before=spoil)
    if rows[0] == 30:
        assert not np.isnan(y[:20]).any() and np.isnan(y[20:30, group:]).all() and not np.isnan(y[20:30, :group]).any()


@pytest.mark.parametrize("rows", [[1], [5], [40]])
def test_keys_and_values_far_from_zero(t0, rt, dev, rows):
    def move(cache, rng):
        cache.k[0] += rng.standard_normal((1, 1, 128)).astype(np.float32) * 4
        cache.v[0] += 3.0
    check_attention(t0, rt, dev, [140], rows, 1, 2, 128, 64, sharp=0.3, before=move)


@pytest.mark.parametrize("dim, rows, group", [(128, 1, 8), (64, 1, 1), (128, 4, 4), (128, 20, 4), (64, 130, 2)])
def test_one_long_sequence_is_cut_and_joined(t0, rt, dev, dim, rows, group):
    # enough tokens for every SM to get a part of the same sums
    check_attention(t0, rt, dev, [20011], [rows], 1, group, dim, 64)


@pytest.mark.parametrize("rows, group", [(1, 4), (2, 16)])
def test_many_short_sequences(t0, rt, dev, rows, group):
    lens = [int(n) for n in np.random.default_rng(3).integers(rows, 90, 400)]
    check_attention(t0, rt, dev, lens, [rows] * len(lens), 1, group, 64, 16, uniform=True)


def test_in_place(t0, rt, dev):
    rng = np.random.default_rng(8)
    for rows in ([1, 1, 1], [2, 40, 7]):
        cache = ref.Cache(rng, [50, 90, 64], 2, 128, 32)
        pool = dev.up(cache.pool())
        b = make_batch(t0, dev, cache, pool, rows)
        q = ref.bf16_bits(rng.standard_normal((sum(rows), 4, 128)).astype(np.float32))
        apart, place, y = dev.up(q), dev.up(q), dev.up(np.zeros_like(q))
        for src, dst in ((apart, y), (place, place)):
            rt.kv4_attention(b, rt.kv4_attention_args(src.gpu_addr(), dst.gpu_addr(), n_q_heads=4, scale=0.1))
        rt.synchronize()
        assert np.array_equal(y.read(q.nbytes, np.uint16), place.read(q.nbytes, np.uint16))
    x = ref.bf16_bits(rng.standard_normal((3, 8, 128)).astype(np.float32))     # q, k and v as columns; q is turned where it lies
    cache = ref.Cache(rng, [50, 90, 64], 2, 128, 32)
    pool, table = dev.up(cache.pool()), dev.up(rope_table(rng, 100, 64))
    b = make_batch(t0, dev, cache, pool, [1, 1, 1])
    wide, out = dev.up(x), dev.up(np.zeros((3, 4, 128), np.uint16))
    at = wide.gpu_addr()
    kw = dict(k_stride=1024, v_stride=1024, q=at, q_stride=1024, n_q_heads=4, rope=table.gpu_addr(), n_positions=100, rot_dim=128)
    rt.kv4_append(b, rt.kv4_append_args(at + 1024, at + 1536, q_out=out.gpu_addr(), **kw))
    rt.kv4_append(b, rt.kv4_append_args(at + 1024, at + 1536, q_out=at, q_out_stride=1024, **kw))
    rt.synchronize()
    got = wide.read(x.nbytes, np.uint16).reshape(x.shape)
    assert np.array_equal(got[:, :4], out.read(3 * 4 * 128 * 2, np.uint16).reshape(3, 4, 128)) and np.array_equal(got[:, 4:], x[:, 4:])


# --------------------------------------------------------------------------- what the device finds wrong

@pytest.fixture()
def own(t0):
    """A runtime of its own: nothing of another test is reported on it."""
    r = t0.GpuRuntime(0)
    yield r
    r.close()


def bounds_error(t0, rt, text):
    with pytest.raises(t0.T0Error) as e:
        rt.synchronize()
    assert e.value.code == 5 and text in e.value.message, e.value.message
    assert not rt.is_poisoned()
    rt.synchronize()                                                      # reported once


@pytest.mark.parametrize("rows", [[1, 1, 1], [1, 1, 30]])
@pytest.mark.parametrize("what, text", [("long", "sequence 1"), ("negative", "sequence 1"), ("page", "sequence 1"), ("negative page", "sequence 1"),
                                        ("rows outside", "sequence 2"), ("too many rows", "sequence 2"), ("descending", "sequence")])
def test_bad_device_arrays_are_left_out_and_reported(t0, own, rows, what, text):
    dev = Device(own)
    rng = np.random.default_rng(2)
    cache = ref.Cache(rng, [40, 33, 35], 2, 128, 16, extra_columns=0)
    good_table, good_lens = cache.table.copy(), list(cache.lens)
    pool_bytes = cache.pool(0)
    n = sum(rows)
    q = ref.bf16_bits(rng.standard_normal((n, 4, 128)).astype(np.float32))
    start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    most, bad_start = max(rows), start.copy()
    if what == "long":
        cache.lens[1] = cache.stride * 16 + 1
    elif what == "negative":
        cache.lens[1] = -5
    elif what == "page":
        cache.table[1, 1] = cache.n_pages
    elif what == "negative page":
        cache.table[1, 1] = -1
    elif what == "rows outside":
        bad_start[3] = n + 1
    elif what == "too many rows":
        bad_start = np.array([0, 1, 2, n + 2], np.int32)
        most, n = max(rows), n + 2
        q = np.concatenate([q, q[:2]])
    elif what == "descending":
        bad_start[2] = 0
    out = {}
    for name, table, lens, starts in (("good", good_table, good_lens, start), ("bad", cache.table, cache.lens, bad_start)):
        bufs = [dev.up(table), dev.up(np.array(lens, np.int32)), dev.up(starts)]
        pool, qb, y = dev.up(pool_bytes), dev.up(q), dev.up(np.full(q.shape, 0xABCD, np.uint16))
        b = own.kv4_batch(pool.gpu_addr(), bufs[0].gpu_addr(), bufs[1].gpu_addr(), n_pages=cache.n_pages, page_size=16, n_kv_heads=2, head_dim=128, n_seqs=3,
                          table_stride=cache.stride, n_rows=n, max_rows=most, row_start=bufs[2].gpu_addr())
        own.kv4_attention(b, own.kv4_attention_args(qb.gpu_addr(), y.gpu_addr(), n_q_heads=4, scale=0.1))
        if name == "bad":
            bounds_error(t0, own, text)
        else:
            own.synchronize()
        out[name] = y.read(q.nbytes, np.uint16).reshape(q.shape)
        k = dev.up(q)                                                     # rows of four heads: two for keys, two for values
        own.kv4_append(b, own.kv4_append_args(k.gpu_addr(), k.gpu_addr() + 512, k_stride=512, v_stride=512))
        if name == "bad" and not ("page" in what and rows[1] == 1):       # (the row of sequence 1 lies on another page)
            bounds_error(t0, own, text)
        else:
            own.synchronize()
    # the first sequence, which is in order, is computed as ever (a row that two sequences claim may be either's)
    assert what == "descending" or np.array_equal(out["bad"][:rows[0]], out["good"][:rows[0]])
    if what in ("long", "negative", "rows outside", "too many rows"):
        s = 2 if text.endswith("2") else 1
        assert np.all(out["bad"][start[s]:start[s + 1]] == 0xABCD)
    own.synchronize()
    dev.free()


@pytest.mark.parametrize("dim", [64, 128])
def test_sequences_with_the_same_rows_are_reported_and_do_no_harm(t0, own, dim):
    # row_start goes down again and again: the sequences have three times the rows that there are.  What y holds is of no use; the next call's is.
    dev = Device(own)
    rng = np.random.default_rng(6)
    cache = ref.Cache(rng, [600] * 6, 2, dim, 16)
    q = ref.bf16_bits(rng.standard_normal((600, 8, dim)).astype(np.float32))
    pool, table, lens, qb = dev.up(cache.pool(0)), dev.up(cache.table), dev.up(np.array(cache.lens, np.int32)), dev.up(q)
    out = []
    for start in ([0, 100, 200, 300, 400, 500, 600], [0, 600, 0, 600, 0, 600, 600], [0, 100, 200, 300, 400, 500, 600]):
        y = dev.up(np.full(q.shape, 0xABCD, np.uint16))
        b = own.kv4_batch(pool.gpu_addr(), table.gpu_addr(), lens.gpu_addr(), n_pages=cache.n_pages, page_size=16, n_kv_heads=2, head_dim=dim, n_seqs=6,
                          table_stride=cache.stride, n_rows=600, max_rows=600, row_start=dev.up(np.array(start, np.int32)).gpu_addr())
        own.kv4_attention(b, own.kv4_attention_args(qb.gpu_addr(), y.gpu_addr(), n_q_heads=8, scale=0.1))
        if start[2] == 0:
            bounds_error(t0, own, "sequence")
        else:
            own.synchronize()
        out.append(y.read(q.nbytes, np.uint16))
    assert np.array_equal(out[0], out[2]) and not np.any(out[0] == 0xABCD)
    dev.free()


@pytest.mark.parametrize("dim, page", [(128, 64), (64, 16)])
def test_pages_beyond_four_gigabytes(t0, own, dim, page):
    # the same calls on a small cache and on one whose pages lie at both ends of 4.8 GB: the same rows, bit for bit
    dev = Device(own)
    rng = np.random.default_rng(12)
    heads, lens = 8, [200, 65]
    cache = ref.Cache(rng, lens, heads, dim, page)
    each = t0.kv4_page_bytes(page, heads, dim)
    n_pages = 4_800_000_000 // each
    far = np.where((cache.table >= 0) & (cache.table % 3 > 0), cache.table + n_pages - cache.n_pages, cache.table).astype(np.int32)
    big = own.alloc(n_pages * each)
    dev.bufs.append(big)
    x = ref.bf16_bits(rng.standard_normal((sum(lens), 2 * heads, dim)).astype(np.float32))
    rows_in, lens_buf, got = dev.up(x), dev.up(np.array(lens, np.int32)), []
    for pages, count, table in ((dev.up(np.zeros(cache.n_pages * each, np.uint8)), cache.n_pages, cache.table), (big, n_pages, far)):
        table_buf, out = dev.up(table), []

        def batch(rows):
            start = dev.up(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32))
            return own.kv4_batch(pages.gpu_addr(), table_buf.gpu_addr(), lens_buf.gpu_addr(), n_pages=count, page_size=page, n_kv_heads=heads, head_dim=dim, n_seqs=2,
                                 table_stride=cache.stride, n_rows=sum(rows), max_rows=max(rows), row_start=start.gpu_addr())

        wide = 2 * heads * dim
        own.kv4_append(batch(lens), own.kv4_append_args(rows_in.gpu_addr(), rows_in.gpu_addr() + wide, k_stride=wide, v_stride=wide))
        k, v = (dev.up(np.zeros((sum(lens), heads, dim), np.uint16)) for _ in range(2))
        own.kv4_dequant(batch(lens), own.kv4_dequant_args(k.gpu_addr(), v.gpu_addr()))
        for rows in ([1, 1], [40, 30]):
            y = dev.up(np.zeros((sum(rows), 2 * heads, dim), np.uint16))
            own.kv4_attention(batch(rows), own.kv4_attention_args(rows_in.gpu_addr(), y.gpu_addr(), n_q_heads=2 * heads, scale=0.1))
            out.append((y, sum(rows) * wide))
        own.synchronize()
        got.append([b.read(2 * n, np.uint16) for b, n in out + [(k, sum(lens) * wide // 2), (v, sum(lens) * wide // 2)]])
    for a, b in zip(*got):
        assert a.any() and np.array_equal(a, b)
    dev.free()


def test_positions_outside_the_rope_table(t0, own):
    dev = Device(own)
    rng = np.random.default_rng(2)
    cache = ref.Cache(rng, [4, 9, 3], 1, 64, 16)
    before = cache.pool(0)
    pool, x, out = dev.up(before), dev.up(rng.standard_normal((3, 3, 64)).astype(np.float32)), dev.up(np.full((3, 64), 0xABCD, np.uint16))
    b = make_batch(t0, dev, cache, pool, [1, 1, 1], uniform=True)
    table = dev.up(rope_table(rng, 8, 32))                                # sequence 1 is at position 8
    at = x.gpu_addr()
    own.kv4_append(b, own.kv4_append_args(at + 256, at + 512, k_stride=192, v_stride=192, in_f32=True, q=at, q_stride=192, q_out=out.gpu_addr(), n_q_heads=1,
                                          rope=table.gpu_addr(), n_positions=8, rot_dim=64))
    bounds_error(t0, own, "row 1")
    got, after = out.read(3 * 128, np.uint16).reshape(3, 64), pool.read(before.size).reshape(before.shape)
    assert np.all(got[1] == 0xABCD) and not np.any(np.all(got[[0, 2]] == 0xABCD, 1))
    assert np.array_equal(after[cache.table[1, 0]], before[cache.table[1, 0]]) and not np.array_equal(after[cache.table[0, 0]], before[cache.table[0, 0]])
    own.synchronize()
    dev.free()


# --------------------------------------------------------------------------- recorded calls, other streams, the whole step

@pytest.mark.parametrize("rows, group", [(1, 4), (2, 2), (20, 4)])
def test_a_recorded_step_follows_the_lengths(t0, own, rows, group):
    # append, attention and read-out recorded once; the replay reads lengths, tables and rows as they are then
    own.synchronize()
    driver, dev = Driver(), Device(own)
    rng = np.random.default_rng(4)
    heads, dim, page, lens = 2, 128, 16, [700, 40, 30]
    cache = ref.Cache(rng, [n + 2 * rows for n in lens], heads, dim, page)
    total, hq = 3 * rows, heads * group
    pool, pool2 = dev.up(cache.pool(0)), dev.up(cache.pool(0))
    length = dev.up(np.array(lens, np.int32))
    table = dev.up(cache.table)
    x = [ref.bf16_bits(rng.standard_normal((total, hq + 2 * heads, dim)).astype(np.float32)) for _ in range(2)]
    data, rope = dev.up(x[0]), dev.up(rope_table(rng, 1000, 64))

    def step(p, src, to):
        b = own.kv4_batch(p.gpu_addr(), table.gpu_addr(), length.gpu_addr(), n_pages=cache.n_pages, page_size=page, n_kv_heads=heads, head_dim=dim, n_seqs=3,
                          table_stride=cache.stride, n_rows=total, max_rows=rows)
        at, wide = src.gpu_addr(), (hq + 2 * heads) * dim
        q, y, k, v = to
        own.kv4_append(b, own.kv4_append_args(at + hq * dim * 2, at + (hq + heads) * dim * 2, k_stride=wide, v_stride=wide, q=at, q_stride=wide, q_out=q.gpu_addr(),
                                              n_q_heads=hq, rope=rope.gpu_addr(), n_positions=1000, rot_dim=128))
        own.kv4_attention(b, own.kv4_attention_args(q.gpu_addr(), y.gpu_addr(), n_q_heads=hq, scale=0.1))
        own.kv4_dequant(b, own.kv4_dequant_args(k.gpu_addr(), v.gpu_addr()))

    outs = [[dev.up(np.zeros((total, w, dim), np.uint16)) for w in (hq, hq, heads, heads)] for _ in range(2)]
    with pytest.raises(t0.T0Error) as e:                                  # the buffer for parts is not there yet
        with driver.record(own):
            step(pool, data, outs[0])
    assert e.value.code == 6
    own.reserve_scratch("kv4", own.kv4_scratch_bytes())
    own.synchronize()
    with driver.record(own) as made:
        step(pool, data, outs[0])
    for turn in range(2):
        new = np.array(lens, np.int32) + (turn + 1) * rows
        if turn == 1:
            new[2] = 0
        length.write(new)
        data.write(x[turn])
        driver.replay(made[0], own.stream())
        step(pool2, data, outs[1])
        own.synchronize()
        for name, a, b, w in zip("qykv", *outs, (hq, hq, heads, heads)):
            a, b = (o.read(total * w * dim * 2, np.uint16).reshape(total, w, dim) for o in (a, b))
            assert a[:rows].any() and np.array_equal(a, b), (name, turn)
    n = cache.n_pages * t0.kv4_page_bytes(page, heads, dim)
    assert np.array_equal(pool.read(n), pool2.read(n))
    driver.drop(ex=made[0])
    dev.free()


def test_two_runtimes_at_once(t0, rt):
    # each has its own stream and its own buffer for parts
    other = t0.GpuRuntime(0)
    runs = []
    for r, seed in ((rt, 1), (other, 2)):
        dev = Device(r)
        rng = np.random.default_rng(seed)
        cache = ref.Cache(rng, [9000, 300], 1, 128, 64)
        q = ref.bf16_bits(rng.standard_normal((2, 8, 128)).astype(np.float32))
        b = make_batch(t0, dev, cache, dev.up(cache.pool()), [1, 1])
        ys = [dev.up(np.zeros_like(q)) for _ in range(30)]
        runs.append((r, dev, b, dev.up(q), ys, q))
        r.synchronize()
    for i in range(30):
        for r, dev, b, qb, ys, q in runs:
            r.kv4_attention(b, r.kv4_attention_args(qb.gpu_addr(), ys[i].gpu_addr(), n_q_heads=8, scale=0.1))
    for r, dev, b, qb, ys, q in runs:
        r.synchronize()
        first = ys[0].read(q.nbytes, np.uint16)
        assert first.any() and all(np.array_equal(y.read(q.nbytes, np.uint16), first) for y in ys)
        dev.free()
    other.close()


def test_a_layer_step_by_step(t0, rt, dev):
    # projections of four-bit weights, append, attention, output projection: as a program generates tokens, against the same steps in 64 bits
    rng = np.random.default_rng(11)
    heads, group, dim, page, seqs, hidden = 2, 2, 64, 16, 3, 256
    hq, wide = heads * group, (heads * group + 2 * heads) * dim
    def weights(k, n):
        packed = rng.integers(0, 2**32, (k // 8, n), dtype=np.uint32)
        scales = rng.uniform(0.005, 0.01, (k // 128, n)).astype(np.float32)
        zeros = np.full((k // 128, n // 8), 0x88888888, np.uint32)
        codes = np.stack([(packed >> np.uint32(4 * i)) & 15 for i in range(8)], 1).reshape(k, n).astype(np.float64)
        w = ref.bf16_round(((codes - 8) * np.repeat(ref.bf16_round(scales), 128, 0)).astype(np.float32)).astype(np.float64)
        args = [dev.up(a) for a in (packed, ref.bf16_bits(scales), zeros)]
        pre = rt.w4_prepack(*(a.gpu_addr() for a in args), k, n)
        dev.bufs.append(pre)
        return pre.gpu_addr(), w
    w_qkv, w_qkv64 = weights(hidden, wide)
    w_out, w_out64 = weights(hq * dim, hidden)
    cache = ref.Cache(rng, [20, 47, 16], heads, dim, page)                # room for four more tokens each
    start_lens = [15, 43, 11]
    k_held, v_held = [ref.held(k)[:n] for k, n in zip(cache.k, start_lens)], [ref.held(v)[:n] for v, n in zip(cache.v, start_lens)]
    pool, table, rope_np = dev.up(cache.pool()), dev.up(cache.table), rope_table(rng, 64, dim // 2)
    rope = dev.up(rope_np)
    qkv, q, y = dev.up(np.zeros((seqs, wide), np.float32)), dev.up(np.zeros((seqs, hq, dim), np.uint16)), dev.up(np.zeros((seqs, hq, dim), np.uint16))
    out, lens_buf = dev.up(np.zeros((seqs, hidden), np.float32)), dev.up(np.zeros(seqs, np.int32))
    for step in range(4):
        lens = [n + step + 1 for n in start_lens]
        lens_buf.write(np.array(lens, np.int32))
        x = ref.bf16_round(rng.standard_normal((seqs, hidden)).astype(np.float32))
        xb = dev.up(ref.bf16_bits(x))
        rt.w4a16_gemm_prepacked(xb.gpu_addr(), w_qkv, qkv.gpu_addr(), seqs, wide, hidden)
        b = rt.kv4_batch(pool.gpu_addr(), table.gpu_addr(), lens_buf.gpu_addr(), n_pages=cache.n_pages, page_size=page, n_kv_heads=heads, head_dim=dim, n_seqs=seqs,
                         table_stride=cache.stride, n_rows=seqs)
        at = qkv.gpu_addr()
        rt.kv4_append(b, rt.kv4_append_args(at + hq * dim * 4, at + (hq + heads) * dim * 4, k_stride=wide, v_stride=wide, in_f32=True, q=at, q_stride=wide,
                                            q_out=q.gpu_addr(), n_q_heads=hq, rope=rope.gpu_addr(), n_positions=64, rot_dim=dim))
        rt.kv4_attention(b, rt.kv4_attention_args(q.gpu_addr(), y.gpu_addr(), n_q_heads=hq, scale=dim**-0.5))
        rt.w4a16_gemm_prepacked(y.gpu_addr(), w_out, out.gpu_addr(), seqs, hidden, hq * dim)
        rt.synchronize()
        got_qkv = qkv.read(seqs * wide * 4, np.float32).reshape(seqs, hq + 2 * heads, dim)
        want_qkv = x.astype(np.float64) @ w_qkv64
        # f32 sums of exact bf16 products: 256 terms, each addition off by 2^-24 of the partial sums
        assert np.all(np.abs(got_qkv.reshape(seqs, -1) - want_qkv) <= 256 * 2.0**-24 * (np.abs(x).astype(np.float64) @ np.abs(w_qkv64)))
        cs = rope_np[np.array(lens) - 1]
        turned = ref.rotate(got_qkv[:, :hq + heads], cs, False)
        q64 = ref.bf16_round(turned[:, :hq]).astype(np.float64)
        got_y = ref.from_bits(y.read(seqs * hq * dim * 2, np.uint16)).reshape(seqs, hq, dim).astype(np.float64)
        for s in range(seqs):
            k_held[s] = np.concatenate([k_held[s], ref.held(turned[s:s + 1, hq:])])
            v_held[s] = np.concatenate([v_held[s], ref.held(got_qkv[s:s + 1, hq + heads:])])
            want, weight, reach = ref.attention(q64[s:s + 1], k_held[s], v_held[s], [lens[s] - 1], np.float64(np.float32(dim**-0.5)), 0)
            bound = ref.U * np.abs(want) + (2 * ref.U + np.expm1(2 * ref.U * reach))[..., None] * weight + 1e-5 * weight
            assert np.all(np.abs(got_y[s] - want[0]) <= bound[0]), (step, s)
        got_out = out.read(seqs * hidden * 4, np.float32).reshape(seqs, hidden)
        flat = got_y.reshape(seqs, -1)
        assert np.all(np.abs(got_out - flat @ w_out64) <= 256 * 2.0**-24 * (np.abs(flat) @ np.abs(w_out64)))
