"""Attention over the four-bit cache on the GPU, held to the roundings that each kernel makes (tests/kv4_bounds.py; tests/test_kv4_bounds.py shows that results which lost a part, took a
neighbour's place or have a mask off by one are over these bounds).  The numbers at the far ends of the types are here too."""
import numpy as np
import pytest

import kv4_bounds as kb
import kv4_reference as ref
from test_kv4_gpu import Device, bounds_error, dev, make_batch, own, rope_table  # noqa: F401  (fixtures)
from test_recorded_launches_gpu import Driver

pytestmark = pytest.mark.gpu


def cache_of(rng, k, v, page, copies=1):
    """A cache of one sequence with these keys and values, `copies` of it on the same pages."""
    cache = ref.Cache(rng, [k.shape[0]], k.shape[1], k.shape[2], page)
    cache.k, cache.v = [k], [v]
    pool = cache.pool()
    cache.lens, cache.table = cache.lens * copies, np.repeat(cache.table, copies, 0)
    return cache, pool


def attend(t0, dev, b, q, scale, window=0):  # noqa: F811
    """q [rows, heads, dim] -> y, f64."""
    rt = dev.rt
    bits = ref.bf16_bits(q.astype(np.float32))
    qb, y = dev.up(bits), dev.up(np.full(bits.shape, 0xABCD, np.uint16))
    rt.kv4_attention(b, rt.kv4_attention_args(qb.gpu_addr(), y.gpu_addr(), n_q_heads=q.shape[1], scale=scale, window=window))
    rt.synchronize()
    return ref.from_bits(y.read(bits.nbytes, np.uint16)).reshape(q.shape).astype(np.float64)


def held_to(t0, dev, k, v, page, q, scale, window=0, whole_q=True):  # noqa: F811
    n, rows = k.shape[0], q.shape[0]
    cache, pool = cache_of(np.random.default_rng(n), k, v, page)
    got = attend(t0, dev, make_batch(t0, dev, cache, dev.up(pool), [rows], uniform=True), q, scale, window)
    e = kb.Exact(q, k, v, np.arange(n - rows, n), np.float64(np.float32(scale)), window, whole_q)
    over = e.over(got)
    assert over.max() <= 0, f"row {np.argmax(over)} is {over.max()} over its bound"


@pytest.mark.parametrize("case", kb.LONG)
def test_every_run_of_a_long_sequence_counts(t0, rt, dev, case):  # noqa: F811
    k, v, _, qs, scale = kb.long_case(*case)
    for q in qs:
        held_to(t0, dev, k, v, case[5], q, scale)


@pytest.mark.parametrize("case", kb.EDGES)
def test_rows_see_what_the_mask_leaves_and_no_more(t0, rt, dev, case):  # noqa: F811
    k, v, q, scale = kb.edge_case(*case)
    held_to(t0, dev, k, v, case[5], q, scale, case[6])


@pytest.mark.parametrize("case", kb.RANDOM)
def test_random_scores(t0, rt, dev, case):  # noqa: F811
    k, v, q, scale = kb.random_case(*case)
    held_to(t0, dev, k, v, case[5], q, scale, whole_q=False)


@pytest.mark.parametrize("rows, copies", [(1, 2000), (2, 1), (20, 1), (20, 40)])
@pytest.mark.parametrize("size", [3e38, 1e36])
def test_values_near_the_end_of_the_range(t0, rt, dev, rows, copies, size):  # noqa: F811
    # the token with such values comes behind others and has 2^6.5 times their weights: less than what moves the maximum that weights are taken against.  (Many copies: several chunks of the
    # sequence are one warp's work.)
    rng = np.random.default_rng(22)
    n, dim, at = 200, 64, 150 if rows <= 16 else 100
    k, v = np.zeros((n, 1, dim), np.float32), rng.standard_normal((n, 1, dim)).astype(np.float32)
    k[at, 0, 0] = 4.5
    v[at, 0] = np.where(rng.integers(0, 2, dim), 0.49, -0.49) * size
    q = np.zeros((rows, 1, dim))
    q[:, :, 0] = 1.0
    cache, pool = cache_of(rng, k, v, 16, copies)
    got = attend(t0, dev, make_batch(t0, dev, cache, dev.up(pool), [rows] * copies, uniform=True), np.tile(q, (copies, 1, 1)), 1.0)
    e = kb.Exact(q, k, v, np.arange(n - rows, n), 1.0, 0, True)
    for y in got.reshape(copies, rows, 1, dim):
        assert e.over(y).max() <= 0


@pytest.mark.parametrize("dim, page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("what", ["k", "v"])
def test_a_number_beyond_bf16_stays_out_of_rows_that_do_not_see_it(t0, rt, dev, dim, page, what):  # noqa: F811
    # step 2.28e37, low -1.73e36: the top code's value, 3.397e38, is a number in f32 and rounds to an infinity in bf16.  Nothing of it may reach rows before the token; rows that see it get
    # their share, and a token of the same chunk that is NaN stays one.
    rng = np.random.default_rng(21)
    n, rows, at, bad = 150, 60, 120, 140
    k, v = (rng.standard_normal((n, 1, dim)).astype(np.float32) for _ in range(2))
    x = k if what == "k" else v
    x[at] = 0.0
    x[at, 0, :2] = 3.376e38, -1.72e36
    assert np.isinf(kb.bf16_once(ref.held(x[at]))).any() and np.isfinite(ref.held(x[at])).all()
    q = ref.bf16_round(rng.standard_normal((rows, 4, dim)).astype(np.float32)).astype(np.float64)
    if what == "k":
        q = np.copysign(2.0**-124, q)                                       # scores of the size of one at that token, of nothing at the others
    spoilt = x.copy()
    spoilt[bad, 0, 3] = np.nan
    cache, pool = cache_of(rng, spoilt if what == "k" else k, spoilt if what == "v" else v, page)
    got = attend(t0, dev, make_batch(t0, dev, cache, dev.up(pool), [rows], uniform=True), q, 0.125)
    tokens = np.arange(n - rows, n)
    e = kb.Exact(q, k, v, tokens, 0.125, 0, True)
    assert e.over(got)[tokens < bad].max() <= 0 and np.isnan(got[tokens >= bad]).all()


def test_the_read_out_rounds_once(t0, rt, dev):  # noqa: F811
    # rows whose least number is next to zero: step * code + low lies beside the middle of two bf16 numbers, by less than an f32 shows
    rng = np.random.default_rng(23)
    n, dim, page = 4096, 64, 64
    x = np.abs(rng.standard_normal((n, 1, dim))).astype(np.float32) * 10
    x[:, 0, 0] = 2.0**-rng.integers(18, 40, n)
    x = ref.bf16_round(x)
    x[0, 0, 0], x[0, 0, 1], x[0, 0, 2:] = 2.0**-30, 15.234375, 5.078125
    cache, pool = cache_of(rng, x, x[::-1].copy(), page)
    b = make_batch(t0, dev, cache, dev.up(pool), [n], uniform=True)
    out = [dev.up(np.zeros((n, dim), np.uint16)) for _ in range(2)]
    rt.kv4_dequant(b, rt.kv4_dequant_args(*(o.gpu_addr() for o in out)))
    rt.synchronize()
    want = kb.bf16_once(ref.held(x)[:, 0])
    assert want[0, 5] == 5.09375 and (want != ref.bf16_round(ref.held(x)[:, 0].astype(np.float32))).sum() > 1000
    for o, w in zip(out, (want, want[::-1])):
        assert np.array_equal(ref.from_bits(o.read(2 * n * dim, np.uint16)).reshape(n, dim), w)


@pytest.mark.parametrize("n, rows, group", [(40, 1, 1), (3000, 1, 4), (3000, 4, 4), (100, 30, 4), (5000, 30, 4), (5000, 20, 1)])
def test_scores_that_are_all_minus_infinity_give_nan(t0, rt, dev, n, rows, group):  # noqa: F811
    # what the formula gives, and no zeros, which stand for rows without tokens
    rng = np.random.default_rng(24)
    dim = 128
    k = 100 + rng.uniform(0, 0.1, (n, 1, dim)).astype(np.float32)
    q = np.zeros((rows, group, dim))
    q[:, 0, 5] = -np.inf
    cache, pool = cache_of(rng, k, rng.standard_normal((n, 1, dim)).astype(np.float32), 64)
    got = attend(t0, dev, make_batch(t0, dev, cache, dev.up(pool), [rows], uniform=True), q, 1.0)
    assert np.isnan(got[:, 0]).all() and np.isfinite(got[:, 1:]).all()
    short, pool = cache_of(rng, k[:3], k[:3], 64)                           # three tokens: rows before the first are zeros, whatever the queries are
    got = attend(t0, dev, make_batch(t0, dev, short, dev.up(pool), [rows], uniform=True), q, 1.0)
    assert np.all(got[:max(rows - 3, 0)] == 0) and np.isnan(got[max(rows - 3, 0):, 0]).all()


@pytest.mark.parametrize("dim, page", [(128, 64), (64, 16)])
def test_a_recorded_batch_of_both_kinds_reads_what_the_append_before_it_wrote(t0, own, dim, page):  # noqa: F811
    # append and attention recorded together, single tokens and chunks of prompts in one batch: each replay has other rows, pages, lengths and places of the rows, and is compared with
    # the same calls with a wait between them
    driver, dev = Driver(), Device(own)  # noqa: F811
    rng = np.random.default_rng(31)
    heads, group, seqs, places = 2, 4, 12, 900
    hq, total, most = heads * group, 600, 300
    wide = (hq + 2 * heads) * dim
    columns = -(-places // page)
    n_pages = seqs * columns
    bytes_of = n_pages * t0.kv4_page_bytes(page, heads, dim)
    first = np.zeros(bytes_of, np.uint8)
    pools, ys, qs = ([dev.up(np.zeros(shape, kind)) for _ in range(2)] for shape, kind in (((bytes_of,), np.uint8), ((total, hq, dim), np.uint16), ((total, hq, dim), np.uint16)))
    table, lens, start = dev.up(np.zeros((seqs, columns), np.int32)), dev.up(np.zeros(seqs, np.int32)), dev.up(np.zeros(seqs + 1, np.int32))
    data, rope = dev.up(np.zeros((total, hq + 2 * heads, dim), np.uint16)), dev.up(rope_table(rng, places, dim // 2))

    def calls(i, between):
        b = own.kv4_batch(pools[i].gpu_addr(), table.gpu_addr(), lens.gpu_addr(), n_pages=n_pages, page_size=page, n_kv_heads=heads, head_dim=dim, n_seqs=seqs,
                          table_stride=columns, n_rows=total, max_rows=most, row_start=start.gpu_addr())
        at = data.gpu_addr()
        own.kv4_append(b, own.kv4_append_args(at + hq * dim * 2, at + (hq + heads) * dim * 2, k_stride=wide, v_stride=wide, q=at, q_stride=wide, q_out=qs[i].gpu_addr(),
                                              n_q_heads=hq, rope=rope.gpu_addr(), n_positions=places, rot_dim=dim))
        between()
        own.kv4_attention(b, own.kv4_attention_args(qs[i].gpu_addr(), ys[i].gpu_addr(), n_q_heads=hq, scale=dim**-0.5))

    own.reserve_scratch("kv4", own.kv4_scratch_bytes())
    own.synchronize()
    with driver.record(own) as made:
        calls(0, lambda: None)
    for turn in range(24):
        rows = np.ones(seqs, int)
        for s in rng.permutation(seqs)[:3]:
            rows[s] = rng.integers(5, most if turn % 2 else 60)
        rows[rng.integers(0, seqs)] = 0
        rows = np.where(np.cumsum(rows) > total, 0, rows)
        lens.write(np.array([rng.integers(max(r, 1), places + 1) for r in rows], np.int32))
        start.write(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32))
        table.write(rng.permutation(n_pages).reshape(seqs, columns).astype(np.int32))
        data.write(ref.bf16_bits(rng.standard_normal((total, hq + 2 * heads, dim)).astype(np.float32)))
        for p in pools:                                                     # what lies before the rows: zeros, the same in both
            p.write(first)
        own.synchronize()
        driver.replay(made[0], own.stream())
        own.synchronize()
        calls(1, own.synchronize)
        own.synchronize()
        got = [y.read(total * hq * dim * 2, np.uint16).reshape(total, -1) for y in ys]
        assert got[0][:rows.sum()].any(1).all() and np.array_equal(*got), turn
        assert np.array_equal(*(p.read(bytes_of) for p in pools)), turn
    driver.drop(ex=made[0])
    dev.free()
