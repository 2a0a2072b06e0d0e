"""Rows and products in eight bits at the ends of what the calls allow, against the restatement of tests/q8_reference.py."""
import ctypes

import numpy as np
import pytest

import q8_reference as ref
import test_q8_gpu as q8
from test_kernel_edges_gpu import run_gemm
from test_q8_gpu import dev, same  # noqa: F401  (dev is a fixture)
from test_recorded_launches_gpu import Driver

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------------- rows that are longer than shared memory

# rows and residual of f32, more rows than there are threads for at once: from dim 28168 on the two rows are longer than the shared memory that a ring has
@pytest.mark.parametrize("rows, dim, w_f32, outputs, place", [(297, 28160, False, "q", "residual"), (297, 28168, True, "qy", "residual"), (300, 32768, False, "q", "x"), (300, 32761, True, "qy", ""),
                                                              (301, 30001, False, "y", "nothing")])
def test_norms_of_the_longest_rows(t0, rt, dev, rows, dim, w_f32, outputs, place):  # noqa: F811
    q8.test_rmsnorm(t0, rt, dev, rows, dim, True, "f32", w_f32, outputs, place)

# --------------------------------------------------------------------------- errors

def test_an_error_is_one_calls_own(t0, rt, dev):  # noqa: F811
    # a launch that the runtime refuses (its stream is in a recording that was broken off) answers with the error; the call behind it, whose launch is fine, does not
    driver = Driver()
    x, q, s = dev.up(np.ones((4, 64), np.float32)), dev.up(np.zeros((4, 64), np.int8)), dev.up(np.zeros(4, np.float32))
    y, w = dev.up(np.zeros((4, 4), np.float32)), dev.up(np.ones((700, 64), np.int8))
    ws, big = dev.up(np.ones(700, np.float32)), dev.up(np.zeros((700, 700), np.float32))
    at = lambda b: b.gpu_addr()  # noqa: E731
    filled = rt.alloc(4096)
    size = dict(n_rows=4, dim=64)
    calls = [lambda: rt.q8_quant(rt.q8_quant_args(at(x), at(q), at(s), x_f32=True, **size)), lambda: rt.q8_dequant(rt.q8_dequant_args(at(q), at(s), at(x), out_f32=True, **size)),
             lambda: rt.q8_rmsnorm(rt.q8_rmsnorm_args(at(x), at(ws), eps=1e-5, x_f32=True, weight_f32=True, q=at(q), scales=at(s), **size)),
             lambda: rt.q8_gemm(rt.q8_gemm_args(at(q), at(s), at(w), at(ws), at(y), m=4, n=4, k=64)),
             lambda: rt.q8_gemm(rt.q8_gemm_args(at(w), at(ws), at(w), at(ws), at(big), m=700, n=700, k=64))]
    for call in calls:
        call()
        rt.synchronize()
        stream, graph = ctypes.c_void_p(rt.stream()), ctypes.c_void_p()
        driver.call("cuStreamBeginCapture_v2", stream, 1)                   # 1 = this thread's recording
        broken = driver.cu.cuStreamSynchronize(stream)                      # not allowed in a recording: breaks it off
        try:
            with pytest.raises(t0.T0Error) as e:
                call()
        finally:
            ended = driver.cu.cuStreamEndCapture(stream, ctypes.byref(graph))
        assert broken != 0 and ended != 0 and e.value.code == 2, (broken, ended, e.value.code)
        rt.fill_uniform_bf16(filled.gpu_addr(), 100, 1)
        call()
        rt.synchronize()
    with pytest.raises(t0.T0Error) as e:                                    # more memory than any GPU has
        rt.alloc(1 << 50)
    assert e.value.code == 2
    rt.fill_uniform_bf16(filled.gpu_addr(), 100, 1)
    rt.synchronize()
    filled.free()


# --------------------------------------------------------------------------- waits that run out

@pytest.mark.parametrize("rows, dim, norm", [(4801, 300, False), (1201, 1500, False), (605, 3001, False), (300, 8192, False), (299, 16384, False), (297, 20001, False), (4800, 500, True), (1200, 2000, True),
                                             (600, 4096, True), (300, 6000, True), (300, 8192, True), (301, 12288, True), (300, 16384, True), (297, 17000, True)])
def test_rows_whose_wait_runs_out_are_left(t0, rt, dev, rows, dim, norm):  # noqa: F811
    # The copy of row 0 is left out: the threads that wait for it give up after the limit, write nothing of it and no row behind it, and the call that synchronises says so.  The other blocks' rows are
    # as ever, and another runtime goes on.
    rng = np.random.default_rng(rows + dim)
    f32 = dim % 2 == 0
    x = rng.standard_normal((rows, dim)).astype(np.float32)
    x = x if f32 else ref.bf16_round(x)
    res = ref.bf16_round(rng.standard_normal((rows, dim)).astype(np.float32))
    weight = ref.bf16_round(rng.uniform(0.5, 1.5, dim).astype(np.float32))
    wide, q_wide = (dim + 7) // 8 * 8, q8.up16(dim)
    bx, bw = dev.up(q8.padded(x if f32 else ref.bf16_bits(x), wide, 0)), dev.up(ref.bf16_bits(weight))
    br = dev.up(q8.padded(ref.bf16_bits(res), wide, 0))
    bh, bq, bs, by = (dev.up(np.zeros(shape, kind)) for shape, kind in (((rows, wide), np.uint16), ((rows, q_wide), np.uint8), (rows, np.float32), ((rows, wide), np.uint16)))
    at = lambda b: b.gpu_addr()  # noqa: E731
    if norm:
        want_y, h = ref.rmsnorm(x, weight, 1e-5, res, True)
        want = [*ref.hold(want_y), ref.bf16_bits(want_y), ref.bf16_bits(h)]
    else:
        want = list(ref.hold(x))

    def run(r):
        for b, fill, kind in ((bh, 0xABCD, np.uint16), (bq, 0x5A, np.uint8), (bs, -7, np.float32), (by, 0xABCD, np.uint16)):
            b.write(np.full(rows * {2: wide, 1: q_wide, 4: 1}[kind().itemsize], fill, kind))
        rt.synchronize()
        if norm:
            r.q8_rmsnorm(r.q8_rmsnorm_args(at(bx), at(bw), n_rows=rows, dim=dim, eps=1e-5, x_f32=f32, x_stride=wide, residual=at(br), residual_stride=wide, residual_out=at(bh), residual_out_stride=wide,
                                           q=at(bq), scales=at(bs), y=at(by), y_stride=wide))
        else:
            r.q8_quant(r.q8_quant_args(at(bx), at(bq), at(bs), n_rows=rows, dim=dim, x_f32=f32, x_stride=wide))

    def read():
        got = [bq.read(rows * q_wide, np.int8).reshape(rows, -1)[:, :dim], bs.read(rows * 4, np.float32), by.read(rows * wide * 2, np.uint16).reshape(rows, -1)[:, :dim],
               bh.read(rows * wide * 2, np.uint16).reshape(rows, -1)[:, :dim]]
        return got[:len(want)]

    def rows_of(parts, others):
        return np.all([(a == b).reshape(rows, -1).all(1) for a, b in zip(parts, others)], axis=0)

    r = t0.GpuRuntime(0)
    run(r)
    r.synchronize()
    assert rows_of(read(), want).all()
    r.set_wait_limit_ns(3_000_000)
    r.selftest_drop_one_load()
    run(r)
    with pytest.raises(t0.T0Error) as e:
        r.synchronize()
    assert e.value.code == 4 and "wait expired" in str(e.value) and r.is_poisoned()
    got = read()
    right, untouched = rows_of(got, want), rows_of(got, [0x5A, -7, 0xABCD, 0xABCD])
    assert untouched[0] and (right | untouched).all() and right.sum() >= rows // 2
    with pytest.raises(t0.T0Error) as e:
        run(r)
    assert e.value.code == 3
    r.close()
    run(rt)
    rt.synchronize()
    assert rows_of(read(), want).all()


# --------------------------------------------------------------------------- gates far from zero

@pytest.mark.parametrize("m", [3, 600, 1000])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gates_far_below_zero(t0, rt, dev, m, bf16, act):  # noqa: F811
    # The sigmoid of the epilogues keeps its values down to 2^-128; times a large number of the other product they are ordinary numbers.  Gates of -0.7 * 127 .. 0.7 * 127 (gelu: through
    # 1.702 of them), each from one code, the other product 2^107.
    # The bound is the restatement's relative one, (14 + 11 |g|) 2^-24, and half a step of bf16; what it allows beside that where the sigmoid has no normal number is not granted here.
    n, k, slope = 255, 16, 1.702 if act == "gelu" else 1.0
    a, gate, up = np.zeros((m, k), np.int8), np.zeros((n, k), np.int8), np.zeros((n, k), np.int8)
    a[:, 0], gate[:, 0], up[:, 0] = 1, np.arange(n) - 127, 64
    one, gs, us = np.ones(m, np.float32), np.full(n, 0.7 / slope, np.float32), np.full(n, 2.0**101, np.float32)
    y = dev.up(np.zeros((m, n), np.uint16 if bf16 else np.float32))
    at = lambda v: dev.up(v).gpu_addr()  # noqa: E731
    rt.q8_gated(rt.q8_gated_args(at(a), at(one), at(gate), at(gs), at(up), at(us), y.gpu_addr(), m=m, n=n, k=k, activation=act, out_bf16=bf16))
    rt.synchronize()
    got = y.read(m * n * (2 if bf16 else 4), np.uint16 if bf16 else np.float32).reshape(m, n)
    got = (ref.from_bits(got) if bf16 else got).astype(np.float64)
    g = (np.arange(n) - 127) * gs.astype(np.float64)
    power = -g * slope * np.log2(np.e)                                       # the sigmoid is 1 / (1 + 2^power)
    want = g / (1 + np.exp2(power)) * 2.0**107
    bound = ((14 + 11 * np.abs(g)) * 2.0**-24 + (2.0**-8 if bf16 else 0)) * np.abs(want)
    kept = power < 128 * (1 - 2.0**-20)
    assert kept.sum() < n and (power[kept] > 126.5).any()                    # both sides of where it ends
    assert (np.abs(got - want) <= bound)[:, kept].all()
    assert ((np.abs(got - want) <= bound) | (got == 0))[:, ~kept].all()


@pytest.mark.parametrize("m", [1, 600, 1000])
@pytest.mark.parametrize("act, factor", [("silu", 1.0), ("gelu", 1.702)])
def test_gates_are_what_the_epilogues_compute(t0, rt, dev, m, act, factor):  # noqa: F811
    # rows of f32: the bits of the epilogue of the same name (its argument the bias of a product of zeros), whatever the argument; the other product is one
    rng = np.random.default_rng(8)
    edges = np.array([0.0, 87.2, 87.4, 88.0, 88.72, 88.73, 89.0, 103.0, 1e4, 3e38, np.inf, np.nan, 1e-30, 1e-40], np.float32) / np.float32(factor)
    v = np.concatenate([edges, rng.uniform(0, 110, 3000), rng.uniform(86, 90, 500) / factor, np.exp(rng.uniform(-80, 6, 500))]).astype(np.float32)
    n, k = 2 * v.size, 16
    sign = np.repeat(np.array([1, -1], np.int8), v.size)
    v = np.tile(v, 2)
    a, gate, up = np.zeros((m, k), np.int8), np.zeros((n, k), np.int8), np.zeros((n, k), np.int8)
    a[:, 0], gate[:, 0], up[:, 0] = 1, sign, 1
    y = dev.up(np.zeros((m, n), np.float32))
    at = lambda b: dev.up(b).gpu_addr()  # noqa: E731
    rt.q8_gated(rt.q8_gated_args(at(a), at(np.ones(m, np.float32)), at(gate), at(v), at(up), at(np.ones(n, np.float32)), y.gpu_addr(), m=m, n=n, k=k, activation=act, out_bf16=False))
    rt.synchronize()
    got = y.read(m * n * 4, np.float32).reshape(m, n)
    want = run_gemm(t0, rt, np.zeros((1, 64), np.float32), np.zeros((n, 64), np.float32), 1, n, 64, bias=v * sign, tile_epilogue=["bias", act])[0]
    assert all(q8.same(row, want) for row in got)


# --------------------------------------------------------------------------- roundings

def test_the_read_out_rounds_to_f32_and_then_to_bf16(t0, rt, dev):  # noqa: F811
    # products next to half way between two numbers of bf16, which are half way as f32: the second rounding goes to the even one, whichever side the product was on
    rng = np.random.default_rng(4)
    codes = rng.integers(1, 128, 400000).astype(np.int8)
    half_way = (2 * rng.integers(128, 256, codes.size) + 1).astype(np.float64)                 # nine bits, the last one set
    scales = (half_way / codes).astype(np.float32)
    exact = scales.astype(np.float64) * codes
    beside = (exact != half_way) & (exact.astype(np.float32) == half_way)
    codes, scales, exact, half_way = codes[beside], scales[beside], exact[beside], half_way[beside]
    once = np.where(exact > half_way, half_way + 1, half_way - 1)
    twice = ref.bf16_round(half_way.astype(np.float32))
    assert codes.size > 10000 and 0.3 < (once != twice).mean() < 0.7
    q = np.zeros((codes.size, 16), np.int8)
    q[:, 0] = codes
    y = dev.up(np.zeros((codes.size, 8), np.uint16))
    rt.q8_dequant(rt.q8_dequant_args(dev.up(q).gpu_addr(), dev.up(scales).gpu_addr(), y.gpu_addr(), n_rows=codes.size, dim=1, y_stride=8))
    rt.synchronize()
    assert np.array_equal(ref.from_bits(y.read(codes.size * 16, np.uint16)).reshape(-1, 8)[:, 0], twice)


def added(squares, threads, chunks):
    """A row's sum of squares as `threads` threads with `chunks` chunks of eight numbers add it in 64 bits."""
    x = squares.reshape(chunks, threads, 8)
    part = [np.zeros(threads) for _ in range(4)]
    for c in range(chunks):
        for i in range(8):
            part[i % 4] = part[i % 4] + x[c, :, i]
    s = ((part[0] + part[1]) + (part[2] + part[3])).reshape(-1, 32)
    for d in (16, 8, 4, 2, 1):
        s = s + s[:, np.arange(32) ^ d]
    four = [0.0] * 4
    for i, v in enumerate(s[:, 0]):
        four[i % 4] += v
    return (four[0] + four[1]) + (four[2] + four[3])


def test_a_norms_row_alone_and_among_many(t0, rt, dev):  # noqa: F811
    # A row is added up by 512 threads where rows are few and by 256 where they are many.  What comes of it is the same, but for rows whose root lies half way between two f32 as closely as 64 bits show:
    # there it may be the one or the other.  Row 0 is made one of those, by its eps.
    rng = np.random.default_rng(12)
    dim, many = 4096, 700
    while True:
        row = rng.standard_normal(dim).astype(np.float32)
        squares = row.astype(np.float64)**2
        sums = [added(squares, 512, 1), added(squares, 256, 2)]
        root = np.float32(1 / np.sqrt(sums[0] / dim))
        half_way = 1 / ((np.float64(root) + np.float64(np.nextafter(root, np.float32(0)))) / 2)**2         # the mean from which on the root is the next lower f32
        eps = half_way - sums[0] / dim
        if sums[0] != sums[1] and 2.0**-31 < eps < 2.0**-29:
            break
    x = np.vstack([row, rng.standard_normal((many - 1, dim)).astype(np.float32)])
    weight = rng.uniform(0.5, 1.5, dim).astype(np.float32)
    bx, bw = dev.up(x), dev.up(weight)
    for step in range(-3, 4):
        e = np.float32(eps) + step * np.spacing(np.float32(eps))
        got = []
        for n in (1, 7, many):
            q, s = dev.up(np.zeros((n, dim), np.int8)), dev.up(np.zeros(n, np.float32))
            rt.q8_rmsnorm(rt.q8_rmsnorm_args(bx.gpu_addr(), bw.gpu_addr(), n_rows=n, dim=dim, eps=float(e), x_f32=True, weight_f32=True, q=q.gpu_addr(), scales=s.gpu_addr()))
            rt.synchronize()
            got.append((q.read(n * dim, np.int8).reshape(n, dim), s.read(4 * n, np.float32)))
        assert np.array_equal(got[1][0][1:], got[2][0][1:7]) and same(got[1][1][1:], got[2][1][1:7])
        either = [ref.hold((row * r) * weight) for r in (root, np.nextafter(root, np.float32(0)))]
        for codes, scales in got:
            assert any(np.array_equal(codes[0], c) and scales[0] == w for c, w in either)


# --------------------------------------------------------------------------- scales that are no numbers, rows far apart

@pytest.mark.parametrize("m", [5, 600, 1000])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_gated_products_of_scales_that_are_no_numbers(t0, rt, dev, m, bf16, act):  # noqa: F811
    # tokens and channels of either matrix whose scales are zero, infinite and NaN: what the formula makes of them, and the others' numbers as ever.  (A row's
    # codes have one sign, so that no sum is zero.)
    rng = np.random.default_rng(6)
    n, k = 130, 64
    a, g, u = (rng.integers(1, 60, (rows, k)).astype(np.int8) * np.repeat(rng.choice([-2, 2], rows), k).reshape(rows, k).astype(np.int8) for rows in (m, n, n))
    a_scales, g_scales, u_scales = (np.exp(rng.uniform(-1, 1, rows)).astype(np.float32) * np.float32(s) for rows, s in ((m, 1e-3), (n, 1e-3), (n, 1.0)))
    a_scales[1:4] = 0, np.inf, np.nan
    g_scales[2:5] = u_scales[7:10] = 0, np.inf, np.nan
    y = dev.up(np.zeros((m, n), np.uint16 if bf16 else np.float32))
    at = lambda b: dev.up(b).gpu_addr()  # noqa: E731
    rt.q8_gated(rt.q8_gated_args(at(a), at(a_scales), at(g), at(g_scales), at(u), at(u_scales), y.gpu_addr(), m=m, n=n, k=k, activation=act, out_bf16=bf16))
    rt.synchronize()
    got = y.read(m * n * (2 if bf16 else 4), np.uint16 if bf16 else np.float32).reshape(m, n)
    got = (ref.from_bits(got) if bf16 else got).astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        gate, up = (((a.astype(np.float64) @ w.T.astype(np.float64)) * a_scales[:, None]) * s for w, s in ((g, g_scales), (u, u_scales)))
        if act == "relu":
            want = np.where(gate < 0, 0.0, gate) * up
        else:
            want = gate * (1 / (1 + np.exp(-gate * (1.702 if act == "gelu" else 1.0)))) * up
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(want).any() and np.isinf(want).any()
        ends = np.isinf(want)
        assert np.array_equal(got[ends], want[ends])
        fine = np.isfinite(want)
        # the restatement's bound; its relative part is zero where the value is, which 0 * infinity does not say (relu of minus infinity, times a finite number)
        relative = np.where(want == 0, 0, (14 + 11 * np.abs(gate)) * 2.0**-24 * np.abs(want))
        bound = relative + 2.0**-118 * np.abs(up) + 2.0**-140 + (2.0**-8 * np.abs(want) if bf16 else 0)
        assert (np.abs(got - want)[fine] <= bound[fine]).all()


class Far:
    """Rows `step` bytes apart in one buffer, several arrays beside one another in each step."""

    def __init__(self, rt, rows, step):
        self.rt, self.rows, self.step, self.used = rt, rows, step, 0
        self.buf = rt.alloc(rows * step)

    def put(self, data):
        at = self.used
        for i, row in enumerate(data):
            self.buf.write_bytes(i * self.step + at, np.ascontiguousarray(row))
        self.used += (data[0].nbytes + 255) // 256 * 256
        assert self.used <= self.step
        return at, self.buf.gpu_addr() + at

    def get(self, at, n, count, kind):
        return np.stack([self.buf.read_bytes(i * self.step + at, count * kind().itemsize, kind) for i in range(n)])


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("wide", [72, 75])
def test_products_on_pairs_of_rows_far_apart(t0, rt, dev, gated, wide):  # noqa: F811
    # offsets beyond 32 bits on CTA pairs, whose y goes out by copies (72 numbers a row) and row by row (75): rows of every array 8 MiB apart
    rng = np.random.default_rng(wide)
    m, n, k, step = 1700, wide, 200, 8 << 20
    far = Far(rt, m, step)
    a, g, u = (rng.integers(-127, 128, (rows, k)).astype(np.int8) for rows in (m, n, n))
    scales = [np.exp(rng.uniform(-1, 1, rows)).astype(np.float32) * np.float32(1e-2) for rows in (m, n, n)]
    (_, pa), (_, pg), (_, pu) = far.put(a), far.put(g), far.put(u)
    y_at, py = far.put(np.zeros((m, n + 4), np.float32))
    sa, sg, su = (dev.up(s).gpu_addr() for s in scales)
    strides = dict(m=m, n=n, k=k, a_stride=step, w_stride=step, y_stride=step // 4)
    if gated:
        rt.q8_gated(rt.q8_gated_args(pa, sa, pg, sg, pu, su, py, activation="relu", out_bf16=False, **strides))
        want = np.maximum(ref.product(a, scales[0], g, scales[1]), 0) * ref.product(a, scales[0], u, scales[2])
    else:
        rt.q8_gemm(rt.q8_gemm_args(pa, sa, pg, sg, py, **strides))
        want = ref.product(a, scales[0], g, scales[1])
    rt.synchronize()
    got = far.get(y_at, m, n + 4, np.float32)
    far.buf.free()
    assert same(got[:, :n].copy(), want) and (got[:, n:] == 0).all()


@pytest.mark.parametrize("rows, dim, step", [(6, 512, 1 << 30), (1300, 1500, 4 << 20), (300, 20000, 16 << 20)])
def test_norms_of_rows_far_apart(t0, rt, dev, rows, dim, step):  # noqa: F811
    # directly and with the ring: x, the residual in place, codes and bf16 rows, each beyond 32 bits
    rng = np.random.default_rng(dim)
    x, res = rng.standard_normal((rows, dim)).astype(np.float32), rng.standard_normal((rows, dim)).astype(np.float32)
    weight = rng.uniform(0.5, 1.5, dim).astype(np.float32)
    far = Far(rt, rows, step)
    _, px = far.put(x)
    r_at, pr = far.put(res)
    q_at, pq = far.put(np.zeros((rows, q8.up16(dim)), np.int8))
    y_at, py = far.put(np.zeros((rows, dim + 8), np.uint16))
    s = dev.up(np.zeros(rows, np.float32))
    rt.q8_rmsnorm(rt.q8_rmsnorm_args(px, dev.up(weight).gpu_addr(), n_rows=rows, dim=dim, eps=1e-5, x_f32=True, weight_f32=True, residual=pr, residual_out=pr, residual_f32=True, q=pq,
                                     scales=s.gpu_addr(), y=py, x_stride=step // 4, residual_stride=step // 4, residual_out_stride=step // 4, q_stride=step, y_stride=step // 2))
    rt.synchronize()
    want, h = ref.rmsnorm(x, weight, 1e-5, res, False)
    codes, scales = ref.hold(want)
    got = [far.get(r_at, rows, dim, np.float32), far.get(q_at, rows, dim, np.int8), far.get(y_at, rows, dim, np.uint16)]
    far.buf.free()
    assert same(got[0], h) and np.array_equal(got[1], codes) and np.array_equal(got[2], ref.bf16_bits(want)) and same(s.read(4 * rows, np.float32), scales)
