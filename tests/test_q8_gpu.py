"""Products in eight bits and the calls around them on the GPU, against the restatement of tests/q8_reference.py.

Codes, scales, the norm's rows and sums, the read-out and the products are compared bit for bit: they are defined operation by operation, and the integer sums are exact.  The gated
product is held to the bound that the restatement derives, plus half a step of bf16 (2^-8 of the value) where the rows are bf16."""
import numpy as np
import pytest

import q8_reference as ref
from test_kv4_gpu import Device
from test_recorded_launches_gpu import Driver

pytestmark = pytest.mark.gpu

NAN = 0x7FC0


@pytest.fixture()
def dev(rt):
    d = Device(rt)
    yield d
    rt.synchronize()
    d.free()


def padded(rows, stride, fill):
    """Rows with `fill` between their ends and the stride."""
    out = np.full((rows.shape[0], stride), fill, rows.dtype)
    out[:, :rows.shape[1]] = rows
    return out


def up16(n):
    return (n + 15) // 16 * 16


def same(got, want):
    """Equal bits, any NaN for a NaN."""
    got, want = np.asarray(got), np.asarray(want)
    assert got.dtype == want.dtype and got.shape == want.shape
    if got.dtype == np.float32:
        return bool(((got.view(np.uint32) == want.view(np.uint32)) | (np.isnan(got) & np.isnan(want)) | ((got == 0) & (want == 0))).all())
    return bool((got == want).all())


def same_bf16(got, want):
    got, want = np.asarray(got), np.asarray(want)
    nan = lambda b: (b & 0x7FFF) > 0x7F80  # noqa: E731
    return bool(((got == want) | (nan(got) & nan(want)) | (((got | want) & 0x7FFF) == 0)).all())


def trouble(x):
    """Rows that eight bits have trouble with, in place of the first ones of x."""
    n, dim = x.shape
    rows = [lambda r: r.fill(0), lambda r: r.__setitem__(dim // 2, np.inf), lambda r: r.__setitem__(dim - 1, np.nan), lambda r: r.__setitem__(0, -np.inf),
            lambda r: r.__imul__(np.float32(1e-38)), lambda r: r.__imul__(np.float32(1e37)), lambda r: r.fill(-1.25),
            lambda r: r.__setitem__(slice(None), (np.arange(dim) % 255 - 127) / 2.0)]
    for row, make in zip(x, rows):
        make(row)
    return x


# --------------------------------------------------------------------------- rows

ROWS = [
    # rows, dim, f32
    (1, 1, True), (1, 7, False), (3, 8, False), (9, 64, True), (17, 100, False), (8, 1023, True), (33, 1024, False), (5, 1025, True), (6, 2048, False), (12, 2049, True),
    (150, 4096, False), (7, 4099, True), (3, 8192, True), (11, 8200, False), (2, 11008, True), (9, 14336, False), (8, 16385, False), (9, 28672, True), (1, 32768, False), (300, 32, True),
    # enough rows for the ring
    (4801, 300, False), (4740, 512, True), (2400, 1000, True), (2371, 1024, False), (1201, 1500, False), (1190, 2048, True), (610, 4096, False), (605, 3001, True), (300, 8192, False), (303, 5003, True),
    (300, 12000, True), (299, 16384, False), (297, 20001, False), (298, 32768, True),
]


@pytest.mark.parametrize("rows, dim, f32", ROWS)
def test_quant_and_dequant(t0, rt, dev, rows, dim, f32):
    rng = np.random.default_rng(rows * 7 + dim)
    x = (rng.standard_normal((rows, dim)) * np.exp(rng.uniform(-5, 5, (rows, 1)))).astype(np.float32)
    if rows >= 8:
        trouble(x)
    if not f32:
        x = ref.bf16_round(x)
    x_stride, q_stride, extra = (dim + 7) // 8 * 8 + 8, up16(dim) + 16, 2
    data = padded(x if f32 else ref.bf16_bits(x), x_stride, np.nan if f32 else NAN)
    q = dev.up(np.full((rows + extra, q_stride), 0x5A, np.uint8))
    scales = dev.up(np.full(rows + extra, -7.0, np.float32))
    at = dev.up(data).gpu_addr()
    rt.q8_quant(rt.q8_quant_args(at, q.gpu_addr(), scales.gpu_addr(), n_rows=rows, dim=dim, x_f32=f32, x_stride=x_stride, q_stride=q_stride))
    outs = []
    for out_f32 in (True, False):
        y_stride = (dim + 7) // 8 * 8 + 16
        y = dev.up(np.full((rows + extra, y_stride), 0xABCD, np.uint32 if out_f32 else np.uint16))
        rt.q8_dequant(rt.q8_dequant_args(q.gpu_addr(), scales.gpu_addr(), y.gpu_addr(), n_rows=rows, dim=dim, out_f32=out_f32, q_stride=q_stride, y_stride=y_stride))
        outs.append((y, y_stride))
    rt.synchronize()
    codes, want_scales = ref.hold(x)
    got = q.read((rows + extra) * q_stride, np.int8).reshape(rows + extra, q_stride)
    want = np.full_like(got, 0x5A)
    want[:rows, :dim] = codes
    assert np.array_equal(got, want)
    assert same(scales.read(4 * (rows + extra), np.float32), np.concatenate([want_scales, np.full(extra, -7, np.float32)]))
    back = codes.astype(np.float32) * want_scales[:, None]
    for (y, y_stride), bits in zip(outs, (back.view(np.uint32), ref.bf16_bits(np.where(np.isnan(back), 0, back)))):
        got = y.read((rows + extra) * y_stride * bits.itemsize, bits.dtype).reshape(rows + extra, y_stride)
        assert (got[rows:] == 0xABCD).all() and (got[:, dim:] == 0xABCD).all()
        got = got[:rows, :dim]
        if bits.itemsize == 4:
            assert same(got.copy().view(np.float32), back)
        else:
            nan = np.isnan(back)
            assert same_bf16(np.where(nan, 0, got), np.where(nan, 0, bits)) and ((got[nan] & 0x7FFF) > 0x7F80).all()


@pytest.mark.parametrize("f32", [True, False])
def test_a_long_quant_is_exact(t0, rt, dev, f32):
    # four million numbers: an operation that is not rounded by itself shows in some of them (codes half way between two)
    rng = np.random.default_rng(78)
    rows, dim = 1024, 4096
    x = rng.standard_normal((rows, dim)).astype(np.float32)
    x = x if f32 else ref.bf16_round(x)
    q, scales = dev.up(np.zeros((rows, dim), np.int8)), dev.up(np.zeros(rows, np.float32))
    rt.q8_quant(rt.q8_quant_args(dev.up(x if f32 else ref.bf16_bits(x)).gpu_addr(), q.gpu_addr(), scales.gpu_addr(), n_rows=rows, dim=dim, x_f32=f32))
    rt.synchronize()
    codes, want = ref.hold(x)
    assert np.array_equal(q.read(rows * dim, np.int8).reshape(rows, dim), codes) and same(scales.read(4 * rows, np.float32), want)


def test_dequant_of_long_rows(t0, rt, dev):
    rng = np.random.default_rng(3)
    codes, scales = rng.integers(-128, 128, (2, 131071)).astype(np.int8), np.array([0.5, -3e-3], np.float32)
    y = dev.up(np.zeros((2, 131072), np.float32))
    rt.q8_dequant(rt.q8_dequant_args(dev.up(padded(codes, 131072, 0)).gpu_addr(), dev.up(scales).gpu_addr(), y.gpu_addr(), n_rows=2, dim=131071, out_f32=True, y_stride=131072))
    rt.synchronize()
    got = y.read(2 * 131072 * 4, np.float32).reshape(2, -1)
    assert same(got[:, :131071].copy(), codes.astype(np.float32) * scales[:, None]) and (got[:, 131071] == 0).all()


NORMS = [
    # rows, dim, x f32, residual (None, "bf16", "f32"), weight f32, outputs, in place
    (1, 4096, True, "bf16", False, "q", "residual"), (1, 1, False, None, True, "qy", ""), (2, 9, True, "f32", True, "qy", ""), (300, 64, False, "bf16", False, "q", "residual"),
    (20, 129, True, None, False, "y", ""), (9, 1000, False, "f32", False, "qy", "residual"), (9, 1024, True, "f32", False, "qy", "x"), (5, 2050, False, "bf16", True, "qy", "x"),
    (40, 4096, False, "bf16", False, "qy", ""), (8, 8191, True, "bf16", True, "q", ""), (8, 11008, False, None, False, "q", ""), (3, 16384, True, "f32", False, "y", ""),
    (8, 20001, False, "bf16", False, "qy", "residual"), (2, 32768, True, None, True, "q", ""), (700, 2048, False, "bf16", False, "q", "nothing"),
    (4800, 500, True, "bf16", False, "qy", "residual"), (4737, 512, True, "f32", True, "q", "x"), (2500, 1021, False, "bf16", False, "q", "residual"), (1200, 2000, True, "f32", False, "qy", "x"),
    (1187, 2048, False, None, False, "y", ""), (600, 4096, True, "bf16", False, "q", "residual"), (610, 3001, False, "f32", True, "qy", ""), (298, 8192, False, "bf16", False, "q", "residual"),
    (300, 5000, True, "f32", False, "q", "residual"), (300, 16384, True, "bf16", True, "q", "residual"), (297, 9999, False, None, False, "qy", ""), (297, 32768, False, "bf16", False, "q", "residual"),
    (298, 17000, True, "f32", False, "y", ""), (299, 6144, False, "bf16", False, "q", "residual"), (300, 6000, True, "f32", True, "qy", "x"), (301, 12288, False, "bf16", True, "q", ""),
    (298, 10001, True, None, False, "q", ""),
]


@pytest.mark.parametrize("rows, dim, f32, residual, w_f32, outputs, place", NORMS)
def test_rmsnorm(t0, rt, dev, rows, dim, f32, residual, w_f32, outputs, place):
    rng = np.random.default_rng(rows + 3 * dim)
    x = (rng.standard_normal((rows, dim)) * np.exp(rng.uniform(-3, 3, (rows, 1)))).astype(np.float32)
    if rows >= 8:
        trouble(x)
    x = x if f32 else ref.bf16_round(x)
    weight = rng.uniform(0.2, 2, dim).astype(np.float32)
    weight = weight if w_f32 else ref.bf16_round(weight)
    stride = (dim + 7) // 8 * 8 + 8
    hold_rows = lambda v, wide: dev.up(padded(v if wide else ref.bf16_bits(v), stride, np.float32(-9) if wide else 0xC110))  # noqa: E731
    bx = hold_rows(x, f32)
    r_f32, res, kw = residual == "f32", None, {}
    if residual:
        res = (rng.standard_normal((rows, dim)) * 2).astype(np.float32)
        res = res if r_f32 else ref.bf16_round(res)
        br = hold_rows(res, r_f32)
        kept = {"residual": br, "x": bx, "": hold_rows(np.zeros_like(res), r_f32), "nothing": None}[place]
        kw = dict(residual=br.gpu_addr(), residual_stride=stride, residual_f32=r_f32)
        if kept:
            kw.update(residual_out=kept.gpu_addr(), residual_out_stride=stride)
    q_stride = up16(dim)
    q, scales = dev.up(np.full((rows, q_stride), 0x5A, np.uint8)), dev.up(np.zeros(rows, np.float32))
    y = dev.up(np.full((rows, stride), 0xABCD, np.uint16))
    if "q" in outputs:
        kw.update(q=q.gpu_addr(), scales=scales.gpu_addr())
    if "y" in outputs:
        kw.update(y=y.gpu_addr(), y_stride=stride)
    wb = dev.up(weight if w_f32 else ref.bf16_bits(weight))
    rt.q8_rmsnorm(rt.q8_rmsnorm_args(bx.gpu_addr(), wb.gpu_addr(), n_rows=rows, dim=dim, eps=1e-5, x_f32=f32, weight_f32=w_f32, x_stride=stride, **kw))
    rt.synchronize()
    want_y, h = ref.rmsnorm(x, weight, 1e-5, res, not r_f32)
    if residual and kept:
        size = 4 if r_f32 else 2
        got = kept.read(rows * stride * size, np.float32 if r_f32 else np.uint16).reshape(rows, stride)
        assert (got[:, dim:] == (np.float32(-9) if r_f32 else 0xC110)).all()
        got = got[:, :dim].copy()
        assert same(got, h) if r_f32 else same(ref.from_bits(got), h)
    if "y" in outputs:
        got = y.read(rows * stride * 2, np.uint16).reshape(rows, stride)
        assert (got[:, dim:] == 0xABCD).all()
        assert same(ref.from_bits(got[:, :dim].copy()), np.where(np.isnan(want_y), np.float32(np.nan), ref.bf16_round(np.where(np.isnan(want_y), 0, want_y))))
    else:
        assert (y.read(rows * stride * 2, np.uint16) == 0xABCD).all()
    got = q.read(rows * q_stride, np.int8).reshape(rows, q_stride)
    if "q" in outputs:
        codes, want_scales = ref.hold(want_y)
        assert np.array_equal(got[:, :dim], codes) and (got[:, dim:] == 0x5A).all()
        assert same(scales.read(4 * rows, np.float32), want_scales)
    else:
        assert (got == 0x5A).all()


def test_rmsnorm_with_no_eps_and_a_row_of_zeros(t0, rt, dev):
    # 1 / sqrt(0): the row is NaN, the one beside it is not
    x = np.zeros((2, 64), np.float32)
    x[1] = np.arange(64)
    q, scales = dev.up(np.ones((2, 64), np.int8)), dev.up(np.zeros(2, np.float32))
    rt.q8_rmsnorm(rt.q8_rmsnorm_args(dev.up(x).gpu_addr(), dev.up(np.ones(64, np.float32)).gpu_addr(), n_rows=2, dim=64, eps=0.0, x_f32=True, weight_f32=True, q=q.gpu_addr(),
                                     scales=scales.gpu_addr()))
    rt.synchronize()
    y, _ = ref.rmsnorm(x, np.ones(64), 0.0)
    assert np.array_equal(q.read(128, np.int8).reshape(2, 64), ref.hold(y)[0]) and same(scales.read(8, np.float32), ref.hold(y)[1])


# --------------------------------------------------------------------------- products

def rows8(rng, dev, n, k, stride, all_codes=False):
    """Codes, scales and their buffers; what lies between the rows' ends and the stride is not zero."""
    codes = rng.integers(-128 if all_codes else -127, 128, (n, k)).astype(np.int8)
    scales = np.exp(rng.uniform(-4, 4, n)).astype(np.float32)
    return codes, scales, dev.up(padded(codes, stride, 77)), dev.up(scales)


def out_rows(dev, m, n, y_stride, bf16, shift):
    """A buffer for m rows and two behind them, `shift` numbers into it."""
    kind = np.uint16 if bf16 else np.uint32
    buf = dev.up(np.full((m + 2) * y_stride + shift, 0xABCD, kind))
    return buf, buf.gpu_addr() + shift * kind().itemsize


def read_rows(buf, m, n, y_stride, bf16, shift):
    """The rows' bits; everything around them is as it was."""
    kind = np.uint16 if bf16 else np.uint32
    all_ = buf.read(((m + 2) * y_stride + shift) * kind().itemsize, kind)
    assert (all_[:shift] == 0xABCD).all()
    grid = all_[shift:].reshape(m + 2, y_stride)
    assert (grid[m:] == 0xABCD).all() and (grid[:, n:] == 0xABCD).all()
    return grid[:m, :n].copy()


# both sides of every bound between kernels, tiles and splits, and sizes that are no multiple of anything
PRODUCTS = [
    (1, 1, 1), (1, 8, 16), (1, 4096, 4096), (1, 11008, 512), (2, 33, 31), (3, 130, 129), (5, 1000, 1357), (7, 20001, 256), (8, 128, 128), (9, 148, 640), (15, 4097, 1000), (16, 4096, 2048),
    (17, 300, 384), (31, 2000, 4096), (32, 128, 8192), (33, 512, 511), (64, 4096, 4096), (65, 777, 1025), (100, 1500, 768), (127, 129, 127), (128, 4096, 1024), (129, 640, 2000),
    (200, 3000, 300), (255, 257, 4096), (256, 1024, 1024), (257, 2049, 640), (300, 5000, 129), (512, 512, 4096), (600, 600, 600), (777, 1111, 1357), (1000, 4096, 256), (1024, 1024, 1024),
    (1500, 2300, 1100), (2048, 4096, 512), (4100, 260, 1024), (300, 20000, 256), (2, 5, 131071), (2100, 1001, 300), (2101, 1003, 300), (2100, 1000, 301), (2500, 999, 127),
]


@pytest.mark.parametrize("m, n, k", PRODUCTS)
def test_products_bit_for_bit(t0, rt, dev, m, n, k):
    rng = np.random.default_rng(m + 3 * n + 7 * k)
    bf16, with_bias, dense = (m + n) % 2 == 0, (m + k) % 3 == 0, (n + k) % 2 == 0
    a_stride, w_stride = up16(k) + (0 if dense else 32), up16(k) + (0 if dense else 16)
    a, a_scales, ab, asb = rows8(rng, dev, m, k, a_stride, True)
    w, w_scales, wb, wsb = rows8(rng, dev, n, k, w_stride, True)
    y_stride, shift = (n, 0) if dense else [(n + 5, 3), (up16(n) + 16, 8)][k % 2]     # the second: rows on 16-byte boundaries
    y, at = out_rows(dev, m, n, y_stride, bf16, shift)
    bias = (rng.standard_normal(n) * 1000).astype(np.float32) if with_bias else None
    rt.q8_gemm(rt.q8_gemm_args(ab.gpu_addr(), asb.gpu_addr(), wb.gpu_addr(), wsb.gpu_addr(), at, m=m, n=n, k=k, bias=dev.up(bias).gpu_addr() if with_bias else 0, out_bf16=bf16,
                               a_stride=0 if dense else a_stride, w_stride=0 if dense else w_stride, y_stride=0 if dense else y_stride))
    rt.synchronize()
    want = ref.product(a, a_scales, w, w_scales, bias)
    got = read_rows(y, m, n, y_stride, bf16, shift)
    assert same_bf16(got, ref.bf16_bits(want)) if bf16 else same(got.view(np.float32), want)


def test_sums_at_the_ends_of_32_bits(t0, rt, dev):
    # the largest sum there is, its negative, and rows whose scales are zero, infinite and NaN
    k, n = 131071, 40
    for m in (5, 40, 300):
        a = np.full((m, k), -128, np.int8)
        a[1::2] = 127
        w = np.full((n, k), -128, np.int8)
        w[1::2] = 127
        a_scales, w_scales = np.ones(m, np.float32), np.ones(n, np.float32)
        a_scales[2], a_scales[3], a_scales[4] = 0, np.inf, np.nan
        w_scales[7], w_scales[8] = np.nan, 0
        y = dev.up(np.zeros((m, n), np.float32))
        rt.q8_gemm(rt.q8_gemm_args(dev.up(padded(a, k + 1, 1)).gpu_addr(), dev.up(a_scales).gpu_addr(), dev.up(padded(w, k + 1, 1)).gpu_addr(), dev.up(w_scales).gpu_addr(), y.gpu_addr(),
                                   m=m, n=n, k=k))
        rt.synchronize()
        assert same(y.read(m * n * 4, np.float32).reshape(m, n), ref.product(a, a_scales, w, w_scales))


GATED = [(1, 1, 1), (1, 11008, 4096), (2, 100, 100), (4, 333, 1357), (8, 2048, 512), (15, 4096, 640), (16, 1000, 4096), (17, 700, 300), (40, 5001, 256), (64, 4096, 1024), (100, 1433, 4096),
         (128, 130, 2000), (129, 2048, 384), (200, 129, 129), (256, 3000, 512), (300, 1111, 1025), (600, 1000, 600), (1024, 2048, 256), (1300, 777, 1357), (2500, 512, 512), (2300, 701, 130), (2301, 705, 131)]


@pytest.mark.parametrize("m, n, k", GATED)
def test_gated_products(t0, rt, dev, m, n, k):
    rng = np.random.default_rng(m + 5 * n + k)
    bf16, act = (m + k) % 2 == 0, ("silu", "gelu", "relu")[(m + n) % 3]
    dense = n % 2 == 0
    stride = up16(k) + (0 if dense else 48)
    a, a_scales, ab, asb = rows8(rng, dev, m, k, stride)
    weights = [rows8(rng, dev, n, k, stride) for _ in range(2)]
    a_scales *= np.float32(1e-4) / np.float32(np.sqrt(k))
    a_scales[0] *= 300                                                    # gates far into both ends of the sigmoid
    asb = dev.up(a_scales)
    (g, g_scales, gb, gsb), (u, u_scales, ub, usb) = weights
    y_stride, shift = (n, 0) if dense else [(n + 3, 5), (up16(n), 0)][k % 2]
    y, at = out_rows(dev, m, n, y_stride, bf16, shift)
    rt.q8_gated(rt.q8_gated_args(ab.gpu_addr(), asb.gpu_addr(), gb.gpu_addr(), gsb.gpu_addr(), ub.gpu_addr(), usb.gpu_addr(), at, m=m, n=n, k=k, activation=act, out_bf16=bf16,
                                 a_stride=stride, w_stride=stride, y_stride=y_stride))
    rt.synchronize()
    want, bound = ref.gated(a, a_scales, g, g_scales, u, u_scales, act)
    bits = read_rows(y, m, n, y_stride, bf16, shift)
    got = ref.from_bits(bits) if bf16 else bits.view(np.float32)
    bound = bound + (2.0**-8 * np.abs(want) if bf16 else 0)
    off = np.abs(got.astype(np.float64) - want)
    assert (off <= bound).all(), float((off / bound).max())


def test_a_rows_result_does_not_depend_on_the_others(t0, rt, dev):
    rng = np.random.default_rng(11)
    n, k = 1500, 1000
    a, a_scales, ab, asb = rows8(rng, dev, 700, k, up16(k))
    w, w_scales, wb, wsb = rows8(rng, dev, n, k, up16(k))
    u, u_scales, ub, usb = rows8(rng, dev, n, k, up16(k))
    first = None
    for m in (700, 256, 130, 60, 16, 1):
        y = [dev.up(np.zeros((m, n), np.uint16)) for _ in range(2)]
        rt.q8_gemm(rt.q8_gemm_args(ab.gpu_addr(), asb.gpu_addr(), wb.gpu_addr(), wsb.gpu_addr(), y[0].gpu_addr(), m=m, n=n, k=k, out_bf16=True))
        rt.q8_gated(rt.q8_gated_args(ab.gpu_addr(), asb.gpu_addr(), wb.gpu_addr(), wsb.gpu_addr(), ub.gpu_addr(), usb.gpu_addr(), y[1].gpu_addr(), m=m, n=n, k=k))
        rt.synchronize()
        got = [b.read(m * n * 2, np.uint16).reshape(m, n) for b in y]
        first = first or got
        assert all(np.array_equal(x, f[:m]) for x, f in zip(got, first))


def test_rows_far_apart(t0, rt, dev):
    # offsets beyond 32 bits: rows a gigabyte apart, in every array
    rng = np.random.default_rng(21)
    step, k, n, m = 1 << 30, 100, 6, 5
    big = rt.alloc(7 * step)
    a, a_scales, _, asb = rows8(rng, dev, m, k, up16(k))
    w, w_scales, _, wsb = rows8(rng, dev, n, k, up16(k))
    for i in range(m):
        big.write_bytes(i * step, a[i])
    for j in range(n):
        big.write_bytes(j * step + 4096, w[j])
    y_at = 8192
    base = big.gpu_addr()
    rt.q8_gemm(rt.q8_gemm_args(base, asb.gpu_addr(), base + 4096, wsb.gpu_addr(), base + y_at, m=m, n=n, k=k, a_stride=step, w_stride=step, y_stride=step // 4))
    q = dev.up(np.zeros((m, 112), np.int8))
    scales = dev.up(np.zeros(m, np.float32))
    x = rng.standard_normal((m, k)).astype(np.float32)
    for i in range(m):
        big.write_bytes(i * step + 16384, x[i])
    rt.q8_quant(rt.q8_quant_args(base + 16384, q.gpu_addr(), scales.gpu_addr(), n_rows=m, dim=k, x_f32=True, x_stride=step // 4))
    rt.q8_dequant(rt.q8_dequant_args(base, asb.gpu_addr(), base + 32768, n_rows=m, dim=k, out_f32=True, q_stride=step, y_stride=step // 4))
    rt.synchronize()
    want = ref.product(a, a_scales, w, w_scales)
    for i in range(m):
        assert same(big.read_bytes(i * step + y_at, 4 * n, np.float32), want[i])
        assert same(big.read_bytes(i * step + 32768, 4 * k, np.float32), a[i].astype(np.float32) * a_scales[i])
    assert np.array_equal(q.read(m * 112, np.int8).reshape(m, 112)[:, :k], ref.hold(x)[0])
    big.free()


# --------------------------------------------------------------------------- together

class Layer:
    """The calls of a feed-forward block with the norm before it: norm, gated pair, rows into eight bits, product."""

    def __init__(self, rng, t0, rt, dev, m, dim, hidden):
        self.rt, self.m, self.dim, self.hidden = rt, m, dim, hidden
        self.norm = ref.bf16_round(rng.uniform(0.5, 1.5, dim).astype(np.float32))
        made = lambda n, k: rows8(rng, dev, n, k, up16(k))  # noqa: E731
        self.gate, self.up, self.down = made(hidden, dim), made(hidden, dim), made(dim, hidden)
        for _, s, _, b in (self.gate, self.up, self.down):
            s *= np.float32(3e-5)
            b.write(s)
        new = lambda *shape, kind=np.float32: dev.up(np.zeros(shape, kind))  # noqa: E731
        self.x, self.res = new(m, dim), new(m, dim, kind=np.uint16)
        self.q, self.qs, self.h = new(m, up16(dim), kind=np.int8), new(m), new(m, hidden, kind=np.uint16)
        self.hq, self.hs, self.y = new(m, up16(hidden), kind=np.int8), new(m), new(m, dim)
        at = lambda b: b.gpu_addr()  # noqa: E731
        R = rt
        self.calls = [
            (rt.q8_rmsnorm, R.q8_rmsnorm_args(at(self.x), at(dev.up(ref.bf16_bits(self.norm))), n_rows=m, dim=dim, eps=1e-6, x_f32=True, residual=at(self.res), residual_out=at(self.res),
                                              q=at(self.q), scales=at(self.qs))),
            (rt.q8_gated, R.q8_gated_args(at(self.q), at(self.qs), at(self.gate[2]), at(self.gate[3]), at(self.up[2]), at(self.up[3]), at(self.h), m=m, n=hidden, k=dim)),
            (rt.q8_quant, R.q8_quant_args(at(self.h), at(self.hq), at(self.hs), n_rows=m, dim=hidden)),
            (rt.q8_gemm, R.q8_gemm_args(at(self.hq), at(self.hs), at(self.down[2]), at(self.down[3]), at(self.y), m=m, n=dim, k=hidden)),
        ]

    def put(self, x, res):
        self.x.write(x)
        self.res.write(ref.bf16_bits(res))

    def run(self):
        for call, args in self.calls:
            call(args)

    def check(self, x, res):
        m, dim, hidden = self.m, self.dim, self.hidden
        y, h = ref.rmsnorm(x, self.norm, 1e-6, res, True)
        assert same(ref.from_bits(self.res.read(m * dim * 2, np.uint16)).reshape(m, dim), h)
        q, qs = ref.hold(y)
        assert np.array_equal(self.q.read(m * up16(dim), np.int8).reshape(m, -1)[:, :dim], q) and same(self.qs.read(4 * m, np.float32), qs)
        want, bound = ref.gated(q, qs, self.gate[0], self.gate[1], self.up[0], self.up[1], "silu")
        got = ref.from_bits(self.h.read(m * hidden * 2, np.uint16)).reshape(m, hidden)
        assert (np.abs(got - want) <= bound + 2.0**-8 * np.abs(want)).all()
        hq, hs = ref.hold(got)
        assert np.array_equal(self.hq.read(m * up16(hidden), np.int8).reshape(m, -1)[:, :hidden], hq) and same(self.hs.read(4 * m, np.float32), hs)
        assert same(self.y.read(m * dim * 4, np.float32).reshape(m, dim), ref.product(hq, hs, self.down[0], self.down[1]))


@pytest.mark.parametrize("m, dim, hidden", [(1, 512, 1408), (37, 512, 1408), (300, 640, 1000)])
def test_a_block_run_and_recorded(t0, rt, dev, m, dim, hidden):
    # eager, then recorded once and replayed on other rows, on the runtime's stream and on another; two graphs of it, one after the other
    rng = np.random.default_rng(m)
    layer = Layer(rng, t0, rt, dev, m, dim, hidden)
    fresh = lambda: (rng.standard_normal((m, dim)).astype(np.float32), ref.bf16_round(rng.standard_normal((m, dim)).astype(np.float32)))  # noqa: E731
    driver = Driver()
    x, res = fresh()
    layer.put(x, res)
    layer.run()
    rt.synchronize()
    layer.check(x, res)
    with driver.record(rt) as one:
        layer.run()
    with driver.record(rt) as two:
        layer.run()
    other = driver.stream()
    for ex, stream in ((one[0], rt.stream()), (two[0], other), (one[0], other), (two[0], rt.stream())):
        x, res = fresh()
        layer.put(x, res)
        rt.synchronize()
        driver.replay(ex, stream)
        driver.sync(stream)
        layer.check(x, res)
    for ex in (one[0], two[0]):
        driver.drop(ex)
    driver.drop(stream=other)


def test_many_calls_behind_one_another(t0, rt, dev):
    # every call reads what the one before it wrote, fifty times over: launches overlap their prologues, never their reads
    rng = np.random.default_rng(9)
    layer = Layer(rng, t0, rt, dev, 20, 256, 640)
    x, res = rng.standard_normal((20, 256)).astype(np.float32), ref.bf16_round(rng.standard_normal((20, 256)).astype(np.float32))
    layer.put(x, res)
    for _ in range(50):
        layer.run()
    rt.synchronize()
    got = ref.from_bits(layer.res.read(20 * 256 * 2, np.uint16)).reshape(20, 256)
    h = res
    for _ in range(50):
        h = ref.bf16_round(h + x)
    assert same(got, h)
    q, qs = ref.hold(ref.rmsnorm(h, layer.norm, 1e-6)[0])
    assert np.array_equal(layer.q.read(20 * 256, np.int8).reshape(20, 256), q) and same(layer.qs.read(80, np.float32), qs)


@pytest.mark.parametrize("m, n, k", [(1, 3000, 1024), (24, 512, 2048), (300, 700, 512)])
def test_weights_made_by_the_call_before(t0, rt, dev, m, n, k):
    # a product asks for its first weights before the launch before it is over: what that launch writes is what it multiplies
    rng = np.random.default_rng(n)
    a, a_scales, ab, asb = rows8(rng, dev, m, k, up16(k))
    sources = [rng.standard_normal((n, k)).astype(np.float32) for _ in range(3)]
    bufs = [dev.up(s) for s in sources]
    q, s = dev.up(np.zeros((n, up16(k)), np.int8)), dev.up(np.zeros(n, np.float32))
    ys = [dev.up(np.zeros((m, n), np.float32)) for _ in range(24)]
    for i, y in enumerate(ys):
        rt.q8_quant(rt.q8_quant_args(bufs[i % 3].gpu_addr(), q.gpu_addr(), s.gpu_addr(), n_rows=n, dim=k, x_f32=True))
        rt.q8_gemm(rt.q8_gemm_args(ab.gpu_addr(), asb.gpu_addr(), q.gpu_addr(), s.gpu_addr(), y.gpu_addr(), m=m, n=n, k=k))
    rt.synchronize()
    want = [ref.product(a, a_scales, *ref.hold(x)) for x in sources]
    for i, y in enumerate(ys):
        assert same(y.read(m * n * 4, np.float32).reshape(m, n), want[i % 3]), i


def test_two_runtimes_at_once(t0, rt):
    # products of every kernel on two streams beside one another: clusters of both wait for room, and nothing of one is another's
    runs = [t0.GpuRuntime(0), t0.GpuRuntime(0)]
    devs = [Device(r) for r in runs]
    shapes = [(1, 2048, 1024), (20, 512, 4096), (40, 1024, 2048), (600, 1024, 512)]
    jobs = []
    for i, (r, d) in enumerate(zip(runs, devs)):
        rng = np.random.default_rng(i)
        for m, n, k in shapes:
            a, w, u = rows8(rng, d, m, k, up16(k)), rows8(rng, d, n, k, up16(k)), rows8(rng, d, n, k, up16(k))
            y, z = d.up(np.zeros((m, n), np.float32)), d.up(np.zeros((m, n), np.float32))
            at = lambda b: b.gpu_addr()  # noqa: E731
            jobs.append((i, r.q8_gemm, r.q8_gemm_args(at(a[2]), at(a[3]), at(w[2]), at(w[3]), at(y), m=m, n=n, k=k), y, ref.product(a[0], a[1], w[0], w[1])))
            with np.errstate(over="ignore"):
                g, v = ref.product(a[0], a[1], w[0], w[1]), ref.product(a[0], a[1], u[0], u[1])
                jobs.append((i, r.q8_gated, r.q8_gated_args(at(a[2]), at(a[3]), at(w[2]), at(w[3]), at(u[2]), at(u[3]), at(z), m=m, n=n, k=k, activation="relu", out_bf16=False), z,
                             np.maximum(g, 0) * v))
    order = np.random.default_rng(5).permutation(np.repeat(np.arange(len(jobs)), 20))
    for j in order:
        jobs[j][1](jobs[j][2])
    for r in runs:
        r.synchronize()
    for _, _, _, y, want in jobs:
        assert same(y.read(want.size * 4, np.float32).reshape(want.shape), want)
    for d, r in zip(devs, runs):
        d.free()
        r.close()


def test_a_decoder_layer(t0, rt, dev):
    """norm, q/k/v product, cache append, attention, rows into eight bits, output product, norm with residual: each step against the restatement of what it was given."""
    import kv4_reference as kv4
    rng = np.random.default_rng(33)
    rows, lens, heads, group, hd, page, dim = [5, 1, 9], [40, 17, 9], 2, 2, 64, 16, 384
    n, hq = sum(rows), heads * group
    wide = (hq + 2 * heads) * hd
    x = rng.standard_normal((n, dim)).astype(np.float32)
    norm = ref.bf16_round(rng.uniform(0.5, 1.5, dim).astype(np.float32))
    wqkv, wo = rows8(rng, dev, wide, dim, up16(dim)), rows8(rng, dev, dim, hq * hd, up16(hq * hd))
    for _, s, _, b in (wqkv, wo):
        s[:] = np.float32(8e-4) * np.exp(rng.uniform(-0.2, 0.2, s.shape)).astype(np.float32)
        b.write(s)
    res = dev.up(ref.bf16_bits(x))
    x = ref.bf16_round(x)
    at = lambda b: b.gpu_addr()  # noqa: E731
    new = lambda *shape, kind=np.float32: dev.up(np.zeros(shape, kind))  # noqa: E731
    q8, q8s, qkv, nb = new(n, up16(dim), kind=np.int8), new(n), new(n, wide), dev.up(ref.bf16_bits(norm))
    rt.q8_rmsnorm(rt.q8_rmsnorm_args(at(res), at(nb), n_rows=n, dim=dim, eps=1e-6, q=at(q8), scales=at(q8s)))
    rt.q8_gemm(rt.q8_gemm_args(at(q8), at(q8s), at(wqkv[2]), at(wqkv[3]), at(qkv), m=n, n=wide, k=dim))
    cache = kv4.Cache(rng, lens, heads, hd, page)
    from test_kv4_gpu import make_batch
    pool = dev.up(np.zeros((cache.n_pages, heads, page * (hd + 8)), np.uint8))
    batch = make_batch(t0, dev, cache, pool, rows)
    qo, y = new(n, hq * hd, kind=np.uint16), new(n, hq * hd, kind=np.uint16)
    rt.kv4_append(batch, rt.kv4_append_args(at(qkv) + hq * hd * 4, at(qkv) + (hq + heads) * hd * 4, k_stride=wide, v_stride=wide, in_f32=True, q=at(qkv), q_stride=wide, q_out=at(qo),
                                            n_q_heads=hq))
    rt.kv4_attention(batch, rt.kv4_attention_args(at(qo), at(y), n_q_heads=hq, scale=hd**-0.5))
    y8, y8s, o, k8, k8s = new(n, up16(hq * hd), kind=np.int8), new(n), new(n, dim), new(n, up16(dim), kind=np.int8), new(n)
    rt.q8_quant(rt.q8_quant_args(at(y), at(y8), at(y8s), n_rows=n, dim=hq * hd))
    rt.q8_gemm(rt.q8_gemm_args(at(y8), at(y8s), at(wo[2]), at(wo[3]), at(o), m=n, n=dim, k=hq * hd))
    rt.q8_rmsnorm(rt.q8_rmsnorm_args(at(o), at(nb), n_rows=n, dim=dim, eps=1e-6, x_f32=True, residual=at(res), residual_out=at(res), q=at(k8), scales=at(k8s)))
    rt.synchronize()
    codes, scales = ref.hold(ref.rmsnorm(x, norm, 1e-6)[0])
    assert np.array_equal(q8.read(n * up16(dim), np.int8).reshape(n, -1)[:, :dim], codes) and same(q8s.read(4 * n, np.float32), scales)
    want = ref.product(codes, scales, wqkv[0], wqkv[1])
    assert same(qkv.read(4 * n * wide, np.float32).reshape(n, wide), want)
    assert np.array_equal(qo.read(2 * n * hq * hd, np.uint16).reshape(n, -1), ref.bf16_bits(want[:, :hq * hd]))
    attended = ref.from_bits(y.read(2 * n * hq * hd, np.uint16)).reshape(n, -1)
    assert np.abs(attended).max() > 0 and np.isfinite(attended).all()
    codes, scales = ref.hold(attended)
    assert np.array_equal(y8.read(n * up16(hq * hd), np.int8).reshape(n, -1)[:, :hq * hd], codes) and same(y8s.read(4 * n, np.float32), scales)
    out = ref.product(codes, scales, wo[0], wo[1])
    assert same(o.read(4 * n * dim, np.float32).reshape(n, dim), out)
    after, h = ref.rmsnorm(out, norm, 1e-6, x, True)
    assert same(ref.from_bits(res.read(2 * n * dim, np.uint16)).reshape(n, dim), h)
    codes, scales = ref.hold(after)
    assert np.array_equal(k8.read(n * up16(dim), np.int8).reshape(n, -1)[:, :dim], codes) and same(k8s.read(4 * n, np.float32), scales)


@pytest.mark.parametrize("m, n, k, gated", [(1, 2048, 1024, False), (20, 512, 4096, False), (40, 1024, 4096, True), (600, 2048, 1024, False), (600, 2048, 1024, True)])
def test_a_wait_that_runs_out_is_reported(t0, m, n, k, gated):
    # the first copy of the first tile is left out (whole sums, parts over a cluster, pairs): the kernel gives up after the wait limit by itself, and says so
    rng = np.random.default_rng(m)
    r = t0.GpuRuntime(0)
    dev = Device(r)
    _, _, a, a_s = rows8(rng, dev, m, k, up16(k))
    _, _, w, w_s = rows8(rng, dev, n, k, up16(k))
    y = dev.up(np.zeros((m, n), np.float32))
    at = lambda b: b.gpu_addr()  # noqa: E731
    call = (lambda: r.q8_gated(r.q8_gated_args(at(a), at(a_s), at(w), at(w_s), at(w), at(w_s), at(y), m=m, n=n, k=k, out_bf16=False))) if gated else (
        lambda: r.q8_gemm(r.q8_gemm_args(at(a), at(a_s), at(w), at(w_s), at(y), m=m, n=n, k=k)))
    call()
    r.synchronize()
    want = y.read(m * n * 4, np.float32)
    r.set_wait_limit_ns(3_000_000)
    r.selftest_drop_one_load()
    call()
    with pytest.raises(t0.T0Error) as e:
        r.synchronize()
    assert e.value.code == 4 and "wait expired" in str(e.value) and r.is_poisoned()
    with pytest.raises(t0.T0Error) as e:
        call()
    assert e.value.code == 3
    dev.free()
    r.close()
    # another runtime on the device goes on, and gives what the first one gave
    r = t0.GpuRuntime(0)
    dev = Device(r)
    rng = np.random.default_rng(m)
    _, _, a, a_s = rows8(rng, dev, m, k, up16(k))
    _, _, w, w_s = rows8(rng, dev, n, k, up16(k))
    y = dev.up(np.zeros((m, n), np.float32))
    call()
    r.synchronize()
    assert same(y.read(m * n * 4, np.float32), want)
    dev.free()
    r.close()


FIRST_CALLS = """
import importlib, sys
sys.path[:0] = [{root!r}, {root!r} + "/tests"]
import numpy as np
t0 = importlib.import_module("rust-gpu_b200")
import q8_reference as ref
from test_q8_gpu import Driver, rows8, same, up16
from test_kv4_gpu import Device
rt = t0.GpuRuntime(0)
dev, rng, d = Device(rt), np.random.default_rng(1), Driver()
at = lambda b: b.gpu_addr()
done = []
with d.record(rt) as graph:
    pass
uploads = []
for m, n, k in ((1, 600, 1024), (24, 256, 4096), (700, 512, 256)):
    a, w = rows8(rng, dev, m, k, up16(k)), rows8(rng, dev, n, k, up16(k))
    uploads.append((m, n, k, a, w, dev.up(np.zeros((m, n), np.float32)), dev.up(np.zeros((m, n), np.float32))))
x = [(rows, dim, rng.standard_normal((rows, dim)).astype(np.float32)) for rows, dim in ((2, 512), (2000, 512))]
x = [(rows, dim, v, dev.up(v), dev.up(np.zeros((rows, dim), np.int8)), dev.up(np.zeros(rows, np.float32)), dev.up(np.zeros((rows, dim), np.float32)), dev.up(np.ones(dim, np.float32))) for rows, dim, v in x]
with d.record(rt) as graph:
    for m, n, k, a, w, y, z in uploads:
        rt.q8_gemm(rt.q8_gemm_args(at(a[2]), at(a[3]), at(w[2]), at(w[3]), at(y), m=m, n=n, k=k))
        rt.q8_gated(rt.q8_gated_args(at(a[2]), at(a[3]), at(w[2]), at(w[3]), at(w[2]), at(w[3]), at(z), m=m, n=n, k=k, activation="relu", out_bf16=False))
    for rows, dim, v, b, q, s, back, one in x:
        rt.q8_quant(rt.q8_quant_args(at(b), at(q), at(s), n_rows=rows, dim=dim, x_f32=True))
        rt.q8_dequant(rt.q8_dequant_args(at(q), at(s), at(back), n_rows=rows, dim=dim, out_f32=True))
        rt.q8_rmsnorm(rt.q8_rmsnorm_args(at(b), at(one), n_rows=rows, dim=dim, eps=1e-5, x_f32=True, weight_f32=True, q=at(q), scales=at(s)))
d.replay(graph[0], rt.stream())
rt.synchronize()
for m, n, k, a, w, y, z in uploads:
    want = ref.product(a[0], a[1], w[0], w[1])
    assert same(y.read(m * n * 4, np.float32).reshape(m, n), want)
    assert same(z.read(m * n * 4, np.float32).reshape(m, n), np.maximum(want, 0) * want)
for rows, dim, v, b, q, s, back, one in x:
    codes, scales = ref.hold(v)
    assert same(back.read(rows * dim * 4, np.float32).reshape(rows, dim), codes.astype(np.float32) * scales[:, None])
    assert np.array_equal(q.read(rows * dim, np.int8).reshape(rows, dim), ref.hold(ref.rmsnorm(v, np.ones(dim), 1e-5)[0])[0])
d.drop(graph[0])
print("recorded")
"""


def test_the_first_calls_of_a_program_may_be_recorded(t0):
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS.format(root=root)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "recorded" in r.stdout, r.stderr[-2000:]
