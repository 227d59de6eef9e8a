"""Root-mean-square norms with a residual, their 8-bit outputs and rows of codes (thhip_rmsnorm, thhip_rmsnorm_i8,
thhip_quantize_rows, thhip_dequantize_rows) against the formulas in 64 bits."""
import numpy as np
import pytest

import gpu_util as G
import w4_util as U
from thnets_amd import api
from w4_util import BF16, F16, F32

pytestmark = pytest.mark.gpu

TYPES = [F32, F16, BF16]
EPS = 1e-5
# rows, cols: around every change of the kernel's row capacity, odd lengths, rows longer than registers hold
SHAPES = [(1, 1), (3, 7), (1, 8), (5, 64), (9, 100), (4, 256), (6, 257), (2, 511), (7, 512), (5, 513), (3, 1000), (2, 1024), (3, 1025), (4, 2048),
          (2, 2050), (3, 4096), (2, 4100), (2, 5003), (1, 8192), (2, 9216), (2, 16384), (1, 16388), (2, 32771), (1, 70001), (130, 96)]


def word(dtype):
    return np.uint32 if dtype == F32 else np.uint16


def chain(cols):
    """Relative error of a sum of `cols` squares: a thread adds at most 64 of them, or cols / 1024 where the row is long; then six
    steps over the lanes and sixteen wavefronts; every addition and product is off by 2^-24."""
    return (max(64, cols / 1024 + 8) + 6 + 16 + 2) * 2.0 ** -24


def inputs(seed, rows, cols, dtype, res, weight):
    g = U.rng(seed)
    x = U.rounded(g.standard_normal((rows, cols)) * 3 + 0.5, dtype)
    r = U.rounded(g.standard_normal((rows, cols)), dtype) if res else None
    w = (1 + 0.2 * g.standard_normal(cols)).astype(np.float32) if weight else None
    return x, r, w


def norm64(x, r, w, eps=EPS):
    h = x.astype(np.float64) + (r.astype(np.float64) if r is not None else 0)
    y = h / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    return h, y * w.astype(np.float64) if w is not None else y


def near(got, want, rel, dtype, what):
    assert (np.abs(got - want) <= rel * np.abs(want) + U.TINY[dtype] * 1.01).all(), "%s: off by %g relative" % (
        what, (np.abs(got - want) / np.maximum(np.abs(want), 1e-30)).max())


class Call:
    """One call on fresh buffers: strides ld, offsets off (elements), sum / y where wanted."""

    def __init__(self, lib, x, r, w, dtype, ld=None, off=0, group=None, norm=True, sum_out=True, eps=EPS):
        rows, cols = x.shape
        G.note("rows %s %dx%d dtype=%d ld=%s off=%d group=%s res=%d w=%d" % (
            "norm" if norm else "codes", rows, cols, dtype, ld, off, group, r is not None, w is not None))
        dx = U.Rows(lib, U.raw(x, dtype), ld, off)
        dr = U.Rows(lib, U.raw(r, dtype), ld, off) if r is not None else None
        dw = api.DeviceArray(lib, w) if w is not None else None
        dsum = U.Rows(lib, None, ld, off, x.shape, word(dtype)) if sum_out and norm else None
        head = (dx.ptr, dx.ld, dr.ptr if dr else None, dr.ld if dr else 0, dw.ptr if dw else None, eps,
                dsum.ptr if dsum else None, dsum.ld if dsum else 0)
        if group is None:
            dy = U.Rows(lib, None, ld, off, x.shape, word(dtype))
            assert lib.thhip_rmsnorm(*head, dy.ptr, dy.ld, rows, cols, dtype) == 0
        else:
            dq = U.Rows(lib, None, ld, off, x.shape, np.int8)
            ds = U.Rows(lib, None, None, 0, (rows, U.groups_of(cols, group)), np.uint32)
            if norm:
                assert lib.thhip_rmsnorm_i8(*head, dq.ptr, dq.ld, ds.ptr, group, rows, cols, dtype) == 0
            else:
                assert lib.thhip_quantize_rows(dx.ptr, dx.ld, dq.ptr, dq.ld, ds.ptr, group, rows, cols, dtype) == 0
        lib.thhip_sync()
        dx.get()
        self.sum = U.unraw(dsum.get(), dtype) if dsum else None
        if group is None:
            self.y = U.unraw(dy.get(), dtype)
        else:
            self.q, self.scale = dq.get(), ds.get().view(np.float32)


def check_codes(c, y, cols, group, err):
    """Scales within `err` of max|y| / 127; codes within half a step of y (and what err moves 127 steps by)."""
    step = group or cols
    for i in range(c.scale.shape[1]):
        part = y[:, i * step:(i + 1) * step]
        top = np.abs(part).max(1) / 127
        near(c.scale[:, i], top, err + 2.0 ** -22, F32, "scale")
        q = c.q[:, i * step:(i + 1) * step].astype(np.float64)
        assert (np.abs(q) <= 127).all() and (np.abs(q).max(1) == 127).all()
        assert (np.abs(q - part / top[:, None]) <= 0.5 + 127 * (2 * err + 2.0 ** -21)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_norm(hiplib, i, dtype):
    rows, cols = SHAPES[i]
    x, r, w = inputs(10 + i, rows, cols, dtype, i % 3 != 0, i % 4 != 1)
    c = Call(hiplib, x, r, w, dtype)
    h, y = norm64(x, r, w)
    near(c.sum, h, U.HALF_STEP[dtype] * (1 + 2.0 ** -8) + 2.0 ** -24, dtype, "sum")
    near(c.y, y, U.HALF_STEP[dtype] * (1 + 2.0 ** -8) + chain(cols) + 8 * 2.0 ** -24, dtype, "y")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_norm_i8(hiplib, i, dtype):
    rows, cols = SHAPES[i]
    group = [0, 32, 64, 128, 256][i % 5]
    x, r, w = inputs(50 + i, rows, cols, dtype, i % 3 != 1, i % 4 != 2)
    c = Call(hiplib, x, r, w, dtype, group=group)
    h, y = norm64(x, r, w)
    near(c.sum, h, U.HALF_STEP[dtype] * (1 + 2.0 ** -8) + 2.0 ** -24, dtype, "sum")
    check_codes(c, y, cols, group, chain(cols) + 8 * 2.0 ** -24)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(3, 4500), (2, 5120), (3, 5121), (2, 6144), (3, 6145), (3, 9000), (2, 10240), (3, 10243), (2, 12288), (3, 12290)])
def test_norms_of_rows_between_four_and_eight_vectors_a_thread(hiplib, dtype, rows, cols):
    x, r, w = inputs(90 + cols, rows, cols, dtype, True, True)
    h, y = norm64(x, r, w)
    err = chain(cols) + 8 * 2.0 ** -24
    c = Call(hiplib, x, r, w, dtype)
    near(c.sum, h, U.HALF_STEP[dtype] * (1 + 2.0 ** -8) + 2.0 ** -24, dtype, "sum")
    near(c.y, y, U.HALF_STEP[dtype] * (1 + 2.0 ** -8) + err, dtype, "y")
    for group in (0, 64):
        check_codes(Call(hiplib, x, r, w, dtype, group=group), y, cols, group, err)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [0, 32, 64, 128, 256])
@pytest.mark.parametrize("cols", [40, 600, 1000, 5000, 20000, 66000])
def test_codes_of_rows_and_back(hiplib, dtype, group, cols):
    g = U.rng(90)
    x = U.rounded(g.standard_normal((5, cols)) * 2, dtype)
    c = Call(hiplib, x, None, None, dtype, group=group, norm=False)
    check_codes(c, x.astype(np.float64), cols, group, 0.0)
    # and back: one product and one rounding
    for ld, off in ((None, 0), (cols + 3, 5)):
        dq = U.Rows(hiplib, c.q, ld, off)
        ds = api.DeviceArray(hiplib, c.scale)
        dy = U.Rows(hiplib, None, ld, off, x.shape, word(dtype))
        assert hiplib.thhip_dequantize_rows(dq.ptr, dq.ld, ds.ptr, group, dy.ptr, dy.ld, 5, cols, dtype) == 0
        hiplib.thhip_sync()
        want = c.q * U.spread_x(c.scale, cols, group)
        assert np.array_equal(U.unraw(dy.get(), dtype), U.rounded(want, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,group", [(1, 2049, 32), (1, 300001, 256), (7, 40003, 64), (511, 2100, 128), (513, 2100, 0), (1024, 2056, 32)])
def test_back_from_codes_of_few_long_rows(hiplib, dtype, rows, cols, group):
    """Rows that several workgroups share: every value is its code times its scale, rounded once; nothing else is written."""
    g = U.rng(95)
    q = g.integers(-127, 128, (rows, cols)).astype(np.int8)
    scale = g.uniform(0.5, 1.5, (rows, U.groups_of(cols, group))).astype(np.float32)
    dq, ds = U.Rows(hiplib, q, cols + 3, 1), api.DeviceArray(hiplib, scale)
    dy = U.Rows(hiplib, None, cols + 5, 3, (rows, cols), word(dtype))
    G.note("back %dx%d group=%d dtype=%d" % (rows, cols, group, dtype))
    assert hiplib.thhip_dequantize_rows(dq.ptr, dq.ld, ds.ptr, group, dy.ptr, dy.ld, rows, cols, dtype) == 0
    hiplib.thhip_sync()
    dq.get()
    assert np.array_equal(dy.get(), U.raw(q.astype(np.float32) * np.repeat(scale, group or cols, 1)[:, :cols], dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [100, 512, 3000, 17000, 70000])
@pytest.mark.parametrize("pad,off", [(5, 3), (8, 8), (1, 0), (0, 1)])
def test_strides_and_offsets(hiplib, dtype, cols, pad, off):
    """Rows apart and off every vector's alignment, NaNs between them: the bits of the contiguous call, nothing else written."""
    x, r, w = inputs(20, 3, cols, dtype, True, True)
    a, b = Call(hiplib, x, r, w, dtype), Call(hiplib, x, r, w, dtype, ld=cols + pad, off=off)
    assert np.array_equal(a.y, b.y) and np.array_equal(a.sum, b.sum)
    a, b = Call(hiplib, x, r, w, dtype, group=128), Call(hiplib, x, r, w, dtype, ld=cols + pad, off=off, group=128)
    assert np.array_equal(a.q, b.q) and np.array_equal(a.scale, b.scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [64, 777, 4096, 33000, 70000])
@pytest.mark.parametrize("sum_to,y_to", [("r", "x"), ("x", "r"), ("r", None), (None, "x")])
def test_in_place(hiplib, dtype, cols, sum_to, y_to):
    x, r, w = inputs(30, 4, cols, dtype, True, True)
    want = Call(hiplib, x, r, w, dtype)
    bufs = {"x": U.Rows(hiplib, U.raw(x, dtype)), "r": U.Rows(hiplib, U.raw(r, dtype))}
    dsum = bufs[sum_to] if sum_to else U.Rows(hiplib, None, None, 0, x.shape, word(dtype))
    dy = bufs[y_to] if y_to else U.Rows(hiplib, None, None, 0, x.shape, word(dtype))
    dw = api.DeviceArray(hiplib, w)
    assert hiplib.thhip_rmsnorm(bufs["x"].ptr, cols, bufs["r"].ptr, cols, dw.ptr, EPS, dsum.ptr, cols, dy.ptr, cols, 4, cols, dtype) == 0
    hiplib.thhip_sync()
    assert np.array_equal(U.unraw(dsum.get(), dtype), want.sum)
    assert np.array_equal(U.unraw(dy.get(), dtype), want.y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [96, 3000, 70000])
def test_rows_of_zeros_nans_and_infinities(hiplib, dtype, cols):
    """A row of zeros: y, codes and scales are 0 (eps keeps the root above 0).  A NaN makes its row NaN, an infinity
    its own place NaN and the rest 0.  The other rows do not see them."""
    x, _, _ = inputs(40, 6, cols, dtype, False, False)
    clean, clean8 = Call(hiplib, x, None, None, dtype), Call(hiplib, x, None, None, dtype, group=32)
    x[1], x[2, 5], x[3, 7] = 0, np.nan, np.inf
    c = Call(hiplib, x, None, None, dtype)
    assert not c.y[1].any() and np.isnan(c.y[2]).all() and np.isnan(c.y[3, 7]) and not np.delete(c.y[3], 7).any()
    assert all(np.array_equal(c.y[i], clean.y[i]) for i in (0, 4, 5))
    c = Call(hiplib, x, None, None, dtype, group=0)
    assert not c.q[1].any() and c.scale[1, 0] == 0 and np.isnan(c.scale[2, 0]) and np.isnan(c.scale[3, 0])
    c = Call(hiplib, x, None, None, dtype, group=32)
    assert not c.q[1].any() and not c.scale[1].any() and np.isnan(c.scale[2]).all() and np.isnan(c.scale[3, 0])
    assert not c.scale[3, 1:].any() and not c.q[3, 32:].any()
    assert all(np.array_equal(c.q[i], clean8.q[i]) and np.array_equal(c.scale[i], clean8.scale[i]) for i in (0, 4, 5))
    c = Call(hiplib, x, None, None, dtype, group=32, norm=False)
    assert not c.scale[1].any() and np.isnan(c.scale[2, 0]) and np.isinf(c.scale[3, 0]) and np.isfinite(c.scale[2:4, 1:]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_values_at_the_ends_of_the_range(hiplib, dtype):
    """Rows around 2^-118, where 127 / max|x| nears the largest number, and around 2^100."""
    g = U.rng(60)
    for e, gone in ((-119, True), (-112, False), (100, False)):
        x = U.rounded(g.uniform(-1, 1, (3, 200)) * 2.0 ** e, dtype)
        c = Call(hiplib, x, None, None, dtype, group=64, norm=False)
        if gone:
            assert not c.q.any() and not c.scale.any()
        else:
            check_codes(c, x.astype(np.float64), 200, 64, 0.0)


@pytest.mark.parametrize("rows", [(1 << 21) + 5])
def test_more_rows_than_a_launch_has(hiplib, rows):
    """Rows past the first launch's are rows like the others."""
    g = U.rng(70)
    some = U.rounded(g.standard_normal((1024, 8)), F16)
    x = np.resize(some, (rows, 8))
    a, b = Call(hiplib, some, None, None, F16), Call(hiplib, x, None, None, F16, sum_out=False)
    assert np.array_equal(b.y, np.resize(a.y, (rows, 8)))
    a, b = Call(hiplib, some, None, None, F16, group=32), Call(hiplib, x, None, None, F16, group=32, sum_out=False)
    assert np.array_equal(b.q, np.resize(a.q, (rows, 8))) and np.array_equal(b.scale, np.resize(a.scale, (rows, 1)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [5, 300, 5000, 70000])
def test_rows_whose_distance_passes_32_bits(hiplib, dtype, cols):
    """Three rows of x, the residual, both outputs and the codes, 2^32 bytes of x or 2^31 codes and more after one another."""
    es = U.ESIZE[dtype]
    ld = (1 << 32) // es + 40
    x, r, w = inputs(75, 3, cols, dtype, True, True)
    near_call = Call(hiplib, x, r, w, dtype)
    near_codes = Call(hiplib, x, r, w, dtype, group=32)
    kind = word(dtype)

    def far(a):
        dev = api.DeviceArray(hiplib, nbytes=2 * ld * a.itemsize + a.shape[1] * a.itemsize)
        for i in range(3):
            hiplib.thhip_memcpy_h2d(dev.ptr + i * ld * a.itemsize, np.ascontiguousarray(a[i]).ctypes.data, a[i].nbytes)
        return dev

    def back(dev, like):
        out = np.empty_like(like)
        for i in range(3):
            hiplib.thhip_memcpy_d2h(out[i].ctypes.data, dev.ptr + i * ld * like.itemsize, like[i].nbytes)
        return out

    dx, dr, dw = far(U.raw(x, dtype)), far(U.raw(r, dtype)), api.DeviceArray(hiplib, w)
    empty = np.zeros((3, cols), kind)
    ds, dy, dq = far(empty), far(empty), far(empty.astype(np.int8))
    n = U.groups_of(cols, 32)
    dscale = api.DeviceArray(hiplib, nbytes=3 * n * 4)
    G.note("far rows 3x%d dtype=%d" % (cols, dtype))
    assert hiplib.thhip_rmsnorm(dx.ptr, ld, dr.ptr, ld, dw.ptr, EPS, ds.ptr, ld, dy.ptr, ld, 3, cols, dtype) == 0
    hiplib.thhip_sync()
    assert np.array_equal(U.unraw(back(ds, empty), dtype), near_call.sum) and np.array_equal(U.unraw(back(dy, empty), dtype), near_call.y)
    assert hiplib.thhip_rmsnorm_i8(dx.ptr, ld, dr.ptr, ld, dw.ptr, EPS, None, 0, dq.ptr, ld, dscale.ptr, 32, 3, cols, dtype) == 0
    hiplib.thhip_sync()
    assert np.array_equal(back(dq, empty.astype(np.int8)), near_codes.q)
    assert np.array_equal(dscale.get((3, n), np.float32), near_codes.scale)
    assert hiplib.thhip_dequantize_rows(dq.ptr, ld, dscale.ptr, 32, dy.ptr, ld, 3, cols, dtype) == 0
    hiplib.thhip_sync()
    spread = np.repeat(near_codes.scale, 32, 1)[:, :cols]
    assert np.array_equal(back(dy, empty), U.raw(near_codes.q.astype(np.float32) * spread, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B", [1, 6, 70])
def test_a_block_of_a_network(hiplib, dtype, B):
    """The operators one after the other, as a network of Linear layers runs them: norm -> 8 bits -> 4-bit layer with
    Threshold -> 8 bits -> 4-bit layer -> the residual of the next norm.  Each step is checked against the formula on what
    the step before it wrote."""
    g = U.rng(80)
    D, H, group = 384, 1100, 128
    up = U.Layer.random(g, H, D, group, dtype, True).lay(hiplib)
    down = U.Layer.random(g, D, H, group, dtype, False).lay(hiplib)
    x, r, w = inputs(81, B, D, dtype, True, True)
    first = Call(hiplib, x, r, w, dtype, group=group)
    h, y = norm64(x, r, w)
    check_codes(first, y, D, group, chain(D) + 8 * 2.0 ** -24)
    mid = U.linear(hiplib, up, first.q, None, act=1, xs=first.scale, xgroup=group)
    want, mag = U.linear64(up, first.q * U.spread_x(first.scale.astype(np.float64), D, group))
    U.check_linear(mid, np.maximum(want, 0), mag, up)
    codes = Call(hiplib, mid, None, None, dtype, group=0, norm=False)
    check_codes(codes, mid.astype(np.float64), H, 0, 0.0)
    out = U.linear(hiplib, down, codes.q, None, xs=codes.scale)
    want, mag = U.linear64(down, codes.q * U.spread_x(codes.scale.astype(np.float64), H, 0))
    U.check_linear(out, want, mag, down)
    last = Call(hiplib, out, first.sum, w, dtype)
    h, y = norm64(out, first.sum, w)
    near(last.y, y, U.HALF_STEP[dtype] * (1 + 2.0 ** -8) + chain(D) + 8 * 2.0 ** -24 + 2.0 ** -22 * 8, dtype, "y")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", [5, 200, 3000, 9216, 70000])
def test_codes_of_the_largest_values(hiplib, dtype, cols):
    """Rows whose largest value is between 2^125 and the type's last number, or a mask of the type's lowest one beside ordinary
    values: every code is the nearest to x / scale."""
    g = U.rng(61)
    top = np.finfo(np.float32).max if dtype == F32 else np.float32((2 - 2.0 ** -7) * 2.0 ** 127)
    x = g.uniform(-1, 1, (6, cols)) * np.array([2.0 ** 125, 2.0 ** 126, 1.5 * 2.0 ** 126, 2.0 ** 127, float(top), 1])[:, None]
    x[:5, 0] = [2.0 ** 125, 2.0 ** 126 * 1.25, 2.0 ** 126 * 1.75, 2.0 ** 127, top]
    x[5, ::32] = -top
    x = U.rounded(x, dtype)
    for group in (0, 32, 256):
        check_codes(Call(hiplib, x, None, None, dtype, group=group, norm=False), x.astype(np.float64), cols, group, 0.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", [5, 200, 3000, 9216, 70000])
@pytest.mark.parametrize("e,eps,weight", [(-121, 1e-5, 0), (-121, 1e-5, 1), (-20, 1e-5, -101), (-130, 1e-12, 0), (-100, 1e-5, 0), (-101, 1e-8, 1)])
def test_codes_of_norms_of_tiny_rows(hiplib, dtype, cols, e, eps, weight):
    """Rows of values around 2^e, which eps makes larger: |y| is above 2^-116, where codes are promised, though 127 / max|h w| is
    past fp32's largest number (or h itself is a denormal).  weight: none, about 1, or about 2^weight."""
    g = U.rng(62)
    x = U.rounded(g.uniform(-1, 1, (4, cols)) * 2.0 ** e, dtype)
    x[:, 0] = 2.0 ** e
    r = U.rounded(g.uniform(-0.25, 0.25, (4, cols)) * 2.0 ** e, dtype)
    w = ((1 + 0.2 * g.uniform(-1, 1, cols)) * 2.0 ** (weight if weight < 0 else 0)).astype(np.float32) if weight else None
    _, y = norm64(x, r, w, eps)
    for group in (0, 32, 256):
        step = group or cols
        assert all(np.abs(y[:, i:i + step]).max(1).min() > 2.0 ** -116 for i in range(0, cols, step)) or cols % step
        c = Call(hiplib, x, r, w, dtype, group=group, eps=eps)
        check_codes(c, y, cols, group, chain(cols) + 8 * 2.0 ** -24)


@pytest.mark.parametrize("group", [0, 32])
@pytest.mark.parametrize("cols", [5, 3000, 70000])
def test_the_largest_number_comes_back_from_its_code(hiplib, cols, group):
    """Codes of rows with masks of fp32's lowest or largest value, and back: finite, each value within half a step of its group
    and what two roundings (the scale's, here up to a whole unit, and the product's) move 127 steps by."""
    g = U.rng(63)
    x = g.uniform(-1, 1, (3, cols)).astype(np.float32)
    x[:, 1::64] = np.array([np.finfo(np.float32).max, np.finfo(np.float32).min, 1e38], np.float32)[:, None]
    c = Call(hiplib, x, None, None, F32, group=group, norm=False)
    dq, ds, dy = U.Rows(hiplib, c.q), api.DeviceArray(hiplib, c.scale), U.Rows(hiplib, None, None, 0, x.shape, np.uint32)
    assert hiplib.thhip_dequantize_rows(dq.ptr, cols, ds.ptr, group, dy.ptr, cols, 3, cols, F32) == 0
    hiplib.thhip_sync()
    y = U.unraw(dy.get(), F32)
    assert np.isfinite(y).all()
    step = U.spread_x(c.scale.astype(np.float64), cols, group)
    assert (np.abs(y - x.astype(np.float64)) <= step * (0.5 + 127 * 3 * 2.0 ** -23)).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", [5, 200, 3000, 9216, 16388, 70000])
@pytest.mark.parametrize("kind,eps", [("masks", 1e-5), ("masks", 0.0), ("largest", 1e-5), (70, 1e-5), (-46, 0.0), (-60, 0.0), (-60, 2.0 ** -118),
                                      (-105, 0.0), (-126, 0.0), (-126, 1e-38)])
def test_norms_whose_squares_leave_fp32(hiplib, dtype, cols, kind, eps):
    """Masks of the type's lowest value beside ordinary ones, rows of the largest values, and rows whose squares are past fp32's
    smallest number with an eps that does not make up for them: sums, norms and codes are the formula's all the same."""
    g = U.rng(64)
    top = np.finfo(np.float32).max if dtype == F32 else np.float32((2 - 2.0 ** -7) * 2.0 ** 127)
    x = g.uniform(1, 2, (5, cols)) * g.choice([-1, 1], (5, cols))
    if kind == "masks":
        x[:4] *= 1024
        x[:4, 1::64] = -top         # (the last row has none)
    elif kind == "largest":
        x[:4] = top * np.sign(x[:4])
    else:
        x[:4] *= 2.0 ** kind
    x = U.rounded(x, dtype)
    w = (1 + 0.2 * g.uniform(-1, 1, cols)).astype(np.float32)
    h, y = norm64(x, None, w, eps)
    err = chain(cols) + 8 * 2.0 ** -24
    c = Call(hiplib, x, None, w, dtype, eps=eps)
    assert np.array_equal(c.sum, x)
    near(c.y, y, U.HALF_STEP[dtype] * (1 + 2.0 ** -8) + err, dtype, "y")
    c = Call(hiplib, x, None, w, dtype, group=0, eps=eps)
    assert np.array_equal(c.sum, x)
    check_codes(c, y, cols, 0, err)


@pytest.mark.parametrize("cols", [200, 3000, 9216, 70000])
@pytest.mark.parametrize("sum_to,y_to", [("r", "x"), ("x", "r")])
def test_rows_with_masks_in_place(hiplib, cols, sum_to, y_to):
    """Rows that are taken again times a power of two, into their own inputs: the bits of the call that writes elsewhere."""
    x, r, w = inputs(65, 4, cols, F32, True, True)
    x[1:3, 5::64] = np.finfo(np.float32).min
    want = Call(hiplib, x, r, w, F32)
    bufs = {"x": U.Rows(hiplib, U.raw(x, F32)), "r": U.Rows(hiplib, U.raw(r, F32))}
    dw = api.DeviceArray(hiplib, w)
    assert hiplib.thhip_rmsnorm(bufs["x"].ptr, cols, bufs["r"].ptr, cols, dw.ptr, EPS, bufs[sum_to].ptr, cols, bufs[y_to].ptr, cols,
                                4, cols, F32) == 0
    hiplib.thhip_sync()
    assert np.array_equal(U.unraw(bufs[sum_to].get(), F32), want.sum) and np.array_equal(U.unraw(bufs[y_to].get(), F32), want.y)
