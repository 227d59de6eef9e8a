"""4-bit Linear layers (thhip_linear_w4, thhip_linear_w4_i8, thhip_w4_pack, thhip_quantize_w4) against the plain product in
64 bits."""
import numpy as np
import pytest

import gpu_util as G
import w4_util as U
from thnets_amd import api
from w4_util import BF16, F16, F32

pytestmark = pytest.mark.gpu

TYPES = [F32, F16, BF16]

# B, nIn, nOut: one of everything, one short of and one past the packed blocks (16 rows, 128 k) and the batch slices
SHAPES = [(1, 1, 1), (1, 32, 16), (2, 33, 17), (1, 127, 5), (3, 128, 16), (5, 129, 31), (16, 512, 48), (17, 1000, 33), (15, 4090, 100),
          (33, 640, 80), (64, 1280, 65), (65, 256, 40), (1, 9216, 64), (1, 4096, 1000), (130, 384, 200), (257, 1100, 300), (128, 512, 128),
          (300, 2048, 256)]
GROUPS = [32, 64, 128, 256, 0]


def data(seed, B, nIn, nOut, dtype):
    g = U.rng(seed)
    return g, U.rounded(g.standard_normal((B, nIn), dtype=np.float32), dtype), (g.standard_normal(nOut) * 0.1).astype(np.float32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_shapes(hiplib, i, dtype):
    B, nIn, nOut = SHAPES[i]
    g, x, b = data(100 + i, B, nIn, nOut, dtype)
    layer = U.Layer.random(g, nOut, nIn, GROUPS[i % 5], dtype, i % 2 == 0).lay(hiplib)
    want, mag = U.linear64(layer, x, b)
    U.check_linear(U.linear(hiplib, layer, x, b), want, mag, layer)


@pytest.mark.parametrize("xgroup", [0, 1])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_shapes_i8(hiplib, i, dtype, xgroup):
    B, nIn, nOut = SHAPES[i]
    g, _, b = data(200 + i, B, nIn, nOut, dtype)
    layer = U.Layer.random(g, nOut, nIn, GROUPS[(i + 1) % 5], dtype, i % 2 == 1).lay(hiplib)
    q = g.integers(-128, 128, (B, nIn)).astype(np.int8)
    xs = (g.uniform(0.5, 1.5, (B, U.groups_of(nIn, layer.group) if xgroup else 1)) / 64).astype(np.float32)
    want, mag = U.linear64(layer, q * U.spread_x(xs.astype(np.float64), nIn, layer.group), b)
    got = U.linear(hiplib, layer, q, b, xs=xs, xgroup=layer.group if xgroup else 0)
    U.check_linear(got, want, mag, layer)


@pytest.fixture
def shape(hiplib):
    """Forces a workgroup shape for a test; the choice by size afterwards."""
    yield hiplib.thhip_w4_set_shape
    hiplib.thhip_w4_set_shape(-1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,nIn,nOut,group,zeros", [(21, 1280, 100, 128, 0), (70, 650, 130, 32, 1), (37, 2077, 257, 64, 0), (150, 384, 40, 0, 1)])
@pytest.mark.parametrize("which", range(6))
def test_every_shape(hiplib, shape, which, B, nIn, nOut, group, zeros, dtype):
    """Every shape of workgroup, also where the choice by size takes another: the tile kernel for few rows, one slice of the
    batch after the other for many."""
    g, x, b = data(1200 + which, B, nIn, nOut, dtype)
    layer = U.Layer.random(g, nOut, nIn, group, dtype, zeros).lay(hiplib)
    want, mag = U.linear64(layer, x, b)
    q = g.integers(-127, 128, (B, nIn)).astype(np.int8)
    xs = (g.uniform(0.5, 1.5, (B, U.groups_of(nIn, group))) / 64).astype(np.float32)
    want8, mag8 = U.linear64(layer, q * U.spread_x(xs.astype(np.float64), nIn, group), b)
    shape(which)
    U.check_linear(U.linear(hiplib, layer, x, b), want, mag, layer)
    U.check_linear(U.linear(hiplib, layer, q, b, xs=xs, xgroup=group), want8, mag8, layer)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("zeros", [0, 1])
@pytest.mark.parametrize("B", [1, 8, 20, 200])
def test_groups(hiplib, dtype, group, zeros, B):
    """Every group size with and without zero points; the last group is a part of one."""
    g, x, b = data(300 + group + B, B, 712, 50, dtype)
    layer = U.Layer.random(g, 50, 712, group, dtype, zeros).lay(hiplib)
    want, mag = U.linear64(layer, x, b)
    U.check_linear(U.linear(hiplib, layer, x, b), want, mag, layer)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("B", [1, 16, 17, 100, 260])
def test_small_integers_are_exact(hiplib, dtype, group, B):
    """Integers times powers of two whose sums stay below 2^24 units (scales are at least 2^-4; a row's own scale moves
    all of its sums alike): no rounding but the last, so the very bits."""
    g = U.rng(400 + B)
    x = g.integers(-8, 9, (B, 300)).astype(np.float32)
    layer = U.Layer.random(g, 70, 300, group, dtype, True, pow2=True).lay(hiplib)
    want, _ = U.linear64(layer, x)
    assert (np.abs(x) @ np.abs(layer.weights()).T).max() * 16 < 2 ** 24
    assert np.array_equal(U.linear(hiplib, layer, x), U.rounded(want, dtype))
    xs = np.exp2(g.integers(-2, 3, (B, 1))).astype(np.float32)
    q = g.integers(-128, 128, (B, 300)).astype(np.int8)
    want, _ = U.linear64(layer, q * xs.astype(np.float64))
    assert (np.abs(q.astype(np.float64)) @ np.abs(layer.weights()).T).max() * 16 < 2 ** 24
    assert np.array_equal(U.linear(hiplib, layer, q, xs=xs), U.rounded(want, dtype))


@pytest.mark.parametrize("B", [1, 5, 40, 150])
def test_fp32_values_keep_all_their_bits(hiplib, B):
    """One element of a row of x is not zero, with 24 random bits and exponents far apart: the output is its product with
    one weight.  n x and z x are sums of three exact products (two additions each), their difference and the scale round
    once more, each by at most 2^-23 of (n + z) |x| s."""
    g = U.rng(500)
    nIn = 260
    layer = U.Layer.random(g, 40, nIn, 64, F32, True).lay(hiplib)
    at = g.integers(0, nIn, B)
    v = (g.uniform(1, 2, B) * np.exp2(g.integers(-90, 90, B)) * g.choice([-1, 1], B)).astype(np.float32)
    x = np.zeros((B, nIn), np.float32)
    x[np.arange(B), at] = v
    want, mag = U.linear64(layer, x)
    assert (np.abs(U.linear(hiplib, layer, x) - want) <= 6 * 2.0 ** -23 * mag).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B", [1, 19, 140])
@pytest.mark.parametrize("ldx,offx,ldy,offy", [(520, 0, 64, 0), (513, 3, 61, 1), (512, 4, 60, 2), (528, 8, 72, 8)])
def test_strides_and_offsets(hiplib, dtype, B, ldx, offx, ldy, offy):
    """Rows apart and off every vector's alignment; what lies between and behind them (NaNs) is neither used nor written."""
    g, x, b = data(600, B, 500, 60, dtype)
    layer = U.Layer.random(g, 60, 500, 128, dtype, False).lay(hiplib)
    want, mag = U.linear64(layer, x, b)
    U.check_linear(U.linear(hiplib, layer, x, b, ldx=ldx, offx=offx, ldy=ldy, offy=offy), want, mag, layer)
    q = g.integers(-127, 128, (B, 500)).astype(np.int8)
    xs = np.full((B, 1), 0.03125, np.float32)
    want, mag = U.linear64(layer, q * 0.03125, b)
    U.check_linear(U.linear(hiplib, layer, q, b, ldx=ldx, offx=offx, ldy=ldy, offy=offy, xs=xs), want, mag, layer)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group,zeros", [(32, 1), (64, 0), (128, 1), (0, 0)])
@pytest.mark.parametrize("B,nOut", [(129, 200), (300, 257)])
def test_rows_of_whole_vectors_that_end_inside_a_step(hiplib, shape, B, nOut, group, zeros, dtype):
    """Rows that begin and end on 16 bytes, but not on 128 k, with NaNs behind each: the tile kernel's loads straight into
    LDS, for a single tile's columns and a part of a third's."""
    nIn, ldx = 656, 672
    g, x, b = data(620, B, nIn, nOut, dtype)
    layer = U.Layer.random(g, nOut, nIn, group, dtype, zeros).lay(hiplib)
    shape(5)
    want, mag = U.linear64(layer, x, b)
    U.check_linear(U.linear(hiplib, layer, x, b, ldx=ldx), want, mag, layer)
    q = g.integers(-127, 128, (B, nIn)).astype(np.int8)
    for xgroup in {0, group}:
        xs = (g.uniform(0.5, 1.5, (B, U.groups_of(nIn, xgroup))) / 64).astype(np.float32)
        want, mag = U.linear64(layer, q * U.spread_x(xs.astype(np.float64), nIn, group), b)
        U.check_linear(U.linear(hiplib, layer, q, b, ldx=ldx, xs=xs, xgroup=xgroup), want, mag, layer)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B", [1500, 2100])
def test_more_tiles_than_the_gpu_holds_at_once(hiplib, dtype, B):
    """Enough tiles for every form of launch that the size chooses among: one value in 50 is compared."""
    nIn, nOut = 384, 6000
    g, x, b = data(630, B, nIn, nOut, dtype)
    layer = U.Layer.random(g, nOut, nIn, 128, dtype, B == 1500).lay(hiplib)
    some = U.Layer(layer.codes[::50], layer.scales[::50], layer.zeros[::50] if layer.zeros is not None else None, 128, dtype)
    want, mag = U.linear64(some, x, b[::50])
    U.check_linear(U.linear(hiplib, layer, x, b)[:, ::50], want, mag, some)
    q = g.integers(-127, 128, (B, nIn)).astype(np.int8)
    xs = (g.uniform(0.5, 1.5, (B, 3)) / 64).astype(np.float32)
    want, mag = U.linear64(some, q * U.spread_x(xs.astype(np.float64), nIn, 128), b[::50])
    U.check_linear(U.linear(hiplib, layer, q, b, xs=xs, xgroup=128)[:, ::50], want, mag, some)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("zeros", [0, 1])
@pytest.mark.parametrize("group", GROUPS)
def test_scales_of_neighbouring_steps_in_large_launches(hiplib, shape, group, zeros, dtype):
    """More tiles than the GPU holds CUs, thirteen steps of K, the last one a part of one: a group's scales (and those of 8-bit x)
    are four or sixteen times those of its neighbours and of the groups two steps on, so that sums which met the scales of
    another step show.  Whole numbers times powers of two below 2^24 units: every output is compared, bit by bit."""
    B, nIn, nOut = 1100, 1552, 3750
    g = U.rng(640 + group)
    n = U.groups_of(nIn, group)
    scales = 0.25 ** ((np.arange(n)[None, :] + np.arange(nOut)[:, None]) % 3)
    z = g.integers(0, 16, (nOut, n)).astype(np.uint8) if zeros else None
    layer = U.Layer(g.integers(0, 16, (nOut, nIn)).astype(np.uint8), scales, z, group, dtype).lay(hiplib)
    w = layer.weights().astype(np.float32)
    x = g.integers(-4, 5, (B, nIn)).astype(np.float32)
    shape(5)
    # units of 2^-4 (with scales of 8-bit x 2^-5): 1552 * 15 * 4 * 2^5 < 2^24, so that fp32 sums are exact in any order
    assert np.array_equal(U.linear(hiplib, layer, x), U.rounded(x @ w.T, dtype))
    for xgroup in (0, group) if group else (0,):
        xs = (0.5 ** ((np.arange(U.groups_of(nIn, xgroup))[None, :] + np.arange(B)[:, None]) // 2 % 2)).astype(np.float32)
        want = (x * U.spread_x(xs, nIn, group)) @ w.T
        assert np.array_equal(U.linear(hiplib, layer, x.astype(np.int8), xs=xs, xgroup=xgroup), U.rounded(want, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("which", range(6))
@pytest.mark.parametrize("B", [1, 130])
def test_rows_that_end_with_their_allocation(hiplib, shape, which, B, dtype):
    """x, its scales, the weights and y lie at the very end of allocations of whole pages: what a kernel asks for past the
    last row has to stay inside."""
    nIn, nOut, pages = 4096, 40, 8 << 20
    g, x, b = data(650, B, nIn, nOut, dtype)
    q = g.integers(-127, 128, (B, nIn)).astype(np.int8)
    xs = (g.uniform(0.5, 1.5, (B, nIn // 128)) / 64).astype(np.float32)
    layer = U.Layer.random(g, nOut, nIn, 128, dtype, True).lay(hiplib)
    nbytes = hiplib.thhip_w4_packed_bytes(*layer.shape_args(), 1)
    raw = layer.packed.get((nbytes,), np.uint8)

    def at_end(words):
        dev = api.DeviceArray(hiplib, nbytes=pages)
        ptr = dev.ptr + pages - words.nbytes
        hiplib.thhip_memcpy_h2d(ptr, words.ctypes.data, words.nbytes)
        return dev, ptr

    kind = np.uint32 if dtype == F32 else np.uint16
    keep = [at_end(np.ascontiguousarray(w)) for w in (U.raw(x, dtype), q, xs, np.concatenate([raw, np.zeros(-nbytes % 16, np.uint8)]),
                                                      b, np.zeros((B, nOut), kind))]
    (_, px), (_, pq), (_, ps), (_, pw), (_, pb), (dy, py) = keep
    shape(which)
    tail = (pw, pb, py, nOut, B, nIn, nOut, 128, 1, 0, 0.0, 0.0, dtype)
    out = np.zeros((B, nOut), kind)
    G.note("at the end: B=%d shape=%d dtype=%d" % (B, which, dtype))
    assert hiplib.thhip_linear_w4(px, nIn, *tail) == 0
    hiplib.thhip_sync()
    hiplib.thhip_memcpy_d2h(out.ctypes.data, py, out.nbytes)
    U.check_linear(U.unraw(out, dtype), *U.linear64(layer, x, b), layer)
    assert hiplib.thhip_linear_w4_i8(pq, nIn, ps, 128, *tail) == 0
    hiplib.thhip_sync()
    hiplib.thhip_memcpy_d2h(out.ctypes.data, py, out.nbytes)
    U.check_linear(U.unraw(out, dtype), *U.linear64(layer, q * U.spread_x(xs.astype(np.float64), nIn, 128), b), layer)


def on_device(hiplib, nbytes, *parts):
    """A device buffer with (byte offset, array) parts written."""
    dev = api.DeviceArray(hiplib, nbytes=nbytes)
    for at, a in parts:
        hiplib.thhip_memcpy_h2d(dev.ptr + at, a.ctypes.data, a.nbytes)
    return dev


def from_device(hiplib, dev, at, shape, kind):
    out = np.zeros(shape, kind)
    hiplib.thhip_memcpy_d2h(out.ctypes.data, dev.ptr + at, out.nbytes)
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B", [2, 3, 40])
def test_rows_whose_distance_passes_32_bits(hiplib, dtype, B):
    """The first rows of x, and those of y, more than 2^32 bytes after another (three of them), or 2^24 elements, which are
    2^31 bytes for 128 rows of 8-bit codes (40)."""
    es = U.ESIZE[dtype]
    ld = (1 << 24) + 5 if B == 40 else (1 << 32) // es + 40
    nIn, nOut = 300, 37
    g, x, b = data(660, B, nIn, nOut, dtype)
    layer = U.Layer.random(g, nOut, nIn, 64, dtype, True).lay(hiplib)
    words, kind = U.raw(x, dtype), np.uint32 if dtype == F32 else np.uint16
    dx = on_device(hiplib, B * ld * es, *[(i * ld * es, words[i]) for i in range(B)])
    dy = api.DeviceArray(hiplib, nbytes=B * ld * es)
    db = api.DeviceArray(hiplib, b)
    G.note("far rows: B=%d ld=%d dtype=%d" % (B, ld, dtype))
    tail = (layer.packed.ptr, db.ptr, dy.ptr, ld, B, nIn, nOut, 64, 1, 0, 0.0, 0.0, dtype)
    assert hiplib.thhip_linear_w4(dx.ptr, ld, *tail) == 0
    hiplib.thhip_sync()
    out = np.concatenate([from_device(hiplib, dy, i * ld * es, (1, nOut), kind) for i in range(B)])
    U.check_linear(U.unraw(out, dtype), *U.linear64(layer, x, b), layer)
    q = g.integers(-127, 128, (B, nIn)).astype(np.int8)
    xs = (g.uniform(0.5, 1.5, (B, 1)) / 64).astype(np.float32)
    for i in range(B):
        hiplib.thhip_memcpy_h2d(dx.ptr + i * ld, q[i].ctypes.data, nIn)
    ds = api.DeviceArray(hiplib, xs)
    assert hiplib.thhip_linear_w4_i8(dx.ptr, ld, ds.ptr, 0, *tail) == 0
    hiplib.thhip_sync()
    out = np.concatenate([from_device(hiplib, dy, i * ld * es, (1, nOut), kind) for i in range(B)])
    U.check_linear(U.unraw(out, dtype), *U.linear64(layer, q * xs.astype(np.float64), b), layer)


@pytest.mark.parametrize("B", [1, 2, 50])
def test_more_outputs_than_a_launch_takes(hiplib, B):
    """2^24 + 300 outputs: the rows before and behind the border between two launches, and the last ones."""
    nIn, nOut, group = 40, (1 << 24) + 300, 32
    g = U.rng(670)
    x = U.rounded(g.standard_normal((B, nIn), dtype=np.float32), BF16)
    codes = g.integers(0, 256, (nOut, nIn // 2), dtype=np.uint8)
    s = U.rounded(g.uniform(0.5, 1.5, (nOut, 2)).astype(np.float32), BF16)
    z = g.integers(0, 16, (nOut, 2), dtype=np.uint8)
    b = g.standard_normal(nOut, dtype=np.float32)
    dc, ds, dz, db = (api.DeviceArray(hiplib, a) for a in (codes, U.raw(s, BF16), z, b))
    packed = api.DeviceArray(hiplib, nbytes=hiplib.thhip_w4_packed_bytes(nOut, nIn, group, BF16, 1))
    assert hiplib.thhip_w4_pack(dc.ptr, ds.ptr, dz.ptr, packed.ptr, nOut, nIn, group, BF16) == 0
    dx, dy = api.DeviceArray(hiplib, U.raw(x, BF16)), api.DeviceArray(hiplib, nbytes=B * nOut * 2)
    G.note("outputs of two launches: B=%d" % B)
    assert hiplib.thhip_linear_w4(dx.ptr, nIn, packed.ptr, db.ptr, dy.ptr, nOut, B, nIn, nOut, group, 1, 0, 0.0, 0.0, BF16) == 0
    hiplib.thhip_sync()
    for o in (0, (1 << 24) - 64, nOut - 128):
        part = slice(o, o + 128)
        layer = U.Layer(U.unpack_codes(codes[part], nIn), s[part], z[part], group, BF16)
        got = np.concatenate([from_device(hiplib, dy, (i * nOut + o) * 2, (1, 128), np.uint16) for i in range(B)])
        U.check_linear(U.unraw(got, BF16), *U.linear64(layer, x, b[part]), layer)


def test_more_rows_than_a_launch_takes(hiplib):
    """2^21 + 3 rows of four inputs and 656 outputs: more threads than one grid may have."""
    B, nIn, nOut = (1 << 21) + 3, 4, 656
    g = U.rng(680)
    x = g.standard_normal((B, nIn), dtype=np.float32)
    layer = U.Layer.random(g, nOut, nIn, 0, F32, True).lay(hiplib)
    dx, dy = api.DeviceArray(hiplib, x), api.DeviceArray(hiplib, nbytes=B * nOut * 4)
    G.note("rows of two launches")
    assert hiplib.thhip_linear_w4(dx.ptr, nIn, layer.packed.ptr, None, dy.ptr, nOut, B, nIn, nOut, 0, 1, 0, 0.0, 0.0, F32) == 0
    hiplib.thhip_sync()
    whole = 0xffffffff // 512 // 48 * 10        # (a launch's rows, near enough: the part around the border is compared)
    for i in (0, whole - 2000, 1 << 20, B - 3000):
        got = from_device(hiplib, dy, i * nOut * 4, (3000, nOut), np.float32)
        U.check_linear(got, *U.linear64(layer, x[i:i + 3000]), layer)


def test_the_largest_batch(hiplib, shape):
    """2^31 - 5 rows in tiles: the first, those around 2^30 and the last ones; a launch's first row is counted past 32 bits."""
    B, nIn, nOut = (1 << 31) - 5, 8, 1
    g = U.rng(690)
    layer = U.Layer.random(g, nOut, nIn, 0, F16, True).lay(hiplib)
    dx, dy = api.DeviceArray(hiplib, nbytes=B * nIn * 2), api.DeviceArray(hiplib, nbytes=B * 2)
    x = U.rounded(g.standard_normal((3000, nIn), dtype=np.float32), F16)
    words = U.raw(x, F16)
    some = (0, (1 << 30) - 1500, B - 3000)
    for i in some:
        hiplib.thhip_memcpy_h2d(dx.ptr + i * nIn * 2, words.ctypes.data, words.nbytes)
    G.note("the largest batch")
    shape(5)
    assert hiplib.thhip_linear_w4(dx.ptr, nIn, layer.packed.ptr, None, dy.ptr, nOut, B, nIn, nOut, 0, 1, 0, 0.0, 0.0, F16) == 0
    hiplib.thhip_sync()
    want = U.linear64(layer, x)
    for i in some:
        U.check_linear(U.unraw(from_device(hiplib, dy, i * 2, (3000, nOut), np.uint16), F16), *want, layer)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B", [1, 18, 129])
def test_threshold(hiplib, dtype, B):
    g, x, b = data(700, B, 384, 45, dtype)
    layer = U.Layer.random(g, 45, 384, 128, dtype, False).lay(hiplib)
    plain = U.linear(hiplib, layer, x, b)
    # (fp32 is compared before it is rounded, so values at the border itself are left out for the half types)
    got = U.linear(hiplib, layer, x, b, act=1, thr=0.25, val=-1.5)
    clear = np.abs(plain - 0.25) > 2 ** -8
    assert np.array_equal(got[clear], np.where(plain > 0.25, plain, np.float32(-1.5))[clear])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B", [3, 33, 200])
def test_a_row_with_nan_stays_alone(hiplib, dtype, B):
    g, x, _ = data(800, B, 512, 40, dtype)
    layer = U.Layer.random(g, 40, 512, 128, dtype, False).lay(hiplib)
    clean = U.linear(hiplib, layer, x)
    x[1, 77] = np.nan
    x[2, 300] = np.inf
    got = U.linear(hiplib, layer, x)
    assert np.isnan(got[1]).all() and not np.isfinite(got[2]).any()
    rest = np.arange(B) > 2
    assert np.array_equal(got[rest], clean[rest]) and np.array_equal(got[0], clean[0])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("group,zeros", [(32, 1), (128, 0), (128, 1), (0, 1)])
@pytest.mark.parametrize("B,which", [(1, -1), (5, -1), (16, -1), (40, 0), (40, 1), (40, 2), (40, 3), (40, 4), (40, 5), (200, 5)])
def test_x_at_the_ends_of_the_range(hiplib, shape, B, which, group, zeros, dtype):
    """Rows of the type's lowest and largest values, alone or as a few masks beside ordinary values, in a layer whose outputs are
    numbers (1300 * 15 * 2^-16 of the largest one at most); and rows of values around 2^-100 and 2^-112."""
    nIn, nOut = 1300, 50
    g = U.rng(850)
    top = np.finfo(np.float32).max if dtype == F32 else np.float32((2 - 2.0 ** -7) * 2.0 ** 127)
    layer = U.Layer.random(g, nOut, nIn, group, dtype, zeros)
    layer = U.Layer(layer.codes, 2.0 ** -17 * g.uniform(1, 2, layer.scales.shape), layer.zeros, group, dtype).lay(hiplib)
    shape(which)
    x = g.standard_normal((B, nIn), dtype=np.float32)
    x[:, 3::97] = -top
    for v in (x, np.full((B, nIn), top), g.choice([-top, top, top / 2], (B, nIn)), g.standard_normal((B, nIn)) * 2.0 ** -100,
              g.standard_normal((B, nIn)) * 2.0 ** -112):
        v = U.rounded(v, dtype)
        want, mag = U.linear64(layer, v)
        U.check_linear(U.linear(hiplib, layer, v), want, mag, layer)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B", [1, 40, 300])
def test_twice_the_same_bits_and_nothing_allocated(hiplib, dtype, B):
    g, x, b = data(900, B, 2048, 256, dtype)
    layer = U.Layer.random(g, 256, 2048, 128, dtype, False).lay(hiplib)
    first = U.linear(hiplib, layer, x, b)
    assert np.array_equal(U.linear(hiplib, layer, x, b), first)
    dx, dy = U.Rows(hiplib, U.raw(x, dtype)), api.DeviceArray(hiplib, nbytes=B * 256 * 4)
    before = hiplib.thhip_alloc_calls()
    assert hiplib.thhip_linear_w4(dx.ptr, dx.ld, layer.packed.ptr, None, dy.ptr, 256, B, 2048, 256, 128, 0, 0, 0.0, 0.0, dtype) == 0
    assert hiplib.thhip_alloc_calls() == before
    hiplib.thhip_sync()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("wtype", TYPES)
@pytest.mark.parametrize("group,zeros,nIn", [(32, 0, 300), (64, 1, 333), (128, 1, 512), (256, 0, 700), (0, 1, 97)])
def test_quantize(hiplib, dtype, wtype, group, zeros, nIn):
    """Codes, scales and zeros are those of the formula, up to a code's choice at the middle between two; a constant-zero
    group is 0; the layer made of them is within half a step of the weights (plus what a rounded scale moves)."""
    g = U.rng(1000)
    nOut, ldw = 21, nIn + 5
    w = U.rounded(g.standard_normal((nOut, nIn)) * 0.05 + 0.02, wtype)
    w[3] = 0
    n = U.groups_of(nIn, group)
    dw = U.Rows(hiplib, U.raw(w, wtype), ldw)
    dc = U.Rows(hiplib, None, None, 0, (nOut, (nIn + 1) // 2), np.uint8)
    ds = U.Rows(hiplib, None, None, 0, (nOut, n), np.uint32 if dtype == F32 else np.uint16)
    dz = U.Rows(hiplib, None, None, 0, (nOut, n), np.uint8)
    assert hiplib.thhip_quantize_w4(dw.ptr, ldw, wtype, dc.ptr, ds.ptr, dz.ptr if zeros else None, nOut, nIn, group, dtype) == 0
    hiplib.thhip_sync()
    codes, s = U.unpack_codes(dc.get(), nIn), U.unraw(ds.get(), dtype).astype(np.float64)
    z = dz.get().astype(np.float64) if zeros else np.full((nOut, n), 8.0)
    step = group or nIn
    for i in range(n):
        part = w[:, i * step:(i + 1) * step].astype(np.float64)
        lo, hi = np.minimum(part.min(1), 0), np.maximum(part.max(1), 0)
        top = (hi - lo) / 15 if zeros else np.maximum(hi, -lo) / 7
        assert (np.abs(s[:, i] - top) <= (2 * U.HALF_STEP[dtype] + 2.0 ** -22) * top).all()
        some = s[:, i] > 0
        assert np.array_equal(some, np.arange(nOut) != 3)
        exact = part[some] / s[some, i:i + 1] + z[some, i:i + 1]
        if zeros:
            assert (np.abs(z[some, i] - np.minimum(-lo[some] / s[some, i], 15)) <= 0.5 + 1e-5).all()
        got = codes[some, i * step:(i + 1) * step]
        assert (np.abs(got - np.clip(exact, 0, 15)) <= 0.5 + 1e-4).all()
        assert (codes[3, i * step:(i + 1) * step] == z[3, i]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("zeros", [0, 1])
def test_quantize_at_the_ends_of_the_range(hiplib, dtype, zeros):
    """Rows of weights from the smallest numbers to fp32's largest: scales are finite and codes those of w / s; a row whose
    scale is under 2^-128, or 0 in its type, stands for 0."""
    nIn, tops = 64, np.array([0, 1e-45, 2.0 ** -130, 2.0 ** -120, 2.0 ** -30, 2.0 ** -20, 1e5, 4e5, 1e9, 3.4e38])
    g = U.rng(1010)
    w = (g.uniform(-1, 1, (len(tops), nIn)) * tops[:, None]).astype(np.float32)
    w[:, 0], w[:, 1] = tops, -tops
    dw, dc, ds, dz = (api.DeviceArray(hiplib, nbytes=n) for n in (w.nbytes, len(tops) * 32, len(tops) * 4, len(tops)))
    hiplib.thhip_memcpy_h2d(dw.ptr, w.ctypes.data, w.nbytes)
    assert hiplib.thhip_quantize_w4(dw.ptr, nIn, F32, dc.ptr, ds.ptr, dz.ptr if zeros else None, len(tops), nIn, 64, dtype) == 0
    hiplib.thhip_sync()
    s = U.unraw(ds.get((len(tops),), np.uint32 if dtype == F32 else np.uint16), dtype).astype(np.float64)
    codes = U.unpack_codes(dc.get((len(tops), 32), np.uint8), nIn).astype(np.float64)
    z = dz.get((len(tops),), np.uint8).astype(np.float64) if zeros else np.full(len(tops), 8.0)
    assert np.isfinite(s).all()
    top = tops.astype(np.float32).astype(np.float64) * (2 / 15 if zeros else 1 / 7)
    for i in range(len(tops)):
        if s[i] < 2.0 ** -128:
            assert top[i] < 2.0 ** -127 + U.TINY[dtype] * 1.01 and (codes[i] == z[i]).all()
        else:
            # (an fp16 scale near the smallest is off by half a step of the denormals)
            want = min(top[i], 65504) if dtype == F16 else top[i]
            assert abs(s[i] - want) <= 2 * U.HALF_STEP[dtype] * want + U.TINY[dtype]
            exact = w[i].astype(np.float64) / s[i] + z[i]
            assert (np.abs(codes[i] - np.clip(exact, 0, 15)) <= 0.5 + 1e-4).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("zeros", [0, 1])
def test_quantize_in_the_middle_between_codes(hiplib, dtype, zeros):
    """Scales that are odd numbers, so that w / s is a whole number and a half without any rounding, and weights a unit of fp32
    beside those: every code and zero point is rint(w / s) (the even one in the middle), as a quotient in 64 bits has it."""
    s0 = np.arange(1, 256, 2)
    nIn, nOut = 64, len(s0)
    w = np.zeros((nOut, nIn), np.float32)
    halves = np.arange(-7, 7) + 0.5
    w[:, 1:15] = halves * s0[:, None]
    w[:, 15:29], w[:, 29:43] = np.nextafter(w[:, 1:15], np.float32(99999)), np.nextafter(w[:, 1:15], np.float32(-99999))
    w[:, 0] = (8 if zeros else 7) * s0
    w[:, 43] = -7 * s0
    dw, dc, ds, dz = (api.DeviceArray(hiplib, nbytes=n) for n in (w.nbytes, nOut * 32, nOut * 4, nOut))
    hiplib.thhip_memcpy_h2d(dw.ptr, w.ctypes.data, w.nbytes)
    assert hiplib.thhip_quantize_w4(dw.ptr, nIn, F32, dc.ptr, ds.ptr, dz.ptr if zeros else None, nOut, nIn, 64, dtype) == 0
    hiplib.thhip_sync()
    s = U.unraw(ds.get((nOut,), np.uint32 if dtype == F32 else np.uint16), dtype).astype(np.float64)[:, None]
    assert (np.abs(s[:, 0] - s0) <= 2.0 ** -23 * s0).all() and (zeros or (s[:, 0] == s0).all())
    z = dz.get((nOut,), np.uint8).astype(np.float64)[:, None] if zeros else 8
    if zeros:
        assert np.array_equal(z, np.rint(7 * s0[:, None] / s))
    codes = U.unpack_codes(dc.get((nOut, 32), np.uint8), nIn)
    assert np.array_equal(codes, np.clip(np.rint(w.astype(np.float64) / s) + z, 0, 15))


@pytest.mark.parametrize("dtype", TYPES)
def test_from_weights_to_outputs(hiplib, dtype):
    """quantise, pack and multiply in one go, as a program does; the product is that of the weights the codes stand for."""
    g, x, b = data(1100, 9, 640, 72, dtype)
    w = U.rounded(g.standard_normal((72, 640)) * 0.05, dtype)
    dw = U.Rows(hiplib, U.raw(w, dtype))
    dc, ds, dz = (api.DeviceArray(hiplib, nbytes=n) for n in (72 * 320, 72 * 10 * 4, 72 * 10))
    assert hiplib.thhip_quantize_w4(dw.ptr, 640, dtype, dc.ptr, ds.ptr, dz.ptr, 72, 640, 64, dtype) == 0
    layer = U.Layer(U.unpack_codes(dc.get((72, 320), np.uint8), 640), U.unraw(ds.get((72, 10), np.uint32 if dtype == F32 else np.uint16), dtype),
                    dz.get((72, 10), np.uint8), 64, dtype)
    layer.packed = api.DeviceArray(hiplib, nbytes=hiplib.thhip_w4_packed_bytes(72, 640, 64, dtype, 1))
    assert hiplib.thhip_w4_pack(dc.ptr, ds.ptr, dz.ptr, layer.packed.ptr, 72, 640, 64, dtype) == 0
    want, mag = U.linear64(layer, x, b)
    U.check_linear(U.linear(hiplib, layer, x, b), want, mag, layer)
    # half a step of 4 bits is a thirtieth of the range: the float layer's outputs are near
    assert np.linalg.norm(want - (x.astype(np.float64) @ w.T.astype(np.float64) + b)) < 0.1 * np.linalg.norm(want)
