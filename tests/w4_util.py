"""4-bit Linear layers and rows of codes on numpy data: plain forms in 64 bits, and calls of the C ABI with
strides, offsets and guarded surroundings of the caller's choice."""
import numpy as np

import cases
import gpu_util as G
from thnets_amd import api

F32, F16, BF16 = G.F32, G.F16, G.BF16
ESIZE = {F32: 4, F16: 2, BF16: 2}
# half a step of the type, relative to the value
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
# half a step of the type's denormals (fp32 and bf16: nothing here comes near them)
TINY = {F32: 0.0, F16: 2.0 ** -25, BF16: 0.0}


def groups_of(n, group):
    return 1 if group == 0 else -(-n // group)


def rounded(a, dtype):
    """float32 values of `a` in the engine's type."""
    a = np.ascontiguousarray(a, np.float32)
    if dtype == F32:
        return a
    if dtype == F16:
        return a.astype(np.float16).astype(np.float32)
    return (api._bf16_bits(a).astype(np.uint32) << 16).view(np.float32)


def raw(a, dtype):
    """The bytes of float32 values in the engine's type, as unsigned integers."""
    a = np.ascontiguousarray(a, np.float32)
    if dtype == F32:
        return a.view(np.uint32)
    if dtype == F16:
        return a.astype(np.float16).view(np.uint16)
    return api._bf16_bits(a)


def unraw(u, dtype):
    if dtype == F32:
        return u.view(np.float32)
    if dtype == F16:
        return u.view(np.float16).astype(np.float32)
    return (u.astype(np.uint32) << 16).view(np.float32)


NAN_BYTE = 0xFF     # fp32, fp16 and bf16 words of ones are NaNs; as a code it is -1


class Rows:
    """rows x cols elements on the device, `ld` apart, `offset` elements behind the allocation's start, with
    bytes of ones around and between them; check() finds whether anything but the rows was written."""

    def __init__(self, lib, words, ld=None, offset=0, shape=None, kind=None):
        rows, cols = shape if words is None else words.shape
        kind = words.dtype if words is not None else kind
        self.shape, self.kind, self.offset = (rows, cols), np.dtype(kind), offset
        self.ld = ld or cols
        n = offset + rows * self.ld + 64
        self.image = np.full(n * self.kind.itemsize, NAN_BYTE, np.uint8).view(self.kind)
        if words is not None:
            self.rows_of(self.image)[:] = words
        self.dev = api.DeviceArray(lib, self.image)
        self.ptr = self.dev.ptr + offset * self.kind.itemsize

    def rows_of(self, image):
        rows, cols = self.shape
        return image[self.offset:self.offset + rows * self.ld].reshape(rows, self.ld)[:, :cols]

    def get(self):
        """The rows now; everything around them has to be as it was."""
        now = self.dev.get(self.image.shape, self.kind)
        rows = self.rows_of(now).copy()
        self.rows_of(now)[:] = self.rows_of(self.image)
        assert np.array_equal(now, self.image), "written outside the rows"
        return rows


def pack_codes(n):
    """One code a value -> two in a byte, the even k low."""
    nOut, nIn = n.shape
    if nIn % 2:
        n = np.concatenate([n, np.zeros((nOut, 1), n.dtype)], 1)
    return (n[:, 0::2] | (n[:, 1::2] << 4)).astype(np.uint8)


def unpack_codes(b, nIn):
    return np.stack([b & 15, b >> 4], -1).reshape(b.shape[0], -1)[:, :nIn]


class Layer:
    """A 4-bit layer: codes, scales (values of `dtype`) and zeros or None, packed on the device by lay()."""

    def __init__(self, codes, scales, zeros, group, dtype):
        self.codes, self.scales, self.zeros, self.group, self.dtype = codes, rounded(scales, dtype), zeros, group, dtype
        self.nOut, self.nIn = codes.shape

    @classmethod
    def random(cls, g, nOut, nIn, group, dtype, zeros, pow2=False):
        n = groups_of(nIn, group)
        s = np.exp2(g.integers(-4, 3, (nOut, n))) if pow2 else g.uniform(0.5, 1.5, (nOut, n)) / np.sqrt(nIn)
        z = g.integers(0, 16, (nOut, n)).astype(np.uint8) if zeros else None
        return cls(g.integers(0, 16, (nOut, nIn)).astype(np.uint8), s, z, group, dtype)

    def spread(self, v):
        return np.repeat(v, self.group or self.nIn, 1)[:, :self.nIn]

    def weights(self):
        z = self.spread(self.zeros.astype(np.float64)) if self.zeros is not None else 8.0
        return (self.codes - z) * self.spread(self.scales.astype(np.float64))

    def magnitudes(self):
        """s (n + z): what the two sums that a weight's products are made of amount to."""
        z = self.spread(self.zeros.astype(np.float64)) if self.zeros is not None else 8.0
        return (self.codes + z) * np.abs(self.spread(self.scales.astype(np.float64)))

    def shape_args(self):
        return (self.nOut, self.nIn, self.group, self.dtype)

    def lay(self, lib):
        hz = 0 if self.zeros is None else 1
        self.packed = api.DeviceArray(lib, nbytes=lib.thhip_w4_packed_bytes(*self.shape_args(), hz))
        dc = api.DeviceArray(lib, pack_codes(self.codes))
        ds = api.DeviceArray(lib, raw(self.scales, self.dtype))
        dz = api.DeviceArray(lib, self.zeros) if hz else None
        assert lib.thhip_w4_pack(dc.ptr, ds.ptr, dz.ptr if dz else None, self.packed.ptr, *self.shape_args()) == 0
        lib.thhip_sync()
        return self


def spread_x(xs, nIn, group):
    return np.repeat(xs, group or nIn, 1)[:, :nIn] if xs.shape[1] > 1 else np.repeat(xs, nIn, 1)


def linear(lib, layer, x, bias=None, act=0, thr=0.0, val=0.0, ldx=None, ldy=None, offx=0, offy=0, xs=None, xgroup=0):
    """thhip_linear_w4 (x: float values) or, with xs, thhip_linear_w4_i8 (x: codes); y as float32."""
    B = x.shape[0]
    G.note("linear_w4%s B=%d %d->%d group=%d zeros=%d dtype=%d ldx=%s offx=%d act=%d" % (
        "_i8" if xs is not None else "", B, layer.nIn, layer.nOut, layer.group, layer.zeros is not None, layer.dtype, ldx, offx, act))
    dx = Rows(lib, x if xs is not None else raw(x, layer.dtype), ldx, offx)
    dy = Rows(lib, None, ldy, offy, (B, layer.nOut), np.uint32 if layer.dtype == F32 else np.uint16)
    db = api.DeviceArray(lib, np.ascontiguousarray(bias, np.float32)) if bias is not None else None
    tail = (layer.packed.ptr, db.ptr if db else None, dy.ptr, dy.ld, B, layer.nIn, layer.nOut, layer.group,
            0 if layer.zeros is None else 1, act, thr, val, layer.dtype)
    if xs is None:
        assert lib.thhip_linear_w4(dx.ptr, dx.ld, *tail) == 0
    else:
        ds = api.DeviceArray(lib, np.ascontiguousarray(xs, np.float32))
        assert lib.thhip_linear_w4_i8(dx.ptr, dx.ld, ds.ptr, xgroup, *tail) == 0
    lib.thhip_sync()
    dx.get()        # (the input as it was)
    return unraw(dy.get(), layer.dtype)


def linear64(layer, x, bias=None):
    """(the layer's outputs, the sum of the magnitudes that went into each) in 64 bits."""
    y = x.astype(np.float64) @ layer.weights().T
    return (y if bias is None else y + bias.astype(np.float64)), np.abs(x).astype(np.float64) @ layer.magnitudes().T


def check_linear(got, want, mag, layer, what=""):
    """Every output within what its roundings can add up to, and all together within what they add up to at random.

    Worst case: each of the products of a group (128 at most between two roundings to the result) and each group's sum
    is added to a sum no larger than `mag`, with an error of at most one unit (2^-23: the matrix core may cut off)
    of it; the groups follow one another in chains of at most steps / 4 and 16 further additions.
    At random: within a group the 16 additions of matrix instructions go wrong by 2^-23 of a sum that is about three
    times the group's result, 16 * 3 * 2^-24 = 3e-6 if they all lean the same way; plus half a step of y's type."""
    steps = -(-layer.nIn // 128)
    half = HALF_STEP[layer.dtype]
    bound = half * np.abs(want) * (1 + 2.0 ** -10) + TINY[layer.dtype] + (128 + steps / 4 + 16) * 2.0 ** -23 * mag
    off = np.abs(got - want)
    assert np.isfinite(got).all() and (off <= bound).all(), "%s: off by %.3g where %.3g is allowed" % (
        what, off.max(), bound.flat[off.argmax()])
    rel = np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-30)
    if want.size >= 64:
        assert rel <= 4e-6 + half, "%s: 2-norm off by %.3g" % (what, rel)


def rng(seed):
    return cases.rng(seed)
