"""Device and host sides of strided rows in fp32, fp16 and bf16 for the tests of the row operators."""
import numpy as np

from ngraph_hip.runtime import NGH_F32, NGH_F16, NGH_BF16

f32, f64 = np.float32, np.float64
DTYPES = {"f32": NGH_F32, "f16": NGH_F16, "bf16": NGH_BF16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
#: half a step relative to the value: the most one rounding to the type is off
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
#: half the smallest step (below the normal numbers)
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}
EPS = 2.0 ** -24
CANARY = 0xC5


def to_storage(x, dtype):
    """fp32 values as the type stores them (round to nearest even)."""
    x = np.ascontiguousarray(x, dtype=f32)
    if dtype == "f32":
        return x
    if dtype == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    bits = x.view(np.uint32)
    nan = np.isnan(x)
    out = ((bits.astype(np.uint64) + 0x7fff + ((bits >> 16) & 1)) >> 16).astype(np.uint16)
    out[nan] = 0x7fc0
    return out


def from_storage(s, dtype):
    """Stored values as fp32 (exact)."""
    if dtype == "bf16":
        return (s.astype(np.uint32) << 16).view(f32)
    return s.astype(f32)


def rounded(x, dtype):
    """fp32 values rounded to what the type holds."""
    return from_storage(to_storage(x, dtype), dtype)


class Rows(object):
    """[rows, width] values on the device with a row stride and a start `shift` elements behind an
    allocation's; what lies between and behind the rows is a canary."""

    def __init__(self, rt, shape, dtype="f32", stride=None, shift=0, values=None):
        self.rt, self.dtype, self.shift = rt, dtype, shift
        self.rows, self.width = shape
        self.stride = self.width if stride is None else stride
        self.count = shift + max(0, self.rows - 1) * self.stride + self.width + 64
        self.host = np.full(self.count * SIZE[dtype], CANARY, np.uint8)
        if values is not None:
            self._window(self.host)[...] = to_storage(values, dtype).reshape(self.rows, self.width)
        self.base = rt.malloc(self.host.nbytes)
        rt.memcpy_h2d(self.base, self.host)
        self.ptr = self.base + shift * SIZE[dtype]

    def _window(self, raw):
        store = {"f32": f32, "f16": np.float16, "bf16": np.uint16}[self.dtype]
        flat = raw.view(store)[self.shift:]
        return np.lib.stride_tricks.as_strided(flat, (self.rows, self.width), (self.stride * flat.itemsize, flat.itemsize))

    def raw(self):
        out = np.empty_like(self.host)
        self.rt.memcpy_d2h(out, self.base)
        return out

    def get(self):
        """The values, after checking that nothing outside the rows changed."""
        raw = self.raw()
        before, after = self.host.copy(), raw.copy()
        if self.rows:
            self._window(before)[...] = 0
            self._window(after)[...] = 0
        np.testing.assert_array_equal(after, before, err_msg="memory outside the rows was written")
        return from_storage(self._window(raw).copy(), self.dtype) if self.rows else np.zeros((0, self.width), f32)

    def free(self):
        if self.base:
            self.rt.free(self.base)
            self.base = None


class Pool(object):
    """Allocations of a test, freed together."""

    def __init__(self, rt):
        self.rt, self.items = rt, []

    def rows(self, shape, dtype="f32", values=None, stride=None, shift=0):
        r = Rows(self.rt, shape, dtype, stride, shift, values)
        self.items.append(r)
        return r

    def array(self, host):
        a = self.rt.array(np.ascontiguousarray(host))
        self.items.append(a)
        return a

    def bytes(self, n):
        a = self.rt.empty((max(int(n), 16),), 7)
        self.items.append(a)
        return a

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for i in self.items:
            i.free()


def assert_within(got, want, bound, what=""):
    got, want, bound = (np.asarray(v, dtype=f64) for v in (got, want, bound))
    off = np.abs(got - want)
    bad = ~(off <= bound)
    assert not bad.any(), "%s: %d of %d values off, the worst %.3g beyond a bound of %.3g (got %r, want %r)" % (
        what, bad.sum(), bad.size, float(np.nanmax(np.where(bad, off, 0))), float(np.broadcast_to(bound, bad.shape)[bad][0]),
        got[bad][0], want[bad][0])
