"""ngh_block_norm / ngh_block_norm_grad against NumPy in float64.

Bounds.  A sum over a row adds at most 16 values a lane, 6 levels of lanes and 16 wavefronts, so that
with the elementwise steps around it no result has more than K = 64 roundings of 2^-24 in a row, each
relative to the magnitudes that meet there; `magnitudes` below carries those sums of absolute values
along the formulas (a mean is off relative to the mean magnitude; a norm's reciprocal root relative to
what the squares are off, the factor `amp`).  Sums over rows add K + rows.  Then one rounding to the
result's type.
"""
import numpy as np
import pytest

from row_helpers import DTYPES, EPS, HALF, TINY, Pool, assert_within, rounded

pytestmark = pytest.mark.gpu

f32, f64 = np.float32, np.float64
K = 64
TYPES = [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f16", "f16")]       # rows, parameters


def mean(x):
    return x.mean(axis=1, keepdims=True)


def norm64(x, size, layer, eps):
    """N(x), the reciprocal root, the magnitude of N(x) and the growth of what x is off by."""
    m = mean(x) if layer else 0.0
    c = x - m
    r = 1.0 / np.sqrt(mean(c * c) + eps)
    size = size + (mean(size) if layer else 0.0)
    amp = 1.0 + mean(size * size) * r * r
    return c * r, r, size * r * amp, amp


class Case(object):
    def __init__(self, rows, width, kind="rms", types=("f32", "f32"), post=True, gate_rows=0, bias=False, alpha=1.0, block=True, gains=True,
                 eps=1e-5, offset=0.1, seed=0):
        self.rows, self.width, self.layer, self.types = rows, width, kind == "layer", types
        self.kind, self.post, self.gate_rows, self.alpha, self.eps = kind, post and block, gate_rows, f64(f32(alpha)), f64(f32(eps))
        rs = np.random.RandomState(seed)
        act = lambda std, mean: rounded(rs.normal(mean, std, (rows, width)), types[0])                # noqa: E731
        vec = lambda n, std, mean: rounded(rs.normal(mean, std, (n, width)), types[1])                # noqa: E731
        self.values = {"x": act(1.5, offset), "dy": act(0.5, 0.05), "dh": act(0.5, -0.02), "gain": vec(1, 0.2, 1.0) if gains else None,
                       "bias": vec(1, 0.3, 0.0) if bias else None}
        self.values["b"] = act(0.7, -offset) if block else None
        self.values["post_gain"] = vec(1, 0.2, 1.0) if self.post and gains else None
        self.values["post_bias"] = vec(1, 0.3, 0.0) if self.post and bias else None
        self.values["gate"] = vec(rows // gate_rows, 0.3, 0.5) if gate_rows and block else None

    def get(self, name, other):
        v = self.values[name]
        return other if v is None else v.astype(f64)

    def branch(self):
        """bh, its root, magnitude and amp; u and its magnitude."""
        b = self.values["b"].astype(f64)
        bh, r, size, amp = norm64(b, np.abs(b), self.layer, self.eps) if self.post else (b, 1.0, np.abs(b), 1.0)
        p, q = self.get("post_gain", 1.0), self.get("post_bias", 0.0)
        return bh, r, size, amp, bh * p + q, size * np.abs(p) + np.abs(q)

    def gates(self):
        g = self.get("gate", None)
        return 1.0 if g is None else np.repeat(g, self.gate_rows, axis=0)

    def forward(self):
        """{name: (value, bound before the rounding to the type)}"""
        x = self.values["x"].astype(f64)
        h, size = self.alpha * x, np.abs(self.alpha * x)
        if self.values["b"] is not None:
            _, _, _, _, u, usize = self.branch()
            h, size = h + self.gates() * u, size + np.abs(self.gates()) * usize
        hh, _, hsize, _ = norm64(h, size, self.layer, self.eps)
        w, z = self.get("gain", 1.0), self.get("bias", 0.0)
        return {"h": (h, K * EPS * size), "y": (hh * w + z, K * EPS * (hsize * np.abs(w) + np.abs(z)))}

    def backward(self, h):
        dy, dh, h = self.values["dy"].astype(f64), self.values["dh"].astype(f64), h.astype(f64)
        out = {}
        hh, r, hsize, amp = norm64(h, np.abs(h), self.layer, self.eps)
        w = self.get("gain", 1.0)

        def through(t, tsize, xh, r, xsize, amp):
            v = t - xh * mean(t * xh)
            s = tsize + xsize * mean(tsize * xsize)
            if self.layer:
                v, s = v - mean(t), s + mean(tsize)
            return r * v, r * s * amp

        d, dsize = through(dy * w, np.abs(dy * w), hh, r, hsize, amp)
        d, dsize = d + dh, dsize + np.abs(dh)
        k = (K + self.rows) * EPS
        out["dgain"] = ((dy * hh).sum(0), k * (np.abs(dy) * hsize).sum(0))
        out["dbias"] = (dy.sum(0), k * np.abs(dy).sum(0))
        out["dx"] = (self.alpha * d, K * EPS * np.abs(self.alpha) * dsize)
        if self.values["b"] is None:
            return out
        bh, rb, bsize, bamp, u, usize = self.branch()
        if self.gate_rows:
            shape = (self.rows // self.gate_rows, self.gate_rows, self.width)
            out["dgate"] = ((d * u).reshape(shape).sum(1), (2 * K + self.gate_rows) * EPS * (dsize * usize).reshape(shape).sum(1))
        e, esize = d * self.gates(), dsize * np.abs(self.gates())
        p = self.get("post_gain", 1.0)
        out["dpost_gain"] = ((e * bh).sum(0), (2 * K + self.rows) * EPS * (esize * bsize).sum(0))
        out["dpost_bias"] = (e.sum(0), (2 * K + self.rows) * EPS * esize.sum(0))
        if self.post:
            t, tsize = through(e * p, esize * np.abs(p), bh, rb, bsize, bamp)
            out["db"] = (t, 2 * K * EPS * tsize)
        else:
            out["db"] = (e, 2 * K * EPS * esize)
        return out


ROWS = ("x", "b", "h", "y", "dy", "dh", "dx", "db")


def place(pool, case, name, values, strides, shift):
    if name in ROWS:
        return pool.rows((case.rows, case.width), case.types[0], values, strides.get(name), shift)
    n = case.rows // case.gate_rows if name in ("gate", "dgate") else 1
    return pool.rows((n, case.width), case.types[1], values, strides.get(name) if name in ("gate", "dgate") else None, shift)


def make_spec(rt, case, tensors, **more):
    names = {k: t.ptr for k, t in tensors.items()}
    strides = {k + "_stride": t.stride for k, t in tensors.items() if k in ROWS + ("gate", "dgate")}
    return rt.block_norm_spec(case.rows, case.width, case.kind, DTYPES[case.types[0]], DTYPES[case.types[1]], case.post,
                              case.gate_rows if "gate" in tensors else 0, float(case.alpha), float(case.eps), **dict(names, **strides), **more)


def check(got, want, bound, dtype, what):
    assert_within(got, want, bound * 1.01 + (np.abs(want) + bound) * HALF[dtype] + TINY[dtype], what)


def run_forward(rt, case, strides={}, shift=0, inplace=False, drop=()):
    with Pool(rt) as pool:
        tensors = {n: place(pool, case, n, case.values[n], strides, shift) for n in ("x", "b", "gain", "bias", "post_gain", "post_bias", "gate")
                   if case.values[n] is not None and not (n in ("gain", "bias") and "y" in drop)}
        for n in ("h", "y"):
            if n not in drop:
                tensors[n] = tensors["x"] if inplace and n == "h" else place(pool, case, n, None, strides, shift)
        rt.block_norm(make_spec(rt, case, tensors))
        want = case.forward()
        if inplace:                              # (the rows of x are what changed)
            raw = tensors["x"].raw()
            tensors["x"].host[:] = raw
        for n in ("h", "y"):
            if n not in drop:
                check(tensors[n].get().reshape(want[n][0].shape), want[n][0], want[n][1], case.types[0], n)


def run_backward(rt, case, strides={}, shift=0, inplace=False, drop=(), runs=1):
    h = rounded(case.forward()["h"][0], case.types[0])
    want = case.backward(h)
    if "dy" in drop:
        case.values["dy"] = np.zeros_like(case.values["dy"])
        want = case.backward(h)
    if "dh" in drop:
        case.values["dh"] = np.zeros_like(case.values["dh"])
        want = case.backward(h)
    wanted = ["dx"] + (["dgain"] if "dy" not in drop else []) + (["dbias"] if case.values["bias"] is not None and "dy" not in drop else [])
    if case.values["b"] is not None:
        wanted += ["db"] + (["dpost_gain"] if case.post else []) + (["dpost_bias"] if case.values["post_bias"] is not None else [])
        wanted += ["dgate"] if case.values["gate"] is not None else []
    wanted = [n for n in wanted if n not in drop]
    kept = []
    for _ in range(runs):
        with Pool(rt) as pool:
            tensors = {n: place(pool, case, n, case.values[n], strides, shift) for n in ("b", "gain", "post_gain", "post_bias", "gate", "dy", "dh")
                       if case.values[n] is not None and n not in drop and not (n == "gain" and "dy" in drop)}
            tensors["h"] = place(pool, case, "h", h, strides, shift)
            for n in wanted:
                tensors[n] = tensors["dh"] if inplace and n == "dx" else place(pool, case, n, None, strides, shift)
            spec = make_spec(rt, case, tensors)
            spec.workspace_bytes = rt.block_norm_grad_workspace(spec)
            work = pool.bytes(spec.workspace_bytes)
            rt.memset32(work.ptr, 0xffffffff, spec.workspace_bytes // 4)
            spec.workspace = work.ptr
            rt.block_norm_grad(spec)
            if inplace:
                tensors["dh"].host[:] = tensors["dh"].raw()
            kept.append({n: tensors[n].get() for n in wanted})
    for n in wanted:
        check(kept[0][n].reshape(want[n][0].shape), want[n][0], want[n][1], case.types[0] if n in ROWS else case.types[1], n)
        for other in kept[1:]:
            np.testing.assert_array_equal(kept[0][n], other[n], err_msg=n)


SHAPES = [(1, 1), (1, 64), (3, 7), (5, 96), (17, 256), (130, 301), (9, 512), (4, 1027), (33, 1024), (6, 2048), (1, 4096), (3, 4097), (5, 5000),
          (2, 8192), (2, 12001), (3, 16384)]


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("types", TYPES, ids="-".join)
@pytest.mark.parametrize("rows,width", SHAPES)
def test_forward(hip_runtime, rows, width, types, kind):
    run_forward(hip_runtime, Case(rows, width, kind, types, gate_rows=rows, bias=kind == "layer", alpha=1.25, seed=rows + width))


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("types", TYPES, ids="-".join)
@pytest.mark.parametrize("rows,width", SHAPES)
def test_backward(hip_runtime, rows, width, types, kind):
    run_backward(hip_runtime, Case(rows, width, kind, types, gate_rows=rows, bias=kind == "layer", alpha=1.25, seed=rows + width), runs=2)


OPTIONS = [dict(post=False), dict(post=False, gate_rows=1), dict(post=False, gate_rows=6), dict(gate_rows=1), dict(gate_rows=2),
           dict(gate_rows=3, bias=True), dict(gate_rows=12), dict(gate_rows=20, bias=True), dict(gate_rows=30), dict(gate_rows=60),
           dict(block=False), dict(block=False, bias=True), dict(gains=False), dict(gains=False, gate_rows=4, bias=True), dict(alpha=0.0),
           dict(alpha=-0.5, gate_rows=60, bias=True), dict(post=False, gains=False)]


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("types", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")], ids="-".join)
@pytest.mark.parametrize("options", OPTIONS, ids=lambda o: "-".join("%s%s" % kv for kv in sorted(o.items())))
@pytest.mark.parametrize("width", [40, 333])
def test_forms(hip_runtime, width, options, types, kind):
    case = Case(60, width, kind, types, seed=3, **options)
    run_forward(hip_runtime, case)
    run_backward(hip_runtime, case)


@pytest.mark.parametrize("rows,gate_rows", [(1200, 300), (1200, 1200), (5000, 50), (6000, 1), (4608, 9), (4100, 17 * 0 + 41)])
@pytest.mark.parametrize("width", [64, 515])
def test_many_rows(hip_runtime, rows, gate_rows, width):
    """Several rows a part, gate rows that end inside, at and behind parts, the last part short."""
    gate_rows = gate_rows if rows % gate_rows == 0 else rows
    run_backward(hip_runtime, Case(rows, width, "layer", ("bf16", "f32"), gate_rows=gate_rows, bias=True, seed=1), runs=2)
    run_backward(hip_runtime, Case(rows, width, "rms", ("f32", "f32"), gate_rows=gate_rows, seed=1))
    run_forward(hip_runtime, Case(rows, width, "rms", ("f32", "f32"), gate_rows=gate_rows, seed=1))


@pytest.mark.parametrize("types", TYPES, ids="-".join)
@pytest.mark.parametrize("shift,strides", [(0, dict(x=136, b=128, h=144, y=256, dy=136, dh=160, dx=128, db=200, gate=136, dgate=128)),
                                           (1, {}), (3, dict(x=129, b=131, h=128, y=133, dy=140, dh=135, dx=130, db=129, gate=131, dgate=130)),
                                           (0, dict(x=130))])
def test_strided_and_shifted_rows(hip_runtime, types, shift, strides):
    case = Case(21, 128, "layer", types, gate_rows=7, bias=True, alpha=0.5, seed=9)
    run_forward(hip_runtime, case, strides, shift)
    run_backward(hip_runtime, case, strides, shift)


@pytest.mark.parametrize("types", TYPES, ids="-".join)
@pytest.mark.parametrize("width", [72, 130, 4100])
def test_stream_and_its_gradient_in_place(hip_runtime, types, width):
    case = Case(11, width, "rms", types, gate_rows=11, alpha=2.0, seed=4)
    run_forward(hip_runtime, case, inplace=True)
    run_backward(hip_runtime, case, inplace=True)


@pytest.mark.parametrize("drop", [("h",), ("y",), ("dgain", "dpost_gain"), ("dgate",), ("dx",), ("dh",), ("dy",)], ids="-".join)
def test_parts_that_are_not_wanted(hip_runtime, drop):
    case = Case(24, 200, "layer", ("bf16", "f32"), gate_rows=8, bias=True, seed=6)
    if drop[0] in ("h", "y"):
        run_forward(hip_runtime, case, drop=drop)
    else:
        run_backward(hip_runtime, case, drop=drop)


def test_a_layer_norm_of_rows_far_from_zero(hip_runtime):
    """Mean 100 times the spread: the variance is taken around the mean."""
    case = Case(40, 512, "layer", ("f32", "f32"), bias=True, offset=150.0, seed=2)
    run_forward(hip_runtime, case)
    run_backward(hip_runtime, case)


def test_rows_of_zeros_and_of_equal_elements(hip_runtime):
    for kind in ("rms", "layer"):
        case = Case(4, 96, kind, ("f32", "f32"), bias=True, gate_rows=4, seed=2)
        case.values["x"][:2] = 0
        case.values["b"][0] = 0
        case.values["b"][3] = 2.5
        run_forward(hip_runtime, case)
        run_backward(hip_runtime, case)


def test_not_a_number_stays_in_its_row(hip_runtime):
    rt = hip_runtime
    x = np.ones((5, 130), f32)
    x[1, 7], x[3, 129] = np.nan, np.inf
    with Pool(rt) as pool:
        a, y = pool.rows((5, 130), "f32", x), pool.rows((5, 130), "f32")
        rt.block_norm(rt.block_norm_spec(5, 130, "layer", x=a.ptr, y=y.ptr))
        got = y.get()
    assert np.isnan(got[[1, 3]]).all() and not got[[0, 2, 4]].any()


def test_gradients_against_differences(hip_runtime):
    """The gradient of sum(dy * y + dh * h) against central differences of the forward kernel in fp32: the second
    difference is below step^2, the rounding of the sum of 2 x 96 terms about 96 * 2^-24 / step."""
    rt = hip_runtime
    for kind in ("rms", "layer"):
        case = Case(3, 32, kind, ("f32", "f32"), gate_rows=3, bias=True, alpha=0.75, seed=12)

        def loss(values):
            with Pool(rt) as pool:
                tensors = {n: place(pool, case, n, v, {}, 0) for n, v in values.items() if n not in ("dy", "dh")}
                tensors["h"], tensors["y"] = (place(pool, case, n, None, {}, 0) for n in ("h", "y"))
                rt.block_norm(make_spec(rt, case, tensors))
                return (tensors["y"].get().astype(f64) * values["dy"]).sum() + (tensors["h"].get().astype(f64) * values["dh"]).sum()

        h = case.forward()["h"][0].astype(f32)
        with Pool(rt) as pool:
            tensors = {n: place(pool, case, n, v, {}, 0) for n, v in case.values.items() if n not in ("x", "bias")}
            tensors["h"] = place(pool, case, "h", h, {}, 0)
            outs = {"x": "dx", "b": "db", "gain": "dgain", "bias": "dbias", "post_gain": "dpost_gain", "post_bias": "dpost_bias", "gate": "dgate"}
            for n in outs.values():
                tensors[n] = place(pool, case, n, None, {}, 0)
            spec = make_spec(rt, case, tensors)
            spec.workspace_bytes = rt.block_norm_grad_workspace(spec)
            spec.workspace = pool.bytes(spec.workspace_bytes).ptr
            rt.block_norm_grad(spec)
            grads = {n: tensors[o].get() for n, o in outs.items()}
        step = 2.0 ** -6
        for n, g in grads.items():
            for at in ((0, 0), (g.shape[0] - 1, 17), (g.shape[0] // 2, 31)):
                both = []
                for sign in (1, -1):
                    moved = {k: v.copy() for k, v in case.values.items()}
                    moved[n][at] += f32(sign * step)
                    both.append(loss(moved))
                slope = (both[0] - both[1]) / (2 * step)
                assert abs(slope - g[at]) < 20 * step * step + 2 * 192 * EPS * 8 / step, (kind, n, at, slope, g[at])


def test_recorded_calls_replay_with_new_rows(hip_runtime):
    rt = hip_runtime
    case = Case(300, 200, "rms", ("f32", "f32"), gate_rows=300, seed=5)
    with Pool(rt) as pool:
        tensors = {n: place(pool, case, n, v, {}, 0) for n, v in case.values.items() if v is not None}
        for n in ("h", "y", "dx", "db", "dgain", "dpost_gain", "dgate"):
            tensors[n] = place(pool, case, n, None, {}, 0)
        spec = make_spec(rt, case, tensors)
        spec.workspace_bytes = rt.block_norm_grad_workspace(spec)
        work = pool.bytes(spec.workspace_bytes)
        spec.workspace = work.ptr
        outs = ("h", "y", "dx", "db", "dgain", "dpost_gain", "dgate")
        rt.graph_begin()
        rt.block_norm(spec)
        rt.block_norm_grad(spec)
        graph = rt.graph_end()
        try:
            for k in range(4):
                rs = np.random.RandomState(k)
                for n in ("x", "b", "dy", "dh"):
                    rt.memcpy_h2d(tensors[n].ptr, rs.normal(0, 1, (300, 200)).astype(f32))
                rt.graph_launch(graph)
                replayed = {n: tensors[n].get() for n in outs}
                rt.memset32(work.ptr, 0x7fc00000, spec.workspace_bytes // 4)
                rt.block_norm(spec)
                rt.block_norm_grad(spec)
                for n in outs:
                    np.testing.assert_array_equal(replayed[n], tensors[n].get(), err_msg=n)
        finally:
            rt.graph_free(graph)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("types", [("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16")], ids="-".join)
@pytest.mark.parametrize("rows,width", [(40, 250), (9, 257), (22, 2049), (7, 2051), (3, 4095), (3, 4097)])
def test_odd_rows_with_all_sums(hip_runtime, rows, width, types, kind):
    """Rows of 16 bits on any boundary with the gradients of biases: the widths where the pieces a lane holds change."""
    run_backward(hip_runtime, Case(rows, width, kind, types, gate_rows=rows, bias=True, seed=rows), runs=2)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("width", [35, 130, 515, 2051])
def test_not_a_number_stays_in_its_row_backward(hip_runtime, dtype, width):
    """What a short last piece reads of the next row is no part of its own."""
    rt, rs = hip_runtime, np.random.RandomState(width)
    clean = {n: rounded(rs.normal(0, 1, (5, width)), dtype) for n in ("h", "b", "dy", "dh")}
    kept = {}
    for bad in (False, True):
        values = {n: v.copy() for n, v in clean.items()}
        if bad:
            for v in values.values():
                v[1], v[3] = np.nan, np.inf
        with Pool(rt) as pool:
            tensors = {n: pool.rows((5, width), dtype, v) for n, v in values.items()}
            tensors.update({n: pool.rows((5, width), dtype) for n in ("dx", "db")})
            names = {n: t.ptr for n, t in tensors.items()}
            names.update({n + "_stride": width for n in tensors})
            rt.block_norm_grad(rt.block_norm_spec(5, width, "layer", DTYPES[dtype], DTYPES[dtype], True, **names))
            kept[bad] = {n: tensors[n].get() for n in ("dx", "db")}
    for n in ("dx", "db"):
        assert np.isnan(kept[True][n][[1, 3]]).all(), n
        np.testing.assert_array_equal(kept[True][n][[0, 2, 4]], kept[False][n][[0, 2, 4]], err_msg=n)
