"""ngh_adamw_* against NumPy.

The moments and the 8-bit codes are defined by fp32 operations in a fixed order, which NumPy's
correctly rounded fp32 repeats: they are compared bit for bit.  The update is compared with float64.
In units of u = 2^-24 its step is off by 2 (root, 1 ulp) + 2 (times a factor that is rounded itself) + 1
(plus eps) + 2 (reciprocal, 1 ulp) + 1 (times m) + 2 (times the rounded rate) = 10 of its size, the parameter
by 2 (times a rounded factor) + 1 (the difference) of its own, the difference by 1 of the step: 11 and
3, 12 and 4 with the second order; then one rounding to the type.
"""
import numpy as np
import pytest

from row_helpers import DTYPES, EPS, HALF, TINY, Pool, assert_within, from_storage, rounded, to_storage

pytestmark = pytest.mark.gpu

f32, f64 = np.float32, np.float64
BLOCK = 256
HYPER = dict(lr=2e-3, beta1=0.9, beta2=0.97, eps=1e-8)


def blocks(x, fill=0):
    n = (len(x) + BLOCK - 1) // BLOCK * BLOCK
    return np.concatenate([x, np.full(n - len(x), fill, x.dtype)]).reshape(-1, BLOCK)


def encode(x, second):
    b = blocks(np.asarray(x, f32))
    s = np.abs(b).max(1, keepdims=True) if len(b) else np.zeros((0, 1), f32)
    s[~np.isfinite(s)] = np.nan
    with np.errstate(all="ignore"):
        share = np.where(s > 0, np.abs(b) / s, f32(0)).astype(f32)
        q = np.rint(np.sqrt(np.sqrt(share)) * f32(255)) if second else np.rint(np.sqrt(share) * f32(127)) * np.sign(b)
        q = np.where(s > 0, q, 0)
    return q.reshape(-1)[:len(x)].astype(np.uint8 if second else np.int8), s.reshape(-1)


def decode(codes, s, second):
    t = codes.astype(f32) * (f32(1.0 / 255.0) if second else f32(1.0 / 127.0))
    v = (t * t) * (t * t) if second else t * np.abs(t)
    return v * np.repeat(s, BLOCK)[:len(codes)]


def moments(m, v, g, k):
    m = m * f32(k["beta1"]) + g * f32(1.0 - k["beta1"])
    return m, v * f32(k["beta2"]) + (g * g) * f32(1.0 - k["beta2"])


def updated(p, m, v, decay, t, k):
    """float64 from the fp32 moments: the new parameter and the bound of what fp32 is off by."""
    m, v, p = m.astype(f64), v.astype(f64), p.astype(f64)
    step = k["lr"] / (1 - k["beta1"] ** t) * m / (np.sqrt(v) / np.sqrt(1 - k["beta2"] ** t) + k["eps"])
    want = p * (1 - k["lr"] * decay) - step
    return want, EPS * (4 * np.abs(p) + 12 * np.abs(step))


class Model(object):
    """Parameters, gradients and states of several tensors on the device and the host."""

    def __init__(self, pool, rt, sizes, types=("f32", "f32"), bits=32, copy=None, shift=0, seed=0):
        self.rt, self.types, self.bits, self.copy = rt, types, bits, copy
        rs = np.random.RandomState(seed)
        self.tensors, rows = [], []
        for i, n in enumerate(sizes):
            size = np.exp(rs.normal(-5, 2))
            t = {"n": n, "decay": 0.1 if i % 2 else 0.0, "p": rounded(rs.normal(0, 0.1, n), types[0]), "g": rounded(rs.normal(0, size, n), types[1]),
                 "m": rs.normal(0, size, n).astype(f32), "v": (rs.normal(0, size, n).astype(f32)) ** 2}
            one = (1, n)
            t["dev_p"] = pool.rows(one, types[0], t["p"], shift=shift)
            t["dev_g"] = pool.rows(one, types[1], t["g"], shift=shift)
            row = dict(param=t["dev_p"].ptr, grad=t["dev_g"].ptr, n=n, weight_decay=t["decay"])
            if bits == 8:
                for name, second in (("m", False), ("v", True)):
                    q, s = encode(t[name], second)
                    t[name] = decode(q, s, second)
                    t["dev_" + name] = pool.array(np.concatenate([np.zeros(shift, np.uint8), q.view(np.uint8), np.full(70, 0xC5, np.uint8)]))
                    t["dev_%s_scale" % name] = pool.array(np.concatenate([s, np.full(3, 7.5, f32)]))
                    row[name], row[name + "_scale"] = t["dev_" + name].ptr + shift, t["dev_%s_scale" % name].ptr
            else:
                for name in ("m", "v"):
                    t["dev_" + name] = pool.rows(one, "f32", t[name], shift=shift)
                    row[name] = t["dev_" + name].ptr
            if copy:
                t["dev_copy"] = pool.rows(one, copy, None, shift=shift)
                row["copy"] = t["dev_copy"].ptr
            self.tensors.append(t)
            rows.append(row)
        self.shift = shift
        self.plan = rt.adamw_plan(rows, DTYPES[types[0]], DTYPES[types[1]], DTYPES[copy] if copy else -1, bits)

    def codes(self, t, name):
        raw = t["dev_" + name].get()
        assert (raw[self.shift + t["n"]:] == 0xC5).all() and not raw[:self.shift].any()
        scales = t["dev_%s_scale" % name].get()
        assert (scales[-3:] == 7.5).all()
        q = raw[self.shift:self.shift + t["n"]]
        return q if name == "v" else q.view(np.int8), scales[:-3]

    def check_step(self, step, scale=1.0, hyper=HYPER):
        for i, t in enumerate(self.tensors):
            with np.errstate(all="ignore"):
                m, v = moments(t["m"], t["v"], t["g"] * f32(scale), hyper)
                want, bound = updated(t["p"], m, v, f64(f32(t["decay"])), step, hyper)
            p = t["dev_p"].get().reshape(-1)
            assert_within(p, want, bound + (np.abs(want) + bound) * HALF[self.types[0]] + TINY[self.types[0]], "tensor %d" % i)
            if self.copy:
                c = t["dev_copy"].get().reshape(-1)
                if self.types[0] == "f32":
                    np.testing.assert_array_equal(c, rounded(p, self.copy))
                else:
                    assert_within(c, want, bound + (np.abs(want) + bound) * HALF[self.copy] + TINY[self.copy])
            for name, x, second in (("m", m, False), ("v", v, True)):
                if self.bits == 32:
                    np.testing.assert_array_equal(t["dev_" + name].get().reshape(-1), x)
                    t[name] = x
                else:
                    q, s = encode(x, second)
                    got_q, got_s = self.codes(t, name)
                    np.testing.assert_array_equal(got_s, s)
                    np.testing.assert_array_equal(got_q, q)
                    t[name] = decode(q, s, second)
            t["p"] = p

    def free(self):
        self.rt.adamw_plan_free(self.plan)


SIZES = [1, 3, 255, 256, 257, 1000, 4095, 4096, 4097, 0, 12345, 2, 70000]
TYPES = [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("bf16", "f16"), ("f16", "f16"), ("f16", "f32"),
         ("f16", "bf16")]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("types", TYPES, ids="-".join)
@pytest.mark.parametrize("shift", [0, 1, 2])
def test_steps(hip_runtime, types, bits, shift):
    with Pool(hip_runtime) as pool:
        model = Model(pool, hip_runtime, SIZES, types, bits, shift=shift)
        for step in (1, 2, 3):
            hip_runtime.adamw_step(model.plan, step, **HYPER)
            model.check_step(step)
        model.free()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("copy", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("types", [("f32", "bf16"), ("bf16", "f32")], ids="-".join)
def test_copy_of_the_parameters(hip_runtime, types, copy, bits):
    with Pool(hip_runtime) as pool:
        model = Model(pool, hip_runtime, [300, 5000, 1], types, bits, copy)
        hip_runtime.adamw_step(model.plan, 10, **HYPER)
        model.check_step(10)
        model.free()


@pytest.mark.parametrize("bits", [32, 8])
def test_hundreds_of_tensors(hip_runtime, bits):
    sizes = list(np.random.RandomState(1).randint(1, 3000, 400))
    with Pool(hip_runtime) as pool:
        model = Model(pool, hip_runtime, [int(s) for s in sizes], ("f32", "bf16"), bits)
        hip_runtime.adamw_step(model.plan, 7, grad_scale=0.25, **HYPER)
        model.check_step(7, 0.25)
        model.free()


@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-13, 1e-12, 1e-3])
@pytest.mark.parametrize("bits", [32, 8])
def test_small_second_moments_and_any_eps(hip_runtime, bits, eps):
    """Gradients down to where their squares leave the normal numbers."""
    with Pool(hip_runtime) as pool:
        model = Model(pool, hip_runtime, [4000], ("f32", "f32"), bits)
        t = model.tensors[0]
        rs = np.random.RandomState(4)
        t["g"] = (rs.normal(0, 1, 4000) * 10.0 ** -(4 + np.arange(4000) // 256)).astype(f32)
        t["g"][t["g"] == 0] = f32(1e-10)
        hip_runtime.memcpy_h2d(t["dev_g"].ptr, t["g"])
        if bits == 32:
            for name in ("m", "v"):
                t[name] = (t["g"] * t["g"] if name == "v" else t["g"]).astype(f32)
                hip_runtime.memcpy_h2d(t["dev_" + name].ptr, t[name])
            hyper = dict(HYPER, eps=eps)
            hip_runtime.adamw_step(model.plan, 3, **hyper)
            model.check_step(3, hyper=hyper)
        else:
            hyper = dict(HYPER, eps=max(eps, 1e-13))          # (8 bits hold moments that are 0)
            hip_runtime.adamw_step(model.plan, 3, **hyper)
            model.check_step(3, hyper=hyper)
        model.free()


@pytest.mark.parametrize("bits", [32, 8])
def test_moments_up_to_the_largest_numbers(hip_runtime, bits):
    """Scales whose reciprocals are below the normal numbers."""
    rt, rs = hip_runtime, np.random.RandomState(8)
    with Pool(rt) as pool:
        model = Model(pool, rt, [4000], ("f32", "f32"), bits)
        t = model.tensors[0]
        size = np.minimum(10.0 ** (24 + np.arange(4000) // 256), 3e38)
        for name in ("m", "v"):
            x = (np.clip(rs.normal(0, 0.4, 4000), -1, 1) * size).astype(f32)
            x = np.abs(x) if name == "v" else x
            if bits == 8:
                q, scales = encode(x, name == "v")
                t[name] = decode(q, scales, name == "v")
                rt.memcpy_h2d(t["dev_" + name].ptr, q.view(np.uint8))
                rt.memcpy_h2d(t["dev_%s_scale" % name].ptr, scales)
            else:
                t[name] = x
                rt.memcpy_h2d(t["dev_" + name].ptr, x)
        rt.adamw_step(model.plan, 9, **HYPER)
        model.check_step(9)
        model.free()


def test_a_plan_is_not_freed_while_recording(hip_runtime):
    from ngraph_hip.runtime import HipLibraryError
    rt = hip_runtime
    with Pool(rt) as pool:
        model = Model(pool, rt, [500])
        rt.graph_begin()
        try:
            with pytest.raises(HipLibraryError) as e:
                model.free()
        finally:
            rt.graph_abandon()
        assert "recorded" in str(e.value)
        rt.adamw_step(model.plan, 1, **HYPER)
        model.check_step(1)
        model.free()


@pytest.mark.parametrize("second", [False, True])
def test_codes_of_more_blocks_than_a_launch_has_wavefronts(hip_runtime, second):
    rt, n = hip_runtime, 64 * 256 * 1024 * 2 + 777
    with Pool(rt) as pool:
        x = np.tile(np.random.RandomState(3).normal(0, 1, 1 << 16).astype(f32), n // (1 << 16) + 1)[:n]
        x = np.abs(x) if second else x
        values, codes = pool.array(x), pool.array(np.zeros(n, np.uint8))
        scales = pool.array(np.zeros((n + BLOCK - 1) // BLOCK, f32))
        rt.adamw_encode(codes.ptr, scales.ptr, values.ptr, n, second)
        q, s = encode(x, second)
        np.testing.assert_array_equal(codes.get().view(q.dtype), q)
        np.testing.assert_array_equal(scales.get(), s)
        rt.adamw_decode(values.ptr, codes.ptr, scales.ptr, n, second)
        np.testing.assert_array_equal(values.get(), decode(q, s, second))


def test_a_plan_of_nothing(hip_runtime):
    plan = hip_runtime.adamw_plan([])
    hip_runtime.adamw_step(plan, 1)
    hip_runtime.adamw_plan_free(plan)


@pytest.mark.parametrize("bits", [32, 8])
def test_scalars_on_the_device_and_recorded_steps(hip_runtime, bits):
    """A recorded step counts on, follows a new rate and a new clipping factor, and equals eager steps."""
    rt = hip_runtime
    with Pool(rt) as pool:
        model = Model(pool, rt, [777, 4096, 5], ("f32", "f32"), bits)
        count, lr, clip = pool.array(np.array([4], np.int32)), pool.array(np.array([1e-3], f32)), pool.array(np.array([1.0], f32))
        given = dict(HYPER, dev_step=count.ptr, dev_lr=lr.ptr, dev_grad_scale=clip.ptr, grad_scale=0.5)
        rt.graph_begin()
        rt.adamw_step(model.plan, **given)
        graph = rt.graph_end()
        try:
            for k in range(5):
                rate, factor = f32(1e-3 * (k + 1)), f32(1.0 / (k + 1))
                lr.set(np.array([rate], f32))
                clip.set(np.array([factor], f32))
                if k % 2:
                    rt.adamw_step(model.plan, **given)
                else:
                    rt.graph_launch(graph)
                assert count.get()[0] == 5 + k
                model.check_step(5 + k, f32(0.5) * factor, dict(HYPER, lr=f64(rate)))
        finally:
            rt.graph_free(graph)
        model.free()


def test_a_plan_while_recording_is_refused(hip_runtime):
    from ngraph_hip.runtime import HipLibraryError
    rt = hip_runtime
    with Pool(rt) as pool:
        a = [pool.rows((1, 8), "f32", np.zeros((1, 8))) for _ in range(4)]
        rt.graph_begin()
        try:
            with pytest.raises(HipLibraryError) as e:
                rt.adamw_plan([dict(param=a[0].ptr, grad=a[1].ptr, m=a[2].ptr, v=a[3].ptr, n=8)])
        finally:
            rt.graph_abandon()
        assert "recorded" in str(e.value)


def test_hyperparameters_out_of_range_are_refused(hip_runtime):
    from ngraph_hip.runtime import HipLibraryError
    plan = hip_runtime.adamw_plan([])
    for change in (dict(step=0), dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1e-8), dict(lr=float("nan")), dict(grad_scale=float("nan"))):
        with pytest.raises(HipLibraryError):
            hip_runtime.adamw_step(plan, **dict(dict(step=1), **change))
    hip_runtime.adamw_plan_free(plan)


def test_a_gradient_that_is_not_finite_shows(hip_runtime):
    """In its element with fp32 states; with 8 bits in its element now and in its block from the next step on."""
    rt = hip_runtime
    for bits in (32, 8):
        with Pool(rt) as pool:
            model = Model(pool, rt, [1000], ("f32", "f32"), bits)
            t = model.tensors[0]
            g = t["g"].copy()
            g[300] = np.inf
            rt.memcpy_h2d(t["dev_g"].ptr, g)
            rt.adamw_step(model.plan, 1, **HYPER)
            p = t["dev_p"].get().reshape(-1)
            assert np.isnan(p[300]) and np.isfinite(np.delete(p, 300)).all()
            rt.adamw_step(model.plan, 2, **HYPER)
            bad = np.isnan(t["dev_p"].get().reshape(-1))
            want = np.zeros(1000, bool)
            want[256:512 if bits == 8 else 257] = True
            if bits == 32:
                want[:] = False
                want[300] = True
            np.testing.assert_array_equal(bad, want)
            model.free()


@pytest.mark.parametrize("second", [False, True])
@pytest.mark.parametrize("n,shift", [(1, 0), (255, 0), (256, 1), (257, 2), (100003, 0), (100003, 3)])
def test_codes_of_states(hip_runtime, n, shift, second):
    rt = hip_runtime
    rs = np.random.RandomState(n)
    x = (rs.normal(0, 1, n) * np.exp(rs.normal(0, 6, n))).astype(f32)
    x[::97] = 0
    if n > 1000:
        x[512:768] = 0                                                # a block of zeros
        x[1024:1280] *= f32(1e-38)                                    # below the normal numbers
    x = x * x if second else x
    q, s = encode(x, second)
    with Pool(rt) as pool:
        values, codes = pool.rows((1, n), "f32", x, shift=shift), pool.array(np.full(shift + n + 9, 0xC5, np.uint8))
        scales, back = pool.array(np.full(len(s) + 2, 7.5, f32)), pool.rows((1, n), "f32", None, shift=shift)
        rt.adamw_encode(codes.ptr + shift, scales.ptr, values.ptr, n, second)
        got = codes.get()
        assert (got[:shift] == 0xC5).all() and (got[shift + n:] == 0xC5).all() and (scales.get()[len(s):] == 7.5).all()
        np.testing.assert_array_equal(got[shift:shift + n], q.view(np.uint8))
        np.testing.assert_array_equal(scales.get()[:len(s)], s)
        rt.adamw_decode(back.ptr, codes.ptr + shift, scales.ptr, n, second)
        np.testing.assert_array_equal(back.get().reshape(-1), decode(q, s, second))


def test_helpers_round_as_the_types_do():
    x = np.array([1.0, 1.0 + 2.0 ** -9, 1.0 + 2.0 ** -8, 1.0 + 3 * 2.0 ** -9, -3.3e38, 1e-40, np.inf], f32)
    got = from_storage(to_storage(x, "bf16"), "bf16")
    np.testing.assert_array_equal(got[:4], np.array([1.0, 1.0, 1.0, 1.0 + 2.0 ** -7], f32))
    assert np.isinf(got[-1]) and abs(got[4] / x[4] - 1) <= 2.0 ** -8
