"""AdamW with 8-bit states after an outlier among a block's gradients: second moments far below the block's largest.

A code of 0 beside a first moment would make the step the moment over eps.  A step stores a second moment above 0 as
code 1 at least (compared with NumPy bit for bit).  Where it meets a code of 0 beside a first moment (states that were encoded
from fp32), (0.5 / 255)^4 of the scale, the most that such a code was rounded from, is the least it divides by the root of.
"""
import numpy as np
import pytest

from test_adamw_gpu import BLOCK, HYPER, Model, decode, encode, moments, updated
from row_helpers import EPS, Pool, assert_within

pytestmark = pytest.mark.gpu

f32, f64 = np.float32, np.float64
LEAST = f32((0.5 / 255.0) ** 4)


def stepped(t, k, scale=1.0):
    """The moments after a step, the second one as it counts in it, and the codes and scales that are stored."""
    m, v = moments(t["m"], t["v"], t["g"] * f32(scale), k)
    counted = np.where((t["v_code"] == 0) & (t["m_code"] != 0), np.maximum(v, LEAST * np.repeat(t["v_scale"], BLOCK)[:t["n"]]), v)
    mq, ms = encode(m, False)
    vq, vs = encode(v, True)
    vq = np.where((v > 0) & np.repeat(vs > 0, BLOCK)[:len(v)] & (vq == 0), 1, vq).astype(np.uint8)
    return m, counted, mq, ms, vq, vs


def loaded(rt, model, m, v):
    """Puts the states that `ngh_adamw_encode` makes of m and v into the model's only tensor."""
    t = model.tensors[0]
    for name, x, second in (("m", m, False), ("v", v, True)):
        q, s = encode(x, second)
        rt.memcpy_h2d(t["dev_" + name].ptr + model.shift, q.view(np.uint8))
        rt.memcpy_h2d(t["dev_%s_scale" % name].ptr, s)
        t[name], t[name + "_code"], t[name + "_scale"] = decode(q, s, second), q, s
    return t


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("n,largest", [(1000, 1.0), (70000, 1.0), (1000, 1e30), (1000, 1e-33)])
def test_small_second_moments_beside_first_ones(hip_runtime, n, largest, shift):
    """Shares of the block's largest from 1 down to 1e-24, some gradients 0; with scales that take the exact chain."""
    rt, rs = hip_runtime, np.random.RandomState(n)
    with Pool(rt) as pool:
        model = Model(pool, rt, [n], ("f32", "f32"), 8, shift=shift)
        share = 10.0 ** -rs.uniform(0, 24, n)
        share[::50] = 1.0
        v = (share * largest).astype(f32)
        v[3::17] = 0
        m = (np.sqrt(share * largest) * rs.normal(0, 0.3, n) * np.where(np.arange(n) % 256 < 128, 1, 1e-6)).astype(f32)
        g = (np.sqrt(share * largest) * rs.normal(0, 1, n)).astype(f32)
        g[::3] = 0
        t = loaded(rt, model, m, v)
        t["g"] = g
        rt.memcpy_h2d(t["dev_g"].ptr, g)
        low = 0
        for step in (5, 6, 7):
            low += int(((t["v_code"] == 0) & (t["m_code"] != 0)).sum())
            m, v, mq, ms, vq, vs = stepped(t, HYPER)
            want, bound = updated(t["p"], m, v, f64(0), step, HYPER)
            rt.adamw_step(model.plan, step, **HYPER)
            p = t["dev_p"].get().reshape(-1)
            assert_within(p, want, bound + EPS * (np.abs(want) + bound), "parameters")
            for name, q, s, second in (("m", mq, ms, False), ("v", vq, vs, True)):
                got_q, got_s = model.codes(t, name)
                np.testing.assert_array_equal(got_s, s)
                np.testing.assert_array_equal(got_q, q)
                t[name], t[name + "_code"], t[name + "_scale"] = decode(q, s, second), q, s
            t["p"] = p
        assert low > 0
        model.free()


@pytest.mark.parametrize("ratio", [1e4, 1e6, 1e7])
@pytest.mark.parametrize("beta2", [0.95, 0.999])
def test_steps_after_an_outlier(hip_runtime, beta2, ratio):
    """Gradients of 1e-5, one of a block `ratio` times that once, then a step without a gradient.

    With states in 32 bits no step of the others is larger than 1.3 rates.  A code that rounding keeps where it is (code 1
    at worst) holds a second moment of at least (1 - beta2) g^2 / ((1.5^4 - 1) beta2): a step after such gradients is at most
    0.9 / sqrt(1 - beta2) rates, one without a gradient 1.9 / sqrt(1 - beta2); the first moment may have been rounded up
    from half a code, to 4 times its size.  By eps alone it was 526 to 765 rates."""
    rt, n, lr = hip_runtime, 256, 1e-3
    hyper = dict(lr=lr, beta1=0.9, beta2=beta2, eps=1e-8)
    with Pool(rt) as pool:
        worst = {}
        for bits in (32, 8):
            rs = np.random.RandomState(0)
            model = Model(pool, rt, [n], ("f32", "f32"), bits)
            t = model.tensors[0]
            for name in ("m", "v", "p"):
                if name == "p" or bits == 32:
                    rt.memcpy_h2d(t["dev_" + name].ptr, np.zeros(n, f32))
                else:
                    rt.memcpy_h2d(t["dev_" + name].ptr, np.zeros(n, np.uint8))
                    rt.memcpy_h2d(t["dev_%s_scale" % name].ptr, np.zeros(1, f32))
            before, worst[bits] = np.zeros(n, f32), 0.0
            for step in range(1, 301):
                g = rs.normal(0, 1e-5, n).astype(f32)
                if step == 20:
                    g[7] = 1e-5 * ratio
                if step % 40 == 0:
                    g[:] = 0
                rt.memcpy_h2d(t["dev_g"].ptr, g)
                rt.adamw_step(model.plan, step, **hyper)
                p = t["dev_p"].get().reshape(-1)
                worst[bits] = max(worst[bits], np.abs(np.delete(p - before, 7)).max() / lr)
                before = p
            model.free()
    assert worst[32] < 1.5
    assert worst[8] < 4 * 1.9 / np.sqrt(1 - beta2), worst
