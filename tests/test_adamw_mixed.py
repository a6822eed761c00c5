"""neon AdamW over variables of several dtypes (an fp16 table and fp32 gains, which `ng.block_norm` takes side by side): one update
for each pair of dtypes, all of them by gradients of the values before the step."""
import numpy as np
import pytest

import ngraph_hip as ng
import ngraph_hip.transformers as ngt
from ngraph_hip.frontends import neon
from ngraph_hip.transformers import hiprows

f32, f64, f16, i32 = np.float32, np.float64, np.dtype(np.float16), np.dtype(np.int32)
RATE = 0.25


def products():
    """sum(a * b + b * c) over a, c in fp32 and b in fp16: each gradient is made of the others' values."""
    F = ng.make_axis(300, name="F")
    rs = np.random.RandomState(0)
    values = [rs.normal(0, 1, 300).astype(t) for t in (f32, f16, f32)]
    variables = [ng.variable([F], initial_value=v, dtype=np.dtype(v.dtype)) for v in values]
    a, b, c = variables
    opt = neon.AdamW(learning_rate=RATE, weight_decay=0.0)
    return variables, values, opt, opt.minimize(ng.sum(a * b + b * c, out_axes=()), variables=variables)


def model(clip_norm=None, state_bits=32):
    """An fp16 table, an fp32 gain, an fp16 scale."""
    V, F, N = (ng.make_axis(n, name=k) for k, n in (("V", 9), ("F", 24), ("N", 14)))
    rs = np.random.RandomState(1)
    values = {"table": rs.normal(0, 1, (9, 24)).astype(f16), "gain": rs.normal(1, 0.2, 24).astype(f32), "scale": rs.normal(1, 0.2, 24).astype(f16)}
    variables = {"table": ng.variable([V, F], initial_value=values["table"], dtype=f16), "gain": ng.variable([F], initial_value=values["gain"]),
                 "scale": ng.variable([F], initial_value=values["scale"], dtype=f16)}
    tokens, target = ng.placeholder([N], dtype=i32), ng.placeholder([N, F])
    y, h = ng.block_norm(ng.embedding(variables["table"], tokens), gain=variables["gain"])
    cost = ng.squared_L2(y * variables["scale"] - target, out_axes=())
    opt = neon.AdamW(learning_rate=RATE, weight_decay=0.0, gradient_clip_norm=clip_norm, state_bits=state_bits)
    return variables, values, tokens, target, opt, opt.minimize(cost, variables=list(variables.values()))


def test_one_update_for_each_pair_of_dtypes():
    variables, values, opt, step = products()
    assert [[v.dtype for v in u.variables] for u in opt.updates] == [[np.dtype(f32)] * 2, [f16]] and opt.update is opt.updates[0]
    variables, values, tokens, target, opt, step = model()
    t = ngt.make_transformer_factory("hipgpu", dry_run=True)()
    try:
        f = t.computation(step, tokens, target)
        t.initialize()
        group = t.kernel_groups[f]
        group.bind()
        kernels = list(group.kernels)
        updates = [k for k in kernels if isinstance(k, hiprows.AdamWKernel)]
        assert sorted(len(k.op.variables) for k in updates) == [len(u.variables) for u in sorted(opt.updates, key=lambda u: len(u.variables))]
        # nothing that reads a variable comes behind the first update
        held = [v.tensor_description().base for v in variables.values()]
        for k in kernels[kernels.index(updates[0]):]:
            if not isinstance(k, hiprows.AdamWKernel):
                assert not any(read and base in held for base, read, _ in k.buffer_uses()), k.describe()
        for k in kernels:
            k.execute()
    finally:
        t.close()


def test_no_variables_are_no_error():
    opt = neon.AdamW()
    x = ng.placeholder([ng.make_axis(4, name="F")])
    opt.minimize(ng.sum(x * x, out_axes=()), variables=[])
    assert len(opt.updates) == 1 and opt.update.n == 0


@pytest.mark.gpu
def test_updates_by_values_before_the_step(hip_runtime):
    """The first step is the rate times g / |g|; a gradient is a value or a sum of two (rounded to fp16 at most: no sign changes where it
    is not 0), a new value is rounded to its type once."""
    variables, values, opt, step = products()
    t = ngt.make_transformer_factory("hipgpu")()
    try:
        f, read = t.computation([step]), [t.computation(v) for v in variables]
        f()
        after = [np.array(r()) for r in read]
        steps = [int(t.get_tensor_view_value(u.step)) for u in opt.updates]
    finally:
        t.close()
    assert steps == [1, 1]
    a, b, c = [v.astype(f64) for v in values]
    for got, before, g in zip(after, (a, b, c), (b, a + c, b)):
        want = before - RATE * np.sign(g)
        # (eps beside |g|, and fp32's roundings, before the one of the type)
        sure = np.abs(g) > 1e-3
        half = 2.0 ** -11 if got.dtype == f16 else 2.0 ** -24
        assert sure.sum() > 250
        np.testing.assert_array_less(np.abs(got - want)[sure], (half * np.abs(want) + RATE * 1e-5 + 2.0 ** -22 * (np.abs(before) + 1))[sure])


@pytest.mark.gpu
@pytest.mark.parametrize("clip_norm,state_bits", [(None, 32), (0.5, 32), (None, 8)])
def test_a_model_of_mixed_types_trains(hip_runtime, clip_norm, state_bits):
    """Every gradient's sign where it is sure: fp16 roundings of the stream, of the adjoints and of their sums leave a gradient
    within 32 * 2^-11 of the sum of the magnitudes of its terms."""
    variables, values, tokens, target, opt, step = model(clip_norm, state_bits)
    rs = np.random.RandomState(2)
    tk, tg = rs.randint(0, 9, 14).astype(np.int32), rs.normal(0, 1, (14, 24)).astype(f32)
    t = ngt.make_transformer_factory("hipgpu")()
    try:
        f, read = t.computation([step], tokens, target), {k: t.computation(v) for k, v in variables.items()}
        f(tk, tg)
        after = {k: np.array(r()) for k, r in read.items()}
        f(tk, tg)
        assert [int(t.get_tensor_view_value(u.step)) for u in opt.updates] == [2] * len(opt.updates)
    finally:
        t.close()
    table, gain, scale = (values[k].astype(f64) for k in ("table", "gain", "scale"))
    x = table[tk]
    dev = np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5)
    xh = x / dev
    dz = 2 * (xh * gain * scale - tg)
    dn = dz * scale * gain
    dx = dn / dev - x * (dn * x).mean(-1, keepdims=True) / dev ** 3
    grads = {"gain": (dz * scale * xh).sum(0), "scale": (dz * xh * gain).sum(0), "table": np.zeros((9, 24))}
    sizes = {"gain": np.abs(dz * scale * xh).sum(0), "scale": np.abs(dz * xh * gain).sum(0), "table": np.zeros((9, 24))}
    np.add.at(grads["table"], tk, dx)
    np.add.at(sizes["table"], tk, np.broadcast_to(np.abs(dn / dev).max(-1, keepdims=True) * 2, dx.shape))
    norm = np.sqrt(sum((g * g).sum() for g in grads.values()))
    factor = 1.0 if clip_norm is None else clip_norm / max(norm, clip_norm)
    for k, g in grads.items():
        sure = np.abs(g) > 32 * 2.0 ** -11 * sizes[k] + 1e-3
        assert sure.sum() > sure.size // 3
        want = values[k].astype(f64) - RATE * np.sign(g)
        half = 2.0 ** -11 if after[k].dtype == f16 else 2.0 ** -24
        # eps is 1e-8 beside the gradient's clipped size, known to within a factor of 2 (8 bits: the step uses the moments before they
        # are rounded)
        with np.errstate(divide="ignore"):
            slack = RATE * (2e-8 / (factor * np.abs(g)) + 2.0 ** -20) + 2.0 ** -22 * np.abs(want)
        np.testing.assert_array_less(np.abs(after[k] - want)[sure], (half * np.abs(want) + slack)[sure])
