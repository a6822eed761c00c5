"""The operators over rows and parameters as graph ops: `ng.embedding`, `ng.block_norm`, neon `AdamW`, their
derivatives, and a training step made of all of them, against NumPy in float64.

Bounds of the single ops are those of the C ABI tests' kernels (a hundred roundings of 2^-24 in a row at
most, relative to the magnitudes that meet): 1e-5 of the largest magnitude.  Of the step: see there.
"""
import numpy as np
import pytest

import ngraph_hip as ng
import ngraph_hip.transformers as ngt
from ngraph_hip.frontends import neon
from ngraph_hip.transformers import hiprows

f32, f64, i32 = np.float32, np.float64, np.dtype(np.int32)


def axes(**kw):
    return [ng.make_axis(v, name=k) for k, v in kw.items()]


def transformer(dry_run=False, **kw):
    return ngt.make_transformer_factory("hipgpu", dry_run=dry_run, **kw)()


# ------------------------------------------------------------------------- without a device
def test_ops_check_their_arguments():
    V, F, T, B = axes(V=10, F=8, T=5, B=3)
    table, tokens = ng.placeholder([V, F]), ng.placeholder([B, T], dtype=i32)
    assert list(ng.embedding(table, tokens).axes) == [B, T, F]
    for bad in (lambda: ng.embedding(ng.placeholder([V]), tokens), lambda: ng.embedding(table, ng.placeholder([B])),
                lambda: ng.embedding(table, ng.placeholder([F], dtype=i32)), lambda: ng.embedding(ng.placeholder([V, F], dtype=i32), tokens)):
        with pytest.raises(ValueError):
            bad()
    x, b, w = ng.placeholder([B, T, F]), ng.placeholder([B, T, F]), ng.placeholder([F])
    y, h = ng.block_norm(x, b, gain=w, post_gain=w, gate=ng.placeholder([B, F]))
    assert y.gate_rows == 5 and y.post_norm and list(h.axes) == [B, T, F]
    assert ng.block_norm(x, b, gate=ng.placeholder([F]))[0].gate_rows == 15
    assert ng.block_norm(x, b, gate=ng.placeholder([B, T, F]))[0].gate_rows == 1
    for bad in (dict(kind="batch"), dict(gain=ng.placeholder([T])), dict(gate=ng.placeholder([T, F])), dict(post_gain=w, post_norm=False),
                dict(b=None, gate=w), dict(b=ng.placeholder([B, F])), dict(gain=ng.placeholder([F], dtype=np.float16)),
                dict(gate=ng.placeholder([B]))):
        with pytest.raises(ValueError):
            ng.block_norm(x, **dict(dict(b=b), **bad))
    v = ng.variable([F], initial_value=0.)
    for bad in (dict(state_bits=16), dict(weight_decay=[]), dict(grads=[x]), dict(variables=[v, v], grads=[w, w], weight_decay=[0, 0]),
                dict(variables=[w * 1.5]), dict(lr=x)):
        with pytest.raises(ValueError):
            hiprows.AdamWOp(**dict(dict(variables=[v], grads=[w], weight_decay=[0.0]), **bad))


def step_graph(kind="rms", state_bits=32, dims=None, **optimizer):
    """Embedding, two blocks (an elementwise one each) between norms, a squared cost, an AdamW step."""
    d = dict(dims or dict(V=50, F=24, T=7, N=6))
    V, F, T, N = axes(**d)
    rs = np.random.RandomState(0)
    init = lambda ax, std, mean=0.0: ng.variable(ax, initial_value=rs.normal(mean, std, [a.length for a in ax]).astype(f32))      # noqa: E731
    p = {"table": init([V, F], 0.5), "gain0": init([F], 0.1, 1), "scale1": init([F], 0.5, 1), "post1": init([F], 0.1, 1), "gate1": init([F], 0.2, 0.5),
         "gain1": init([F], 0.1, 1), "scale2": init([F], 0.5, 1), "gain2": init([F], 0.1, 1)}
    if kind == "layer":
        p.update(bias0=init([F], 0.1), postbias1=init([F], 0.1), bias1=init([F], 0.1))
    tokens, target = ng.placeholder([N, T], dtype=i32), ng.placeholder([N, T, F])
    x0 = ng.embedding(p["table"], tokens, scale=2.0, pad_idx=0)
    y0, h0 = ng.block_norm(x0, gain=p["gain0"], bias=p.get("bias0"), kind=kind)
    b1 = ng.tanh(y0 * p["scale1"])
    y1, h1 = ng.block_norm(h0, b1, gain=p["gain1"], bias=p.get("bias1"), post_gain=p["post1"], post_bias=p.get("postbias1"), gate=p["gate1"], kind=kind,
                           residual_scale=0.5)
    b2 = ng.tanh(y1 * p["scale2"])
    y2, h2 = ng.block_norm(h1, b2, gain=p["gain2"], kind=kind)
    cost = ng.squared_L2(y2 - target, out_axes=[N])
    opt = neon.AdamW(learning_rate=1e-2, weight_decay=0.1, state_bits=state_bits, **optimizer)
    step = opt.minimize(cost, variables=list(p.values()))
    return d, p, tokens, target, cost, opt, step


@pytest.mark.parametrize("state_bits", [32, 8])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_a_step_lowers_without_a_device(kind, state_bits):
    d, p, tokens, target, cost, opt, step = step_graph(kind, state_bits)
    t = transformer(dry_run=True)
    f = t.computation(step, tokens, target)
    t.initialize()
    group = t.kernel_groups[f]
    group.bind()
    names = [k.describe()[0][0] for k in group.kernels if isinstance(k, hiprows.RowKernel)]
    # (the padded tokens' gradient, both norms' passes of three norms, one update for everything)
    assert sorted(names) == sorted(["embedding", "embedding_grad", "adamw"] + ["block_norm", "block_norm_grad"] * 3)
    for k in group.kernels:
        k.execute()
    t.close()


def test_only_what_is_used_is_written():
    F, N = axes(F=16, N=4)
    x, b, w = ng.placeholder([N, F]), ng.placeholder([N, F]), ng.placeholder([F])
    y, h = ng.block_norm(x, b, gain=w, post_gain=w, gate=w)
    t = transformer(dry_run=True)
    f = t.computation(y, x, b, w)
    t.initialize()
    t.kernel_groups[f].bind()
    spec = t.kernel_groups[f].kernels[0].spec
    assert spec.y and not spec.h and spec.gate_rows == 4
    t.close()
    y, h = ng.block_norm(x, b, gain=w)
    dx = ng.deriv(ng.sum(y, out_axes=()), x)
    t = transformer(dry_run=True)
    f = t.computation(dx, x, b, w)
    t.initialize()
    t.kernel_groups[f].bind()
    spec = [k.spec for k in t.kernel_groups[f].kernels if isinstance(k, hiprows.BlockNormGradKernel)][0]
    assert spec.dx and spec.dy and not spec.db and not spec.dgain
    t.close()


def test_flex_tensors_are_refused():
    F, N = axes(F=16, N=4)
    y, _ = ng.block_norm(ng.placeholder([N, F]))
    t = ngt.make_transformer_factory("flexhip", dry_run=True)()
    try:
        with pytest.raises(Exception) as e:
            f = t.computation(y, *[p for p in [y.args[0].tensor]])
            t.initialize()
            t.kernel_groups[f].bind()
        assert "flex" in str(e.value)
    finally:
        t.close()


# ------------------------------------------------------------------------- with one
def norm64(x, kind, eps=1e-5):
    c = x - x.mean(-1, keepdims=True) if kind == "layer" else x
    return c / np.sqrt((c * c).mean(-1, keepdims=True) + eps)


@pytest.mark.gpu
def test_embedding_and_its_derivative(hip_runtime):
    V, F, T, N = axes(V=40, F=12, T=5, N=8)
    table, tokens = ng.placeholder([V, F]), ng.placeholder([N, T], dtype=i32)
    y = ng.embedding(table, tokens, scale=1.5, pad_idx=3)
    c = ng.placeholder([N, T, F])
    grad = ng.deriv(ng.sum(y * c, out_axes=()), table)
    rs = np.random.RandomState(0)
    w, cc = rs.normal(0, 1, (40, 12)).astype(f32), rs.normal(0, 1, (8, 5, 12)).astype(f32)
    tt = rs.randint(-1, 42, (8, 5)).astype(np.int32)
    t = transformer()
    try:
        got, dw = t.computation([y, grad], table, tokens, c)(w, tt, cc)
    finally:
        t.close()
    has = (tt >= 0) & (tt < 40) & (tt != 3)
    np.testing.assert_array_equal(got, np.where(has[..., None], w[np.where(has, tt, 0)] * f32(1.5), 0))
    want = np.zeros((40, 12))
    np.add.at(want, tt[has], 1.5 * cc[has].astype(f64))
    np.testing.assert_allclose(dw, want, atol=1e-5 * np.abs(want).max())


@pytest.mark.gpu
def test_two_lookups_of_one_table_add_their_gradients(hip_runtime):
    V, F, N = axes(V=9, F=4, N=6)
    table, a, b = ng.placeholder([V, F]), ng.placeholder([N], dtype=i32), ng.placeholder([N], dtype=i32)
    cost = ng.sum(ng.embedding(table, a, scale=2.0) * ng.embedding(table, b), out_axes=())
    rs = np.random.RandomState(1)
    w, aa, bb = rs.normal(0, 1, (9, 4)).astype(f32), rs.randint(0, 9, 6).astype(np.int32), rs.randint(0, 9, 6).astype(np.int32)
    t = transformer()
    try:
        got = t.computation(ng.deriv(cost, table), table, a, b)(w, aa, bb)
    finally:
        t.close()
    want = np.zeros((9, 4))
    np.add.at(want, aa, 2.0 * w[bb].astype(f64))
    np.add.at(want, bb, 2.0 * w[aa].astype(f64))
    np.testing.assert_allclose(got, want, atol=1e-5 * np.abs(want).max())


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["rows", "transposed"])
@pytest.mark.parametrize("gate_axes", ["F", "NF", "NTF"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_block_norm_and_its_derivatives_against_differences(hip_runtime, kind, gate_axes, order):
    ax = dict(zip("NTF", axes(N=3, T=4, F=20)))
    N, T, F = ax["N"], ax["T"], ax["F"]
    stored = [F, N, T] if order == "transposed" else [N, T, F]               # (rows that have to be copied first)
    names = dict(x=stored, b=stored, gain=[F], bias=[F], post_gain=[F], post_bias=[F], gate=[ax[k] for k in gate_axes])
    p = {k: ng.placeholder(a) for k, a in names.items()}
    rows = lambda q: ng.axes_with_order(q, ng.make_axes([N, T, F]))                                    # noqa: E731
    y, h = ng.block_norm(rows(p["x"]), rows(p["b"]), p["gain"], p["bias"], p["post_gain"], p["post_bias"], p["gate"], kind, residual_scale=0.7)
    cy, ch = ng.placeholder([N, T, F]), ng.placeholder([N, T, F])
    cost = ng.sum(y * cy, out_axes=()) + ng.sum(h * ch, out_axes=())
    grads = [ng.deriv(cost, q) for q in p.values()]
    rs = np.random.RandomState(3)
    values = {k: rs.normal(1.0 if "gain" in k else 0.2, 0.5, [a.length for a in axs]).astype(f32) for k, axs in names.items()}
    cyv, chv = (rs.normal(0, 1, (3, 4, 20)).astype(f32) for _ in range(2))

    def forward(v):
        v = {k: a.astype(f64) for k, a in v.items()}
        x, b = (np.moveaxis(v[k], 0, -1) if order == "transposed" else v[k] for k in ("x", "b"))
        gate = v["gate"][:, None, :] if gate_axes == "NF" else v["gate"]
        h = 0.7 * x + gate * (norm64(b, kind) * v["post_gain"] + v["post_bias"])
        return norm64(h, kind) * v["gain"] + v["bias"], h

    t = transformer()
    try:
        out = t.computation([y, h] + grads, *(list(p.values()) + [cy, ch]))(*(list(values.values()) + [cyv, chv]))
    finally:
        t.close()
    want = forward(values)
    for got, w in zip(out[:2], want):
        np.testing.assert_allclose(got, w, atol=1e-5 * np.abs(w).max())
    # central differences of the float64 model: their error is below step^2 times the third derivative (some hundreds)
    step = 1e-4
    for (k, v), g in zip(values.items(), out[2:]):
        for at in [tuple(rs.randint(0, n) for n in v.shape) for _ in range(6)]:
            cost = []
            for sign in (1, -1):
                moved = {n: a.astype(f64) for n, a in values.items()}
                moved[k][at] += sign * step
                yy, hh = forward(moved)
                cost.append((yy * cyv).sum() + (hh * chv).sum())
            slope = (cost[0] - cost[1]) / (2 * step)
            assert abs(slope - g[at]) < 1e-4 + 1e-5 * np.abs(g).max(), (k, at, slope, g[at])


@pytest.mark.gpu
def test_gradient_of_the_stream_alone(hip_runtime):
    N, F = axes(N=5, F=16)
    x, b, g = ng.placeholder([N, F]), ng.placeholder([N, F]), ng.placeholder([F])
    y, h = ng.block_norm(x, b, gate=g, residual_scale=3.0)
    cost = ng.sum(h * h, out_axes=())
    rs = np.random.RandomState(3)
    xv, bv, gv = rs.normal(0, 1, (5, 16)).astype(f32), rs.normal(0, 1, (5, 16)).astype(f32), rs.normal(0, 1, 16).astype(f32)
    t = transformer()
    try:
        dx, db, dg = t.computation([ng.deriv(cost, q) for q in (x, b, g)], x, b, g)(xv, bv, gv)
    finally:
        t.close()
    hv = 3.0 * xv.astype(f64) + bv * gv
    np.testing.assert_allclose(dx, 6.0 * hv, atol=1e-5 * 6 * np.abs(hv).max())
    np.testing.assert_allclose(db, 2.0 * hv * gv, atol=1e-4)
    np.testing.assert_allclose(dg, (2.0 * hv * bv).sum(0), atol=1e-4)


def step64(p, m, v, tokens, target, kind, t, d, bits, clip_norm=None):
    """The step of step_graph in float64: the cost of each row of the batch, and the parameters after it."""
    P = {k: a.astype(f64) for k, a in p.items()}
    n = d["N"]
    has = tokens != 0

    def norm_back(x, dz):
        c = x - x.mean(-1, keepdims=True) if kind == "layer" else x
        dev = np.sqrt((c * c).mean(-1, keepdims=True) + 1e-5)
        dx = dz / dev - c * (dz * c).sum(-1, keepdims=True) / (x.shape[-1] * dev ** 3)
        return dx - (dz / dev).mean(-1, keepdims=True) if kind == "layer" else dx
    get = lambda k: P.get(k, 0.0)                                                                      # noqa: E731
    x0 = np.where(has[..., None], 2.0 * P["table"][tokens], 0.0)
    y0 = norm64(x0, kind) * P["gain0"] + get("bias0")
    b1 = np.tanh(y0 * P["scale1"])
    u1 = norm64(b1, kind) * P["post1"] + get("postbias1")
    h1 = 0.5 * x0 + P["gate1"] * u1
    y1 = norm64(h1, kind) * P["gain1"] + get("bias1")
    b2 = np.tanh(y1 * P["scale2"])
    h2 = h1 + b2
    y2 = norm64(h2, kind) * P["gain2"]
    g = {}
    dy2 = 2 * (y2 - target)
    s = lambda a: a.reshape(-1, a.shape[-1]).sum(0)                                                     # noqa: E731
    g["gain2"] = s(dy2 * norm64(h2, kind))
    dh = norm_back(h2, dy2 * P["gain2"])
    db2 = dh * (1 - b2 * b2)
    g["scale2"] = s(db2 * y1)
    dy1 = db2 * P["scale2"]
    g["gain1"], g["bias1"] = s(dy1 * norm64(h1, kind)), s(dy1)
    dh = dh + norm_back(h1, dy1 * P["gain1"])
    g["gate1"] = s(dh * u1)
    e = dh * P["gate1"]
    g["post1"], g["postbias1"] = s(e * norm64(b1, kind)), s(e)
    db1 = norm_back(b1, e * P["post1"]) * (1 - b1 * b1)
    g["scale1"] = s(db1 * y0)
    dy0 = db1 * P["scale1"]
    g["gain0"], g["bias0"] = s(dy0 * norm64(x0, kind)), s(dy0)
    dx0 = 0.5 * dh + norm_back(x0, dy0 * P["gain0"])
    g["table"] = np.zeros_like(P["table"])
    np.add.at(g["table"], tokens[has], 2.0 * dx0[has])
    g = {k: g[k] / n for k in P}
    if clip_norm is not None:
        total = np.sqrt(sum((a * a).sum() for a in g.values()))
        g = {k: a * clip_norm / max(total, clip_norm) for k, a in g.items()}
    out = {}
    for k in P:
        m[k] = 0.9 * m[k] + 0.1 * g[k]
        v[k] = 0.999 * v[k] + 0.001 * g[k] ** 2
        root = np.sqrt(v[k] / (1 - 0.999 ** t)) + 1e-8
        out[k] = P[k] * (1 - 1e-2 * (0.1 if k == "table" else 0.0)) - 1e-2 * m[k] / (1 - 0.9 ** t) / root
    return ((y2 - target) ** 2).sum((1, 2)), out, g


@pytest.mark.gpu
@pytest.mark.parametrize("kind,state_bits,clip_norm", [("rms", 32, None), ("layer", 32, None), ("rms", 8, None), ("layer", 8, 0.5)])
def test_training_steps_of_all_of_them(hip_runtime, kind, state_bits, clip_norm):
    """Three steps: the cost within 1e-4 of float64's (relative: it is a sum of thousands of squares of values that
    went through three norms), and parameters within what their gradients are off by.  A gradient of fp32 sums is
    within 2e-5 of the largest of its tensor; the first step of Adam is lr * sign(g) wherever |g| is far above that,
    so parameters are compared where every |g| was at least 100 times it: 1 % of lr a step.  With 8 bits the moments
    are off by up to 1.6 % (first) and 0.8 % (root of the second) more after the first step: 3 % of lr a step."""
    d, p, tokens, target, cost, opt, step = step_graph(kind, state_bits, gradient_clip_norm=clip_norm)
    rs = np.random.RandomState(5)
    t = transformer()
    try:
        train = t.computation([step], tokens, target)            # (its value is the batch's cost before the update)
        read = {k: t.computation(q) for k, q in p.items()}
        values = {k: np.array(f()) for k, f in read.items()}
        m, v = ({k: np.zeros(a.shape) for k, a in values.items()} for _ in range(2))
        sure = {k: np.ones(a.shape, bool) for k, a in values.items()}
        want = values
        for n in range(1, 4):
            tk = rs.randint(0, d["V"], (d["N"], d["T"])).astype(np.int32)
            tg = rs.normal(0, 1, (d["N"], d["T"], d["F"])).astype(f32)
            total, = train(tk, tg)
            # (each step is compared from where the device is)
            expected, want, g = step64(values, m, v, tk, tg, kind, n, d, state_bits, clip_norm)
            np.testing.assert_allclose(total, expected.sum(), rtol=1e-4)
            values = {k: np.array(f()) for k, f in read.items()}
            for k, a in values.items():
                sure[k] &= np.abs(g[k]) > 100 * 2e-5 * np.abs(g[k]).max()
                off = np.abs(a - want[k])[sure[k]]
                assert off.size and off.max() <= (0.01 if state_bits == 32 else 0.03) * n * 1e-2 + 1e-6, (k, n, off.max())
        assert int(t.get_tensor_view_value(opt.update.step)) == 3
    finally:
        t.close()


@pytest.mark.gpu
def test_learning_rate_from_the_graph(hip_runtime):
    """A rate that is a scalar op, followed step by step."""
    N, F = axes(N=4, F=300)
    w, x, lr = ng.variable([F], initial_value=1.0), ng.placeholder([N, F]), ng.placeholder(())
    opt = neon.AdamW(learning_rate=lr * 2.0, weight_decay=0.0)
    step = opt.minimize(ng.sum(w * x, out_axes=[N]), variables=[w])
    t = transformer()
    try:
        f, read = t.computation([step], x, lr), t.computation(w)
        xv = np.ones((4, 300), f32)
        at = 1.0
        for rate in (0.5, 0.25, 0.0):
            f(xv, f32(rate))
            at -= 2.0 * rate                    # a constant gradient: every step is the rate
            np.testing.assert_allclose(read(), at, atol=1e-5)
    finally:
        t.close()


@pytest.mark.gpu
@pytest.mark.parametrize("param", [f32, np.float16])
def test_a_step_of_half_precision_tensors(hip_runtime, param):
    """fp16 table, stream and gradients.  A result is rounded once (2^-11).  The gradients are taken at the stored
    stream, each of whose values is off by 2^-11 of itself, at most 4 standard deviations here, and meets three
    terms of the norm's Jacobian: 12 * 2^-11 of the largest gradient, the rows' own rounding and that of their sum
    making it 16 (the gains' sums over 30 rows: of the sum of the largest terms)."""
    f16, half = np.dtype(np.float16), 2.0 ** -11
    V, F, T, N = axes(V=11, F=24, T=5, N=6)
    rs = np.random.RandomState(2)
    tv, wv = rs.normal(0, 1, (11, 24)).astype(f16), rs.normal(1, 0.2, 24).astype(f16).astype(param)
    cv, tk = rs.normal(0, 1, (6, 5, 24)).astype(f16), rs.randint(0, 11, (6, 5)).astype(np.int32)
    table, w = ng.variable([V, F], initial_value=tv, dtype=f16), ng.variable([F], initial_value=wv, dtype=np.dtype(param))
    tokens, c = ng.placeholder([N, T], dtype=i32), ng.placeholder([N, T, F], dtype=f16)
    x = ng.embedding(table, tokens, scale=2.0)
    y, h = ng.block_norm(x, c, gain=w, kind="layer")
    cost = ng.sum(y * c, out_axes=())
    dtable, dw = ng.deriv(cost, table), ng.deriv(cost, w)
    update = hiprows.AdamWOp([table], [dtable], lr=0.125, weight_decay=[0.0])
    t = transformer()
    try:
        step = t.computation([y, h, dtable, dw, update], tokens, c)
        read = t.computation(table)
        got = [np.array(a) for a in step(tk, cv)[:4]]
        after = np.array(read())
    finally:
        t.close()
    t64, w64, c64 = tv.astype(f64), wv.astype(f64), cv.astype(f64)
    h64 = 2.0 * t64[tk] + c64
    y64 = norm64(h64, "layer") * w64
    m = h64 - h64.mean(-1, keepdims=True)
    dev = np.sqrt((m * m).mean(-1, keepdims=True) + 1e-5)
    dz = c64 * w64
    dx = dz / dev - m * (dz * m).mean(-1, keepdims=True) / dev ** 3 - (dz / dev).mean(-1, keepdims=True)
    want = np.zeros((11, 24))
    np.add.at(want, tk, 2.0 * dx)
    size = np.zeros((11, 24))
    np.add.at(size, tk, np.full(dx.shape, 2.0 * np.abs(dx).max()))
    np.testing.assert_allclose(got[0], y64, rtol=half, atol=1e-5)
    np.testing.assert_allclose(got[1], h64, rtol=half, atol=1e-6)
    assert (np.abs(got[2] - want) <= 16 * half * size).all()
    terms = np.abs(c64 * norm64(h64, "layer"))
    assert np.abs(got[3] - (c64 * norm64(h64, "layer")).sum((0, 1))).max() <= 16 * half * 30 * terms.max()
    # the first step is lr * sign(g), off by eps / |g| of it, and rounded to fp16
    sure = np.abs(want) > np.maximum(16 * half * size, 1e-3)
    assert sure.any()
    stepped = t64 - 0.125 * np.sign(want)
    assert (np.abs(after - stepped) <= half * np.abs(stepped) + 0.125 * 1e-4)[sure].all()


def test_numbers_that_do_not_fit_are_refused():
    V, F, N = axes(V=10, F=8, N=5)
    table, tokens = ng.placeholder([V, F]), ng.placeholder([N], dtype=i32)
    for pad in (2 ** 31, -2 ** 31 - 1):
        with pytest.raises(ValueError):
            ng.embedding(table, tokens, pad_idx=pad)
