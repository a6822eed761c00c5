"""Operands of the row operators whose layout the graph passes change: 1 * x and x + 0 become views of x, a product
with a constant a broadcast of it, and x16 * 1.0 (float32) becomes x16.  Each graph is lowered without a device, where
every operand that a kernel is bound to has to be what the kernel reads, and run against NumPy in float64.

Bounds: a hundred roundings of 2^-24 in a row at most, relative to the magnitudes that meet: 1e-5 of the largest.
"""
import numpy as np
import pytest

import ngraph_hip as ng
import ngraph_hip.transformers as ngt
from ngraph_hip.frontends import neon
from ngraph_hip.runtime import NGH_F16, NGH_F32
from ngraph_hip.transformers import hiprows
from ngraph_hip.transformers.hipdevice import _td

f32, f64, i32, f16 = np.float32, np.float64, np.dtype(np.int32), np.dtype(np.float16)
DIMS = dict(N=3, T=4, F=20, V=7)
EPS = 1e-5


def axes(names):
    return [ng.make_axis(DIMS[k], name=k) for k in names]


class Case(object):
    """Returns of a computation, its parameters with values, and what float64 says of the returns."""

    def __init__(self, returns, given, want):
        self.returns, self.given, self.want = returns, given, want


def rms(x):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS)


def rms_back(x, dz):
    dev = np.sqrt((x * x).mean(-1, keepdims=True) + EPS)
    return dz / dev - x * (dz * x).sum(-1, keepdims=True) / (x.shape[-1] * dev ** 3)


def norm_graph(cost_of):
    """Derivatives of a cost of y and h in x, b and the gain."""
    N, T, F = axes("NTF")
    rs = np.random.RandomState(0)
    x, b, w, s = ng.placeholder([N, T, F]), ng.placeholder([N, T, F]), ng.placeholder([F]), ng.placeholder(())
    xv, bv, wv, sv = rs.normal(0, 1, (3, 4, 20)).astype(f32), rs.normal(0, 1, (3, 4, 20)).astype(f32), rs.normal(1, 0.3, 20).astype(f32), f32(0.7)
    y, h = ng.block_norm(x, b, gain=w, residual_scale=0.5)
    cost, dy, dh = cost_of(y, h, w, s, wv.astype(f64), f64(sv))
    through_gain = dy if isinstance(dy, np.ndarray) or dy != 0 else None
    hv = 0.5 * xv.astype(f64) + bv
    dy, dh = np.broadcast_to(dy, hv.shape), np.broadcast_to(dh, hv.shape)
    d = dh + rms_back(hv, dy * wv)
    returns, want = [ng.deriv(cost, x), ng.deriv(cost, b)], [0.5 * d, d]
    if through_gain is not None and cost_of is not times_vector:
        returns.append(ng.deriv(cost, w))
        want.append((dy * rms(hv)).sum((0, 1)))
    return Case(returns, [(x, xv), (b, bv), (w, wv), (s, sv)], want)


def times_vector(y, h, w, s, wv, sv):
    return ng.sum(y * w, out_axes=()), wv, 0.0


def times_two(y, h, w, s, wv, sv):
    return ng.sum(2.0 * y, out_axes=()), 2.0, 0.0


def times_scalar(y, h, w, s, wv, sv):
    return ng.sum(y * s, out_axes=()), sv, 0.0


def plain_sum(y, h, w, s, wv, sv):
    return ng.sum(y, out_axes=()), 1.0, 0.0


def stream_times_vector(y, h, w, s, wv, sv):
    return ng.sum(h * w, out_axes=()), 0.0, wv


def both(y, h, w, s, wv, sv):
    return ng.sum(3.0 * y, out_axes=()) + ng.sum(h * s, out_axes=()), 3.0, sv


def embedding_times_vector():
    V, N, T, F = axes("VNTF")
    rs = np.random.RandomState(1)
    table, tokens, w = ng.placeholder([V, F]), ng.placeholder([T, N], dtype=i32), ng.placeholder([F])
    tv, kv, wv = rs.normal(0, 1, (7, 20)).astype(f32), rs.randint(-1, 8, (4, 3)).astype(np.int32), rs.normal(0, 1, 20).astype(f32)
    e = ng.embedding(table * 1.0, ng.axes_with_order(tokens, ng.make_axes([N, T])), scale=1.5, pad_idx=2)
    want = np.zeros((7, 20))
    has = (kv >= 0) & (kv < 7) & (kv != 2)
    np.add.at(want, kv[has], 1.5 * wv.astype(f64))
    rows = np.where(has.T[..., None], 1.5 * tv[np.where(has, kv, 0).T].astype(f64), 0.0)
    return Case([e, ng.deriv(ng.sum(e * w, out_axes=()), table)], [(table, tv), (tokens, kv), (w, wv)], [rows, want])


def broadcast_vectors():
    """A gain, a bias and a gate that are one number each."""
    N, T, F = axes("NTF")
    rs = np.random.RandomState(2)
    x, s, q = ng.placeholder([N, T, F]), ng.placeholder(()), ng.placeholder([N])
    xv, qv = rs.normal(0, 1, (3, 4, 20)).astype(f32), rs.normal(1, 0.2, 3).astype(f32)
    y, h = ng.block_norm(x, x * 2.0, gain=ng.broadcast(s, [F]) * 1.0, bias=ng.broadcast(ng.constant(0.25), [F]), post_gain=ng.broadcast(s, [F]) + 0.0,
                         gate=ng.broadcast(q, [N, F]) * 1.0)
    v = xv.astype(f64)
    hv = v + rms(2 * v) * 0.75 * qv[:, None, None]
    return Case([y, h], [(x, xv), (s, f32(0.75)), (q, qv)], [rms(hv) * 0.75 + 0.25, hv])


def transposed_rows():
    N, T, F = axes("NTF")
    rs = np.random.RandomState(3)
    x, p = ng.placeholder([F, N, T]), ng.placeholder([N, F])
    xv, pv = rs.normal(0, 1, (20, 3, 4)).astype(f32), rs.normal(0, 1, (3, 20)).astype(f32)
    whole = ng.make_axes([N, T, F])
    y, h = ng.block_norm(ng.axes_with_order(x, whole) + 0.0, ng.axes_with_order(ng.broadcast(p, [N, F, T]), whole) * 1.0)
    hv = np.moveaxis(xv, 0, -1).astype(f64) + pv[:, None, :]
    return Case([y, h], [(x, xv), (p, pv)], [rms(hv), hv])


def zero_block():
    N, F = axes("NF")
    x = ng.placeholder([N, F])
    xv = np.random.RandomState(4).normal(0, 1, (3, 20)).astype(f32)
    return Case(list(ng.block_norm(x, x * 0.0)), [(x, xv)], [rms(xv.astype(f64)), xv.astype(f64)])


def half_as_single():
    """x16 * 1.0 and w16 + 0.0 have dtype float32 until the passes make them x16 and w16."""
    N, F = axes("NF")
    rs = np.random.RandomState(5)
    x, b, w = ng.placeholder([N, F], dtype=f16), ng.placeholder([N, F]), ng.placeholder([F], dtype=f16)
    xv, bv, wv = rs.normal(0, 1, (3, 20)).astype(f16), rs.normal(0, 1, (3, 20)).astype(f32), rs.normal(1, 0.3, 20).astype(f16)
    hv = xv.astype(f64) + bv
    return Case(list(ng.block_norm(x * 1.0, b, gain=w + 0.0)), [(x, xv), (b, bv), (w, wv)], [rms(hv) * wv.astype(f64), hv])


CASES = {f.__name__: (lambda f=f: norm_graph(f)) for f in (times_vector, times_two, times_scalar, plain_sum, stream_times_vector, both)}
CASES.update((f.__name__, f) for f in (embedding_times_vector, broadcast_vectors, transposed_rows, zero_block, half_as_single))


def adamw_case(kind):
    """One step of W [V, F] with a gradient that is a broadcast, a transposed or a half precision view."""
    V, F = axes("VF")
    rs = np.random.RandomState(6)
    w0 = rs.normal(0, 1, (7, 20)).astype(f32)
    W = ng.variable([V, F], initial_value=w0)
    if kind == "broadcast":
        c, cv = ng.placeholder([F]), rs.normal(0, 1, 20).astype(f32)
        cost, g = ng.sum(W * c, out_axes=()), np.broadcast_to(cv.astype(f64), (7, 20))
    elif kind == "transposed":
        c, cv = ng.placeholder([F, V]), rs.normal(0, 1, (20, 7)).astype(f32)
        cost, g = ng.sum(W * ng.axes_with_order(c, ng.make_axes([V, F])), out_axes=()), cv.T.astype(f64)
    else:
        c, cv = ng.placeholder([V, F], dtype=f16), rs.normal(0, 1, (7, 20)).astype(f16)
        cost, g = ng.sum(W * (c * 1.0), out_axes=()), cv.astype(f64)
    rate = ng.placeholder((), dtype=f16)
    opt = neon.AdamW(learning_rate=rate * 1.0, weight_decay=0.0)
    step = opt.minimize(cost, variables=[W])
    return W, w0, c, cv, rate, opt, step, g


GRADS = ["broadcast", "transposed", "half"]


def lowered(returns, *params):
    t = ngt.make_transformer_factory("hipgpu", dry_run=True)()
    f = t.computation(returns, *params)
    t.initialize()
    group = t.kernel_groups[f]
    group.bind()
    for k in group.kernels:
        k.execute()
    return t, [k for k in group.kernels if isinstance(k, hiprows.RowKernel)]


def assert_rows_in_order(td, dtype):
    """The elements of the description follow one another in memory that holds them all, stored as dtype."""
    acc = 1
    for n, stride in zip(reversed(td.axes.lengths), reversed(td.full_strides)):
        assert n == 1 or stride == acc, (td.axes, td.full_strides)
        acc *= n
    assert td.dtype == dtype and td.base.tensor_size >= acc * dtype.itemsize


@pytest.mark.parametrize("name", sorted(CASES))
def test_what_kernels_are_bound_to(name):
    case = CASES[name]()
    t, kernels = lowered(case.returns, *[p for p, _ in case.given])
    try:
        assert kernels
        for k in kernels:
            if isinstance(k, (hiprows.EmbeddingKernel, hiprows.EmbeddingGradKernel)):
                codes = [k.spec.table_dtype, NGH_F32] if isinstance(k, hiprows.EmbeddingKernel) else [NGH_F32, k.spec.y_dtype]
                dtypes = [np.dtype(f32), i32] if isinstance(k, hiprows.EmbeddingKernel) else [i32, np.dtype(f32)]
                assert codes == [NGH_F32, NGH_F32]
            else:
                names = k.op.operand_names
                kind = {NGH_F32: np.dtype(f32), NGH_F16: f16}
                vectors = ("gain", "bias", "post_gain", "post_bias", "gate")
                dtypes = [kind[k.spec.param_dtype if n in vectors else k.spec.dtype] for n in names]
            for a, dtype in zip(k.op.args, dtypes):
                assert_rows_in_order(_td(a.forwarded), dtype)
    finally:
        t.close()


@pytest.mark.parametrize("kind", GRADS)
def test_what_the_update_is_bound_to(kind):
    W, w0, c, cv, rate, opt, step, g = adamw_case(kind)
    t, kernels = lowered(step, c, rate)
    try:
        update, = [k for k in kernels if isinstance(k, hiprows.AdamWKernel)]
        assert len(update.op.args) == 2
        for a in update.op.args:
            assert_rows_in_order(_td(a.forwarded), np.dtype(f32))
    finally:
        t.close()


def test_a_view_behind_the_last_pass_is_refused():
    """A pass that somebody adds behind the others can still make a view of an operand: no kernel takes it."""
    from ngraph_hip.op_graph import op_graph as og
    from ngraph_hip.transformers.passes.passes import PeepholeGraphPass
    N, F = axes("NF")
    x, w = ng.placeholder([N, F]), ng.placeholder([F])
    marked = w * 3.0

    class Late(PeepholeGraphPass):
        def visit(self, op, *args):
            if op is marked.forwarded and not isinstance(op, og.BroadcastOp):
                self.replace_op(op, ng.broadcast(ng.constant(3.0), [F]))
    t = ngt.make_transformer_factory("hipgpu", dry_run=True)()
    t.register_graph_pass(Late())
    try:
        f = t.computation(ng.block_norm(x, gain=marked)[0], x, w)
        with pytest.raises(NotImplementedError) as e:
            t.initialize()
            t.kernel_groups[f].bind()
        assert "BlockNormOp" in str(e.value) and "strides (0,)" in str(e.value)
    finally:
        t.close()


def test_flex_operands_behind_a_view_are_refused():
    N, F = axes("NF")
    x = ng.placeholder([N, F])
    t = ngt.make_transformer_factory("flexhip", dry_run=True)()
    try:
        with pytest.raises(Exception) as e:
            f = t.computation(ng.block_norm(x * 1.0)[0], x)
            t.initialize()
            t.kernel_groups[f].bind()
        assert "flex" in str(e.value)
    finally:
        t.close()


def product_of_variables(state_bits):
    """sum(v * w * 1) + sum(v * u): the gradient of either factor is the other one's memory."""
    F, = axes("F")
    rs = np.random.RandomState(7)
    values = [rs.normal(0, 1, 20).astype(f32) for _ in range(3)]
    v, w, u = variables = [ng.variable([F], initial_value=a) for a in values]
    opt = neon.AdamW(learning_rate=0.25, weight_decay=0.0, state_bits=state_bits)
    step = opt.minimize(ng.sum(v * w, out_axes=()) + ng.sum(v * u, out_axes=()), variables=variables)
    return variables, values, opt, step


@pytest.mark.parametrize("state_bits", [32, 8])
def test_a_gradient_that_is_another_variable_is_copied(state_bits):
    variables, values, opt, step = product_of_variables(state_bits)
    t, kernels = lowered(step)
    try:
        update, = [k for k in kernels if isinstance(k, hiprows.AdamWKernel)]
        held = [x.tensor_description().base for x in variables]
        for a in update.op.args:
            assert_rows_in_order(_td(a.forwarded), np.dtype(f32))
            assert _td(a.forwarded).base not in held
    finally:
        t.close()


@pytest.mark.gpu
@pytest.mark.parametrize("state_bits", [32, 8])
def test_updates_by_gradients_that_are_other_variables(hip_runtime, state_bits):
    """Steps of 0.25 by the signs of the values before the step, first moments a tenth of them (8 bits: to half a code)."""
    variables, values, opt, step = product_of_variables(state_bits)
    t = ngt.make_transformer_factory("hipgpu")()
    try:
        f, read = t.computation([step]), [t.computation(x) for x in variables]
        f()
        after = [np.array(r()) for r in read]
        m = [np.array(t.get_tensor_view_value(x)) for x in opt.update.m]
    finally:
        t.close()
    v, w, u = [a.astype(f64) for a in values]
    for a, before, g, mk in zip(after, (v, w, u), (w + u, v, v), m):
        np.testing.assert_allclose(a, before - 0.25 * g / (np.abs(g) + 1e-8), rtol=0, atol=2.0 ** -24 * (12 * 0.25 + 4 * np.abs(before).max()))
        if state_bits == 32:
            np.testing.assert_allclose(mk, (1 - 0.9) * g, rtol=6 * 2.0 ** -24, atol=0)
        else:
            np.testing.assert_allclose(mk, np.sign(g) * 127 * np.sqrt(np.abs(g) / np.abs(g).max()), rtol=0, atol=0.501)


@pytest.mark.gpu
@pytest.mark.parametrize("name", sorted(CASES))
def test_results_against_float64(hip_runtime, name):
    case = CASES[name]()
    t = ngt.make_transformer_factory("hipgpu")()
    try:
        got = [np.array(a) for a in t.computation(case.returns, *[p for p, _ in case.given])(*[v for _, v in case.given])]
    finally:
        t.close()
    for g, w in zip(got, case.want):
        # (a gradient through a norm is a difference of terms of the size of the cotangent over the row's deviation)
        np.testing.assert_allclose(g, w, rtol=0, atol=1e-5 * max(np.abs(w).max(), 1.0))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", GRADS)
def test_updates_against_float64(hip_runtime, kind):
    W, w0, c, cv, rate, opt, step, g = adamw_case(kind)
    t = ngt.make_transformer_factory("hipgpu")()
    try:
        f, read = t.computation([step], c, rate), t.computation(W)
        f(cv, np.float16(0.25))
        after, m = np.array(read()), np.array(t.get_tensor_view_value(opt.update.m[0]))
    finally:
        t.close()
    np.testing.assert_allclose(m, (1 - 0.9) * g, rtol=4 * 2.0 ** -24, atol=0)
    # the first step is the rate times g / (|g| + eps), within 12 roundings of it and 4 of the parameter
    want = w0 - 0.25 * g / (np.abs(g) + 1e-8)
    np.testing.assert_allclose(after, want, rtol=0, atol=2.0 ** -24 * (12 * 0.25 + 4 * np.abs(w0).max()))
