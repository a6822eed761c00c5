"""The operators over rows and parameters in the graphs of a foreign package (`plugin.bind(...).hiprows`), whose tensor descriptions
have strides and offsets in bytes: the kernels are bound to what the native graph binds them to, and give the same bits."""
import importlib

import numpy as np
import pytest

import ngraph_hip.plugin as plugin
import plugin_clone

f32, f64, i32 = np.float32, np.float64, np.dtype(np.int32)
DIMS = dict(V=11, F=20, N=3, T=4)


@pytest.fixture(scope="module")
def fronts(tmp_path_factory):
    """(graph module, row operators, transformer factory) of the package and of this repository."""
    import ngraph_hip.op_graph.op_graph as own_og
    import ngraph_hip.transformers as own_ngt
    from ngraph_hip.transformers import hiprows
    name = plugin_clone.make_clone(tmp_path_factory.mktemp("clone"), "ngrows")
    bound = plugin.bind(name, adapt=lambda td: plugin.adapt_tensor_description(plugin_clone.ByteDescription(td)))
    og, base = (importlib.import_module(name + m) for m in (".op_graph.op_graph", ".transformers.base"))
    return (og, bound.hiprows, base.make_transformer_factory), (own_og, hiprows, own_ngt.make_transformer_factory)


def values():
    rs = np.random.RandomState(0)
    return dict(table=rs.normal(0, 1, (11, 20)).astype(f32), gain=rs.normal(1, 0.2, 20).astype(f32), gate=rs.normal(1, 0.2, (3, 20)).astype(f32),
                tokens=rs.randint(-1, 12, (4, 3)).astype(np.int32), c=rs.normal(0, 1, (20, 3, 4)).astype(f32), w=rs.normal(0, 1, 20).astype(f32))


def step(og, hiprows, state_bits):
    """Tokens and a cotangent in another order than the rows', a gate for each sequence, a folded adjoint of the stream, one update."""
    autodiff = importlib.import_module(og.__name__.replace(".op_graph.op_graph", ".op_graph.autodiff"))
    V, F, N, T = (og.make_axis(DIMS[k], name=k) for k in "VFNT")
    v = values()
    table, gain, gate = (og.variable(a, initial_value=v[k]) for k, a in (("table", [V, F]), ("gain", [F]), ("gate", [N, F])))
    tokens, c, w = og.placeholder([T, N], dtype=i32), og.placeholder([F, N, T]), og.placeholder([F])
    e = hiprows.embedding(table, og.axes_with_order(tokens, og.make_axes([N, T])), 2.0, 3)
    y, h = hiprows.block_norm(e, og.tanh(e), gain=gain, gate=gate, post_norm=True, kind="layer", residual_scale=0.5)
    cost = og.sum(y * og.axes_with_order(c, og.make_axes([N, T, F])), out_axes=()) + og.sum(h * w, out_axes=())
    variables = [table, gain, gate]
    grads = [autodiff.deriv(cost, x) for x in variables]
    update = hiprows.AdamWOp(variables, grads, lr=0.125, weight_decay=[0.1, 0.0, 0.0], state_bits=state_bits)
    return update, [y, h] + grads, (tokens, c, w), variables


def fields(spec):
    """What does not depend on where things lie."""
    return {n: getattr(spec, n) for n, t in spec._fields_ if n not in POINTERS} if spec is not None else None


POINTERS = ("tokens", "table", "y", "workspace", "x", "b", "gain", "bias", "post_gain", "post_bias", "gate", "h", "dy", "dh", "dx", "db", "dgain", "dbias",
            "dpost_gain", "dpost_bias", "dgate")


@pytest.mark.parametrize("state_bits", [32, 8])
def test_the_package_lowers_to_the_same_calls(fronts, state_bits):
    lowered = []
    for og, hiprows, factory in fronts:
        t = factory("hipgpu", dry_run=True)()
        try:
            update, results, given, variables = step(og, hiprows, state_bits)
            f = t.computation([update] + results, *given)
            t.initialize()
            group = t.kernel_groups[f]
            group.bind()
            rows = [k for k in group.kernels if isinstance(k, hiprows.RowKernel)]
            lowered.append(([type(k).__name__ for k in group.kernels], [(k.name, fields(k.spec)) for k in rows],
                            [sorted(n for n in POINTERS if getattr(k.spec, n, None)) for k in rows]))
            for k in group.kernels:
                k.execute()
        finally:
            t.close()
    assert lowered[0] == lowered[1]
    assert sorted(n for n, _ in lowered[0][1]) == ["adamw", "block_norm", "block_norm_grad", "embedding", "embedding_grad"]


@pytest.mark.gpu
@pytest.mark.parametrize("state_bits", [32, 8])
def test_the_package_gets_the_same_bits(hip_runtime, fronts, state_bits):
    v, got = values(), []
    for og, hiprows, factory in fronts:
        t = factory("hipgpu")()
        try:
            update, results, given, variables = step(og, hiprows, state_bits)
            f, read = t.computation([update] + results, *given), [t.computation(x) for x in variables]
            out = f(v["tokens"], v["c"], v["w"])
            got.append([np.array(a) for a in out[1:]] + [np.array(r()) for r in read])
        finally:
            t.close()
    for a, b in zip(*got):
        np.testing.assert_array_equal(a, b)
    y, h, dtable = got[0][0], got[0][1], got[0][2]
    # (the numbers themselves: the native graph's have tests of their own)
    tk = v["tokens"].T
    has = (tk >= 0) & (tk < 11) & (tk != 3)
    e = np.where(has[..., None], 2.0 * v["table"][np.where(has, tk, 0)].astype(f64), 0.0)
    b = np.tanh(e)
    b = b - b.mean(-1, keepdims=True)
    want = 0.5 * e + v["gate"][:, None, :] * (b / np.sqrt((b * b).mean(-1, keepdims=True) + 1e-5))
    np.testing.assert_allclose(h, want, rtol=0, atol=1e-5 * np.abs(want).max())
    assert np.abs(dtable).max() > 0 and np.isfinite(y).all()
