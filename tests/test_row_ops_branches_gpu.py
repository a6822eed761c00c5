"""The kernels that only larger or differently laid out calls reach, against NumPy: AdamW's four pieces a lane, the embedding
gradient's one-chunk sort, its sorts with rows on any boundary, and tables of which the sort's launches clear only a part."""
import numpy as np
import pytest

from test_adamw_gpu import HYPER, Model
from test_embedding_gpu import GRAD_PAIRS, gradient, tokens_for
from row_helpers import DTYPES, EPS, HALF, Pool, assert_within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("types", [("f32", "f32"), ("f32", "bf16"), ("bf16", "f16")], ids="-".join)
def test_adamw_plans_of_many_elements(hip_runtime, types, bits, shift):
    """5.3 M elements: above 16 pieces of 1024 for each compute unit a lane has four pieces of a chunk of 4096.  Chunks that are
    full, one element short or long, end within a piece, a block or a lane's elements, and tensors far smaller than one."""
    sizes = [4096 * 400, 4096 * 300 + 1, 4096 * 300 - 1, 4096 * 200 + 1024, 4096 * 90 + 2050, 4095, 4097, 3 * 1024 + 256, 255, 1, 0, 12289]
    assert sum(n // 1024 for n in sizes) > 16 * 304
    with Pool(hip_runtime) as pool:
        model = Model(pool, hip_runtime, sizes, types, bits, copy="bf16" if types[0] == "f32" else None, shift=shift)
        for step in (1, 2):
            hip_runtime.adamw_step(model.plan, step, **HYPER)
            model.check_step(step)
        model.free()


@pytest.mark.parametrize("accumulate", [False, True], ids=["written", "added"])
@pytest.mark.parametrize("pair", GRAD_PAIRS, ids="-".join)
@pytest.mark.parametrize("n,vocab,width,kind", [(2048, 300, 40, "zipf"), (2049, 300, 40, "zipf"), (3000, 5000, 33, "any"), (3001, 77, 264, "two"),
                                                (4095, 4, 8, "one"), (4096, 20011, 72, "zipf"), (4096, 4096, 16, "distinct")])
def test_gradient_of_one_chunk(hip_runtime, pair, accumulate, n, vocab, width, kind):
    tokens = tokens_for(np.random.RandomState(n), n, vocab, kind)
    with Pool(hip_runtime) as pool:
        got, want, bound = gradient(hip_runtime, pool, tokens, vocab, width, pair[0], pair[1], 2.5, 1, accumulate, runs=2)
    np.testing.assert_array_equal(got[0], got[1])
    assert_within(got[0], want, bound)


@pytest.mark.parametrize("pair", GRAD_PAIRS, ids="-".join)
@pytest.mark.parametrize("accumulate", [False, True], ids=["written", "added"])
@pytest.mark.parametrize("n", [3000, 10000, 17000])
@pytest.mark.parametrize("y_stride,table_stride,shift", [(136, 160, 0), (131, 129, 0), (128, 128, 1), (133, 128, 5)])
def test_gradient_of_strided_and_shifted_rows_by_every_sort(hip_runtime, pair, accumulate, n, y_stride, table_stride, shift):
    tokens = tokens_for(np.random.RandomState(n), n, 900, "zipf")
    with Pool(hip_runtime) as pool:
        got, want, bound = gradient(hip_runtime, pool, tokens, 900, 128, pair[0], pair[1], 1.5, -1, accumulate, y_stride, table_stride, shift)
    assert_within(got[0], want, bound)


@pytest.mark.parametrize("n", [1500, 3000, 5000, 10000, 17000])
@pytest.mark.parametrize("y_dtype,table_dtype,width", [("f32", "f32", 1024), ("f16", "f32", 1023), ("bf16", "bf16", 2048)])
def test_gradient_into_a_table_of_several_64_mebibytes(hip_runtime, y_dtype, table_dtype, width, n):
    """195 MiB: the sort has cleared nothing, 64 (one launch) or 128 MiB (two) of it, and the sums clear the rest; every row starts as
    something else.  Whole numbers: any order adds up exactly."""
    rt, rs, vocab = hip_runtime, np.random.RandomState(n), 50003
    tokens = tokens_for(rs, n, vocab, "any")
    edges = [0, 16383, 16384, 16385, 32767, 32768, 32769, 49151, 49152, vocab - 1]      # of 64 MiB in rows of 4 KiB
    tokens[::7] = rs.choice(edges, len(tokens[::7]))
    few, which = rs.randint(-4, 5, (64, width)).astype(np.float32), rs.randint(0, 64, n)
    with Pool(rt) as pool:
        dy, t, table = pool.rows((n, width), y_dtype, few[which]), pool.array(tokens), pool.rows((vocab, width), table_dtype)
        spec = rt.embedding_grad_spec(n, vocab, width, t.ptr, dy.ptr, table.ptr, DTYPES[y_dtype], DTYPES[table_dtype], 0.5)
        spec.workspace_bytes = rt.embedding_grad_workspace(spec)
        spec.workspace = pool.bytes(spec.workspace_bytes).ptr
        rt.embedding_grad(spec)
        got = table.get()
    weight = np.zeros((vocab, 64), np.float32)
    np.add.at(weight, (tokens, which), np.float32(0.5))
    want = weight @ few                                          # (halves of whole numbers below 2^23: exact in any order)
    np.testing.assert_array_less(np.abs(got - want), np.abs(want) * (HALF["bf16"] if table_dtype == "bf16" else 0.0) + 1e-30)


def layer_norm64(x, off):
    """The layer norm of rows x whose elements are off by up to `off`: the result, what it is off by, the reciprocal root and what
    that is off by (relative).  A sum of a row has 16 roundings in a row here at most (up to 8 elements a lane, 6 levels of lanes,
    2 wavefronts): a mean is off by 18 * 2^-24 of the magnitudes' mean, the variance around it by what the differences are."""
    m = x.mean(1, keepdims=True)
    c = x - m
    var = (c * c).mean(1, keepdims=True) + 1e-5
    c_off = off + off.mean(1, keepdims=True) + 18 * EPS * np.abs(x).mean(1, keepdims=True) + EPS * np.abs(c)
    r_off = ((np.abs(c) * c_off).mean(1, keepdims=True) + (c_off * c_off).mean(1, keepdims=True)) / var + 24 * EPS
    r = 1.0 / np.sqrt(var)
    return c * r, (c_off * r + np.abs(c) * r * (r_off + EPS)) * (1 + r_off), r, r_off


def back64(t, t_off, xh, xh_off, r, r_off):
    """r (t - xh mean(t xh) - mean(t)) and what it is off by."""
    mean = lambda a: a.mean(1, keepdims=True)                                                           # noqa: E731
    along, along_off = mean(t * xh), mean(t_off * np.abs(xh) + np.abs(t) * xh_off + t_off * xh_off) + 20 * EPS * mean(np.abs(t * xh))
    level, level_off = mean(t), mean(t_off) + 20 * EPS * mean(np.abs(t))
    inner = t - xh * along - level
    size = np.abs(t) + np.abs(xh * along) + np.abs(level)
    off = t_off + np.abs(xh) * along_off + xh_off * (np.abs(along) + along_off) + level_off + 4 * EPS * size
    return r * inner, r * (off + np.abs(inner) * r_off) * (1 + r_off)


@pytest.mark.parametrize("far", ["stream", "block"])
def test_layer_norms_of_rows_two_thousand_from_zero(hip_runtime, far):
    """A mean a thousand times the spread: the variance is taken around the mean.  The bounds are followed along the formulas; zeros, and
    a variance as the mean square less the mean's square in fp32, lie outside them."""
    rt, rows, width = hip_runtime, 40, 512
    rs = np.random.RandomState(2)
    f32, f64 = np.float32, np.float64
    x = (rs.normal(2000.0 if far == "stream" else 0.0, 1.5, (rows, width))).astype(f32)
    b = (rs.normal(2000.0 if far == "block" else 0.0, 1.5, (rows, width))).astype(f32)
    dy, dh = (rs.normal(0, 1, (rows, width)).astype(f32) for _ in range(2))
    gain, post = (rs.normal(1, 0.2, (1, width)).astype(f32) for _ in range(2))
    X, B, DY, DH, W, P = (a.astype(f64) for a in (x, b, dy, dh, gain, post))
    zero = np.zeros_like(X)
    bh, bh_off, rb, rb_off = layer_norm64(B, zero)
    u, u_off = bh * P, bh_off * np.abs(P) + 2 * EPS * np.abs(bh * P)
    h, h_off = X + u, u_off + 2 * EPS * (np.abs(X) + np.abs(u))
    n, n_off, _, _ = layer_norm64(h, h_off)
    want = {"h": (h, h_off), "y": (n * W, n_off * np.abs(W) + EPS * np.abs(n * W))}
    stored = h.astype(f32)
    hh, hh_off, r, r_off = layer_norm64(stored.astype(f64), zero)
    d, d_off = back64(DY * W, EPS * np.abs(DY * W), hh, hh_off, r, r_off)
    d, d_off = d + DH, d_off + 2 * EPS * (np.abs(d) + np.abs(DH))
    db, db_off = back64(d * P, d_off * np.abs(P) + EPS * np.abs(d * P), bh, bh_off, rb, rb_off)
    k = (64 + rows) * EPS
    want.update(dx=(d, d_off), db=(db, db_off),
                dgain=((DY * hh).sum(0), (np.abs(DY) * hh_off).sum(0) + k * np.abs(DY * hh).sum(0)),
                dpost_gain=((d * bh).sum(0), (np.abs(d) * bh_off + d_off * np.abs(bh) + d_off * bh_off).sum(0) + k * np.abs(d * bh).sum(0)))
    with Pool(rt) as pool:
        t = {n: pool.rows(a.shape, "f32", a) for n, a in (("x", x), ("b", b), ("dy", dy), ("dh", dh), ("gain", gain), ("post_gain", post))}
        t.update((n, pool.rows((rows, width), "f32")) for n in ("h", "y", "dx", "db"))
        t.update((n, pool.rows((1, width), "f32")) for n in ("dgain", "dpost_gain"))
        spec = rt.block_norm_spec(rows, width, "layer", post_norm=True, **{n: a.ptr for n, a in t.items()})
        spec.workspace_bytes = rt.block_norm_grad_workspace(spec)
        spec.workspace = pool.bytes(spec.workspace_bytes).ptr
        rt.block_norm(spec)
        forward = {n: t[n].get() for n in ("h", "y")}
        rt.memcpy_h2d(t["h"].ptr, stored)
        rt.block_norm_grad(spec)
        got = dict(forward, **{n: t[n].get() for n in ("dx", "db", "dgain", "dpost_gain")})
    for n, (value, off) in want.items():
        assert_within(got[n].reshape(value.shape), value, off * 1.01 + EPS * np.abs(value), n)
        # what the bound is worth: a result of zeros lies outside it
        assert (np.abs(value) > off * 1.01 + EPS * np.abs(value)).mean() > 0.5, n
    name, rough = ("y", stored) if far == "stream" else ("h", b)
    one_pass = 1 / np.sqrt((rough * rough).mean(1, keepdims=True, dtype=f32) - np.square(rough.mean(1, keepdims=True, dtype=f32)) + f32(1e-5))
    centred = rough - rough.mean(1, keepdims=True, dtype=f32)
    spoiled = centred * one_pass * gain if far == "stream" else x + centred * one_pass * post
    assert (np.abs(spoiled - want[name][0]) > want[name][1] * 1.01 + EPS * np.abs(want[name][0])).any()
