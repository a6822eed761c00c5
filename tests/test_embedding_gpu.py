"""ngh_embedding / ngh_embedding_grad against NumPy in float64.

Bounds.  Lookup: one product in fp32 and one rounding to the result's type.  Gradient: a sum of c terms
in fp32 in any order is off by at most c * 2^-24 times the sum of the magnitudes (first order), then
one product, one addition when accumulating and one rounding to the table's type; 2^-24 more of
each covers the second order for the c here.
"""
import numpy as np
import pytest

from row_helpers import DTYPES, EPS, HALF, TINY, Pool, assert_within, rounded

pytestmark = pytest.mark.gpu

f32, f64 = np.float32, np.float64
PAIRS = [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")]      # table, rows


def tokens_for(rs, n, vocab, kind):
    if kind == "zipf":
        t = np.minimum((np.exp(rs.uniform(size=n) * np.log(vocab + 1.0)) - 1).astype(np.int64), vocab - 1)
        t = rs.permutation(vocab)[t]
    elif kind == "one":
        t = np.full(n, rs.randint(vocab))
    elif kind == "two":
        t = np.where(rs.uniform(size=n) < 0.9, vocab - 1, 0)
    elif kind == "distinct":
        t = rs.permutation(vocab)[:n]
    else:
        t = rs.randint(0, vocab, n)
    return t.astype(np.int32)


def lookup(rt, pool, tokens, vocab, width, table_dtype, y_dtype, scale=1.0, pad=-1, table_stride=None, y_stride=None, shift=0, seed=0):
    rs = np.random.RandomState(seed)
    values = rounded(rs.normal(0, 1, (vocab, width)), table_dtype)
    table = pool.rows((vocab, width), table_dtype, values, table_stride, shift)
    y = pool.rows((len(tokens), width), y_dtype, None, y_stride, shift)
    t = pool.array(tokens if len(tokens) else np.zeros(1, np.int32))
    spec = rt.embedding_spec(len(tokens), vocab, width, t.ptr, table.ptr, y.ptr, DTYPES[table_dtype], DTYPES[y_dtype], scale, pad,
                             table.stride, y.stride)
    rt.embedding(spec)
    has = (tokens >= 0) & (tokens < vocab) & (tokens != pad)
    want = np.where(has[:, None], values[np.where(has, tokens, 0)].astype(f64) * f64(f32(scale)), 0.0)
    return y.get(), want


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("n,vocab,width", [(1, 7, 8), (1, 100, 2048), (5, 3, 1), (63, 50, 33), (1000, 777, 301), (4, 9, 4099), (129, 1000, 512),
                                           (2, 1, 5000)])
def test_lookup(hip_runtime, pair, n, vocab, width):
    rs = np.random.RandomState(n + width)
    tokens = rs.randint(0, vocab, n).astype(np.int32)
    with Pool(hip_runtime) as pool:
        got, want = lookup(hip_runtime, pool, tokens, vocab, width, pair[0], pair[1], scale=3.7)
    assert_within(got, want, np.abs(want) * (EPS + HALF[pair[1]]) * 1.01 + TINY[pair[1]])


@pytest.mark.parametrize("pair", PAIRS, ids="-".join)
@pytest.mark.parametrize("table_stride,y_stride,shift", [(264, 272, 0), (259, 257, 0), (256, 256, 1), (263, 256, 3)])
def test_lookup_of_strided_and_shifted_rows(hip_runtime, pair, table_stride, y_stride, shift):
    tokens = np.random.RandomState(3).randint(0, 90, 130).astype(np.int32)
    with Pool(hip_runtime) as pool:
        got, want = lookup(hip_runtime, pool, tokens, 90, 256, pair[0], pair[1], 1.0, -1, table_stride, y_stride, shift)
    assert_within(got, want, np.abs(want) * (EPS + HALF[pair[1]]) * 1.01 + TINY[pair[1]])


def test_lookup_of_padding_and_of_tokens_outside_the_table_gives_zeros(hip_runtime):
    tokens = np.array([0, 4, -1, 5, 6, 2 ** 31 - 1, -2 ** 31, 3, 0, 2], np.int32)
    with Pool(hip_runtime) as pool:
        got, want = lookup(hip_runtime, pool, tokens, 5, 40, "bf16", "bf16", pad=3)
    np.testing.assert_array_equal(got, want.astype(f32))
    assert not got[[2, 3, 4, 5, 6, 7]].any() and got[0].any()


def test_lookup_of_no_rows_writes_nothing(hip_runtime):
    with Pool(hip_runtime) as pool:
        got, want = lookup(hip_runtime, pool, np.zeros(0, np.int32), 5, 40, "f32", "f32")
    assert got.shape == (0, 40)


def test_lookup_in_a_table_longer_than_32_bit_offsets(hip_runtime):
    rt = hip_runtime
    vocab, width = 300000, 16384                     # 4.9e9 fp16 elements, 9.8 GB
    row = np.arange(width, dtype=np.float16)
    with Pool(rt) as pool:
        table = rt.malloc(vocab * width * 2)
        for v in (0, 131071, 131072, 262144, 299999):
            rt.memcpy_h2d(table + v * width * 2, row + np.float16(v % 7))
        tokens = pool.array(np.array([299999, 262144, 0, 131072, 131071], np.int32))
        y = pool.rows((5, width), "f16")
        rt.embedding(rt.embedding_spec(5, vocab, width, tokens.ptr, table, y.ptr, DTYPES["f16"]))
        got = y.get()
        rt.free(table)
    for i, v in enumerate((299999, 262144, 0, 131072, 131071)):
        np.testing.assert_array_equal(got[i], (row + np.float16(v % 7)).astype(f32))


def gradient(rt, pool, tokens, vocab, width, y_dtype, table_dtype, scale=1.0, pad=-1, accumulate=False, y_stride=None, table_stride=None,
             shift=0, seed=0, runs=1):
    rs = np.random.RandomState(seed)
    n = len(tokens)
    dy_values = rounded(rs.normal(0.1, 1, (n, width)), y_dtype)
    old = rounded(rs.normal(0, 1, (vocab, width)), table_dtype)
    dy = pool.rows((n, width), y_dtype, dy_values, y_stride, shift)
    t = pool.array(tokens if n else np.zeros(1, np.int32))
    got = []
    for _ in range(runs):
        # (without accumulate every row has to be written: the rows start as the canary's bytes)
        dtable = pool.rows((vocab, width), table_dtype, old if accumulate else None, table_stride, shift)
        spec = rt.embedding_grad_spec(n, vocab, width, t.ptr, dy.ptr, dtable.ptr, DTYPES[y_dtype], DTYPES[table_dtype], scale, pad,
                                      accumulate, dtable.stride, dy.stride)
        spec.workspace_bytes = rt.embedding_grad_workspace(spec)
        work = pool.bytes(spec.workspace_bytes)
        rt.memset32(work.ptr, 0xffffffff, spec.workspace_bytes // 4)          # nothing may be expected of it
        spec.workspace = work.ptr
        rt.embedding_grad(spec)
        got.append(dtable.get())
    has = (tokens >= 0) & (tokens < vocab) & (tokens != pad)
    total, size = np.zeros((vocab, width)), np.zeros((vocab, width))
    np.add.at(total, tokens[has], dy_values[has].astype(f64))
    np.add.at(size, tokens[has], np.abs(dy_values[has]).astype(f64))
    count = np.bincount(tokens[has], minlength=vocab)[:, None]
    s = f64(f32(scale))
    want = s * total
    bound = np.abs(s) * size * (count + 3) * EPS
    if accumulate:
        want = np.where(count > 0, want + old, old)
        bound = np.where(count > 0, bound + EPS * (np.abs(old) + np.abs(want)), 0.0)
    bound = bound + np.where(count > 0, (np.abs(want) + bound) * HALF[table_dtype] + TINY[table_dtype], 0.0)
    return got, want, bound


GRAD_PAIRS = [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")]        # rows, table


@pytest.mark.parametrize("accumulate", [False, True], ids=["written", "added"])
@pytest.mark.parametrize("pair", GRAD_PAIRS, ids="-".join)
@pytest.mark.parametrize("n,vocab,width,kind", [
    (1, 1, 1, "any"), (1, 5, 2048, "any"), (7, 3, 33, "any"), (64, 64, 64, "distinct"), (65, 1, 8, "one"), (777, 50, 301, "zipf"),
    (1999, 20011, 40, "zipf"), (4097, 63, 72, "two"), (16384, 64, 16, "zipf"), (16385, 65537, 16, "zipf"), (40000, 511, 24, "one"),
    (33000, 262145, 9, "any")])
def test_gradient(hip_runtime, pair, accumulate, n, vocab, width, kind):
    tokens = tokens_for(np.random.RandomState(n), n, vocab, kind)
    with Pool(hip_runtime) as pool:
        got, want, bound = gradient(hip_runtime, pool, tokens, vocab, width, pair[0], pair[1], 2.5, -1, accumulate, runs=2)
    np.testing.assert_array_equal(got[0], got[1])                 # the same bits from run to run
    assert_within(got[0], want, bound)


@pytest.mark.parametrize("pair", GRAD_PAIRS, ids="-".join)
@pytest.mark.parametrize("accumulate", [False, True], ids=["written", "added"])
@pytest.mark.parametrize("y_stride,table_stride,shift", [(136, 160, 0), (131, 129, 0), (128, 128, 1), (133, 128, 5)])
def test_gradient_of_strided_and_shifted_rows(hip_runtime, pair, accumulate, y_stride, table_stride, shift):
    tokens = tokens_for(np.random.RandomState(5), 600, 300, "zipf")
    with Pool(hip_runtime) as pool:
        got, want, bound = gradient(hip_runtime, pool, tokens, 300, 128, pair[0], pair[1], 1.0, -1, accumulate, y_stride, table_stride, shift)
    assert_within(got[0], want, bound)


@pytest.mark.parametrize("accumulate", [False, True], ids=["written", "added"])
@pytest.mark.parametrize("n", [10, 900, 17000])
def test_gradient_skips_padding_and_tokens_outside_the_table(hip_runtime, accumulate, n):
    rs = np.random.RandomState(n)
    tokens = rs.randint(-3, 20, n).astype(np.int32)
    tokens[rs.uniform(size=n) < 0.3] = 2 ** 31 - 1
    tokens[rs.uniform(size=n) < 0.1] = -2 ** 31
    with Pool(hip_runtime) as pool:
        got, want, bound = gradient(hip_runtime, pool, tokens, 17, 24, "bf16", "f32", 1.5, 4, accumulate)
        none = np.full(n, -1, np.int32)
        empty, zero, _ = gradient(hip_runtime, pool, none, 17, 24, "bf16", "f32", 1.5, 4, accumulate)
    assert_within(got[0], want, bound)
    np.testing.assert_array_equal(empty[0], zero.astype(f32))
    if not accumulate:
        assert not got[0][4].any()


def test_gradient_of_no_rows(hip_runtime):
    none = np.zeros(0, np.int32)
    with Pool(hip_runtime) as pool:
        got, want, _ = gradient(hip_runtime, pool, none, 11, 24, "f32", "f32")
        np.testing.assert_array_equal(got[0], want)
        got, want, _ = gradient(hip_runtime, pool, none, 11, 24, "f32", "f32", accumulate=True)
        np.testing.assert_array_equal(got[0], want)


def test_gradient_of_many_places_and_a_table_of_more_than_27_bits_of_tokens(hip_runtime):
    """Three and four digits of the tiled sort: a table of one column."""
    rt = hip_runtime
    rs = np.random.RandomState(8)
    n, vocab = 50000, (1 << 27) + 5
    tokens = rs.choice(rs.randint(0, vocab, 3000), n).astype(np.int32)
    values = rs.randint(-8, 9, (n, 1)).astype(f32)                       # whole numbers: any order adds up exactly
    with Pool(rt) as pool:
        dy, t = pool.rows((n, 1), "f32", values), pool.array(tokens)
        table = rt.empty((vocab,))
        spec = rt.embedding_grad_spec(n, vocab, 1, t.ptr, dy.ptr, table.ptr)
        spec.workspace_bytes = rt.embedding_grad_workspace(spec)
        work = pool.bytes(spec.workspace_bytes)
        spec.workspace = work.ptr
        rt.embedding_grad(spec)
        got = table.get()
        table.free()
    want = np.bincount(tokens, weights=values[:, 0].astype(f64), minlength=vocab)
    np.testing.assert_array_equal(got, want.astype(f32))


@pytest.mark.parametrize("n,vocab,kind", [(262145, 300, "zipf"), (600001, 70001, "zipf"), (400000, 70001, "one"), (524289, 2000000, "any")])
def test_gradient_of_more_tiles_than_a_tile_adds_up(hip_runtime, n, vocab, kind):
    """One, two and three digits with the counts of all tiles added by a launch of its own."""
    rt, rs = hip_runtime, np.random.RandomState(n)
    tokens = tokens_for(rs, n, vocab, kind)
    values = rs.randint(-8, 9, (n, 2)).astype(f32)                       # whole numbers: any order adds up exactly
    want = np.stack([np.bincount(tokens, weights=values[:, i].astype(f64), minlength=vocab) for i in (0, 1)], 1)
    with Pool(rt) as pool:
        dy, t, table = pool.rows((n, 2), "f32", values), pool.array(tokens), pool.rows((vocab, 2), "f32")
        spec = rt.embedding_grad_spec(n, vocab, 2, t.ptr, dy.ptr, table.ptr)
        spec.workspace_bytes = rt.embedding_grad_workspace(spec)
        work = pool.bytes(spec.workspace_bytes)
        rt.memset32(work.ptr, 0xffffffff, spec.workspace_bytes // 4)
        spec.workspace = work.ptr
        rt.embedding_grad(spec)
        got = table.get()
    np.testing.assert_array_equal(got, want.astype(f32))


def test_recorded_calls_replay_with_new_tokens(hip_runtime):
    """Lookup and gradient in one graph, replayed between eager calls that share the workspace."""
    rt = hip_runtime
    rs = np.random.RandomState(2)
    n, vocab, width = 900, 333, 64
    values = rounded(rs.normal(0, 1, (vocab, width)), "f32")
    with Pool(rt) as pool:
        table, y = pool.rows((vocab, width), "f32", values), pool.rows((n, width), "f32")
        dtable = pool.rows((vocab, width), "f32")
        t = pool.array(np.zeros(n, np.int32))
        fwd = rt.embedding_spec(n, vocab, width, t.ptr, table.ptr, y.ptr, scale=2.0)
        bwd = rt.embedding_grad_spec(n, vocab, width, t.ptr, y.ptr, dtable.ptr, scale=0.5)
        bwd.workspace_bytes = rt.embedding_grad_workspace(bwd)
        work = pool.bytes(bwd.workspace_bytes)
        bwd.workspace = work.ptr
        rt.graph_begin()
        rt.embedding(fwd)
        rt.embedding_grad(bwd)
        graph = rt.graph_end()
        try:
            for k in range(4):
                tokens = tokens_for(rs, n, vocab, ("zipf", "any", "one", "two")[k])
                t.set(tokens)
                rt.graph_launch(graph)
                replayed = y.get(), dtable.get()
                rt.memset32(work.ptr, 0x7fc00000, bwd.workspace_bytes // 4)
                rt.embedding(fwd)
                rt.embedding_grad(bwd)
                np.testing.assert_array_equal(replayed[0], y.get())
                np.testing.assert_array_equal(replayed[1], dtable.get())
                np.testing.assert_array_equal(replayed[0], 2 * values[tokens])
        finally:
            rt.graph_free(graph)
