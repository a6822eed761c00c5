"""What the operators over rows and parameters refuse, without a device (ngh_validate_*)."""
import ctypes

import pytest

from ngraph_hip.runtime import NGH_BF16, NGH_F16, NGH_F32, NGH_FLEX16, FusedSpecBuilder, HipLibraryError, load_library, row_ops
from ngraph_hip.runtime.hiplib import NGH_ABI_VERSION, _check


class Calls(row_ops.OperatorCalls):
    """The spec builders without a device."""
    abi_version = NGH_ABI_VERSION

    def __init__(self):
        self.lib, self.ctx = load_library(), None

    def _check(self, rc):
        _check(self.lib, rc)


calls = Calls()


def refused(fn, code, words):
    with pytest.raises(HipLibraryError) as e:
        fn()
    assert e.value.code == code and words in str(e.value), str(e.value)


def embedding(gradient=False, **change):
    s = calls.embedding_spec(10, 100, 64, 0x1000, 0x100000, 0x200000)
    for k, v in change.items():
        setattr(s, k, v)
    calls._check(calls.lib.ngh_validate_embedding(ctypes.byref(s), 1 if gradient else 0))


def test_embedding_takes_what_it_documents():
    embedding()
    embedding(True)
    embedding(table_dtype=NGH_BF16, y_dtype=NGH_BF16)
    embedding(y_dtype=NGH_F16)
    embedding(rows=0, y=None, tokens=None)
    embedding(vocab=0, table=None)
    embedding(rows=1, y_stride=0)


@pytest.mark.parametrize("gradient", [False, True])
@pytest.mark.parametrize("code,words,change", [
    (-1, "abi_version", dict(abi_version=6)), (-1, "dtypes", dict(table_dtype=NGH_FLEX16)), (-1, "dtypes", dict(y_dtype=2)),
    (-4, "dtype", dict(table_dtype=NGH_BF16)), (-4, "dtype", dict(table_dtype=NGH_F16, y_dtype=NGH_BF16)),
    (-1, "rows", dict(rows=-1)), (-1, "vocab", dict(vocab=-5)), (-1, "width", dict(width=-5)), (-4, "extent", dict(vocab=1 << 31)),
    (-4, "extent", dict(rows=1 << 31)), (-1, "y_stride", dict(y_stride=63)), (-1, "table_stride", dict(table_stride=10)),
    (-4, "stride", dict(table_stride=1 << 40)), (-1, "NULL", dict(tokens=None)), (-1, "NULL", dict(y=None)), (-1, "NULL", dict(table=None)),
    (-1, "misaligned", dict(tokens=0x1002)), (-1, "misaligned", dict(y=0x200002)), (-1, "misaligned", dict(table=0x100001)),
    (-1, "overlaps", dict(y=0x100400))])
def test_embedding_refusals(gradient, code, words, change):
    refused(lambda: embedding(gradient, **change), code, words)


def test_calls_without_a_context_are_refused():
    s = calls.embedding_spec(10, 100, 64, 0x1000, 0x100000, 0x200000)
    for fn in (calls.embedding, calls.embedding_grad):
        refused(lambda: fn(s), -1, "ctx is NULL")
    n = calls.block_norm_spec(4, 64, x=0x1000, y=0x10000)
    for fn in (calls.block_norm, calls.block_norm_grad):
        refused(lambda: fn(n), -1, "ctx is NULL")
    refused(lambda: calls.adamw_plan([]), -1, "ctx is NULL")
    refused(lambda: calls.adamw_decode(0x1000, 0x2000, 0x3000, 4), -1, "ctx is NULL")
    refused(lambda: calls.adamw_step(row_ops.AdamWPlan(None, 0, 32), 1), -1, "ctx is NULL")


def test_gate_rows_beyond_any_number_of_rows_are_refused():
    """(of no rows every number of them is a whole share)"""
    refused(lambda: norm(gate_rows=1 << 32, rows=0), -1, "gate_rows")
    refused(lambda: norm(True, gate_rows=1 << 32, rows=0), -1, "gate_rows")
    norm(True, gate_rows=7, rows=0)


def test_spans_beyond_64_bits_are_seen_to_overlap():
    far = dict(rows=(1 << 30) + 12, h_stride=(1 << 40) - 4, gate_rows=4)
    refused(lambda: norm(**far), -1, "overlaps")


def test_the_gradients_workspace_grows_with_what_it_holds():
    small = calls.embedding_grad_workspace(calls.embedding_grad_spec(10, 100, 64, 1, 2, 3))
    large = calls.embedding_grad_workspace(calls.embedding_grad_spec(100000, 100, 64, 1, 2, 3))
    assert 0 < small < large
    refused(lambda: calls.embedding_grad_workspace(calls.embedding_grad_spec(-1, 100, 64, 1, 2, 3)), -1, "rows")


ADDRESS = {k: 0x1000000 * (i + 1) for i, k in enumerate(
    ("x", "b", "h", "y", "gain", "bias", "post_gain", "post_bias", "gate", "dy", "dh", "dx", "db", "dgain", "dbias", "dpost_gain",
     "dpost_bias", "dgate"))}
FORWARD = ("x", "b", "h", "y", "gain", "bias", "post_gain", "post_bias", "gate")
BACKWARD = ("b", "h", "gain", "post_gain", "post_bias", "gate", "dy", "dh", "dx", "db", "dgain", "dbias", "dpost_gain", "dpost_bias", "dgate")


def norm(gradient=False, drop=(), **change):
    names = [n for n in (BACKWARD if gradient else FORWARD) if n not in drop]
    build = {k: change.pop(k) for k in ("kind",) if k in change}
    s = calls.block_norm_spec(12, 64, post_norm=True, gate_rows=4, **dict(build, **{n: ADDRESS[n] for n in names}))
    for k, v in change.items():
        setattr(s, k, v)
    calls._check(calls.lib.ngh_validate_block_norm(ctypes.byref(s), 1 if gradient else 0))


def test_block_norm_takes_what_it_documents():
    norm()
    norm(True)
    norm(dtype=NGH_BF16, param_dtype=NGH_BF16)
    norm(True, dtype=NGH_F16)
    norm(drop=("h",))
    norm(drop=("y", "gain", "bias"))
    norm(drop=("b", "post_gain", "post_bias", "gate"), post_norm=0, gate_rows=0)
    norm(h=ADDRESS["x"])
    norm(True, dx=ADDRESS["dh"])
    norm(True, drop=("dh", "dgain", "dbias", "dpost_gain", "dpost_bias", "dgate"))
    norm(True, drop=("dy", "gain", "dgain", "dbias", "h"))
    norm(True, drop=("dx",))
    norm(rows=0, drop=("x", "h", "y", "gain", "bias"))


@pytest.mark.parametrize("gradient", [False, True])
@pytest.mark.parametrize("code,words,change", [
    (-1, "abi_version", dict(abi_version=0)), (-1, "kind", dict()), (-1, "dtype", dict(dtype=NGH_FLEX16)),
    (-1, "dtype", dict(dtype=NGH_BF16, param_dtype=NGH_F16)), (-1, "dtype", dict(dtype=NGH_F32, param_dtype=NGH_BF16)),
    (-1, "rows", dict(rows=-4)), (-1, "width", dict(width=0)), (-4, "elements", dict(width=16385)), (-4, "rows", dict(rows=1 << 31)),
    (-1, "eps", dict(eps=-1.0)), (-1, "eps", dict(eps=float("nan"))), (-1, "residual_scale", dict(residual_scale=float("inf"))),
    (-1, "gate_rows", dict(gate_rows=5)), (-1, "gate_rows", dict(gate_rows=0)), (-1, "without a gate", dict(gate=None, dgate=None)),
    (-1, "without post_norm", dict(post_norm=0)), (-1, "aligned", dict(b=ADDRESS["b"] + 2)), (-1, "stride", dict(h_stride=63)),
    (-1, "stride", dict(gate_stride=1)), (-4, "stride", dict(b_stride=1 << 40))])
def test_block_norm_refusals(gradient, code, words, change):
    if words == "kind":
        with pytest.raises(ValueError):
            norm(gradient, kind="batch")
        change = dict(kind=2)
        s = calls.block_norm_spec(2, 8, x=0x1000, y=0x2000)
        s.kind = 2
        refused(lambda: calls._check(calls.lib.ngh_validate_block_norm(ctypes.byref(s), 0)), code, words)
        return
    refused(lambda: norm(gradient, **change), code, words)


@pytest.mark.parametrize("words,change,drop", [
    ("x is NULL", dict(x=None), ()), ("neither h nor y", dict(), ("h", "y", "gain", "bias")), ("without y", dict(y=None), ()),
    ("no block output", dict(), ("b",)), ("overlaps", dict(y=ADDRESS["x"]), ()), ("overlaps", dict(h=ADDRESS["b"]), ()),
    ("overlaps", dict(h=ADDRESS["x"], h_stride=65), ()), ("overlaps", dict(h=ADDRESS["y"] + 256), ()),
    ("overlaps", dict(gain=ADDRESS["y"]), ())])
def test_block_norm_forward_refusals(words, change, drop):
    refused(lambda: norm(False, drop, **change), -1, words)


@pytest.mark.parametrize("words,change,drop", [
    ("neither dy nor dh", dict(), ("dy", "dh")), ("dy without h", dict(), ("h",)), ("b and db", dict(), ("db",)),
    ("b and db", dict(), ("b",)), ("neither dx nor db", dict(post_norm=0, gate_rows=0), ("b", "dx", "db", "gate", "dgate", "post_gain",
     "post_bias", "dpost_gain", "dpost_bias")), ("without dy", dict(), ("dy",)), ("without a gate", dict(gate_rows=0), ("gate",)),
    ("overlaps", dict(dx=ADDRESS["dy"]), ()), ("overlaps", dict(db=ADDRESS["dx"]), ()), ("overlaps", dict(db=ADDRESS["h"]), ()),
    ("overlaps", dict(dgain=ADDRESS["gain"]), ()), ("overlaps", dict(workspace=ADDRESS["db"], workspace_bytes=16), ())])
def test_block_norm_gradient_refusals(words, change, drop):
    refused(lambda: norm(True, drop, **change), -1, words)


def adamw(rows=None, param_dtype=NGH_F32, grad_dtype=NGH_F32, copy_dtype=-1, bits=32, n_tensors=None):
    rows = [tensor(0)] if rows is None else rows
    calls._check(calls.lib.ngh_validate_adamw(row_ops.adamw_tensors(rows), len(rows) if n_tensors is None else n_tensors, param_dtype,
                                              grad_dtype, copy_dtype, bits))


def tensor(k, n=1000, **change):
    at = 0x10000000 * (k + 1)
    t = dict(param=at, grad=at + 0x1000000, m=at + 0x2000000, v=at + 0x3000000, n=n, m_scale=at + 0x4000000, v_scale=at + 0x5000000)
    t.update(change)
    return t


def test_adamw_takes_what_it_documents():
    adamw()
    adamw([])
    adamw([tensor(0), tensor(1, 0, param=None, grad=None, m=None, v=None), tensor(2, 1)], NGH_BF16, NGH_F16, bits=8)
    adamw([tensor(0, copy=0x900)], copy_dtype=NGH_BF16)
    adamw([tensor(0), tensor(1, grad=tensor(0)["grad"])])                # two may share a gradient


@pytest.mark.parametrize("code,words,kw", [
    (-1, "bits", dict(bits=16)), (-1, "dtypes", dict(param_dtype=NGH_FLEX16)), (-1, "dtypes", dict(grad_dtype=2)),
    (-1, "dtypes", dict(copy_dtype=5)), (-1, "tensors", dict(n_tensors=-1)), (-1, "length", dict(rows=[tensor(0, -1)])),
    (-4, "too long", dict(rows=[tensor(0, 1 << 42)])), (-1, "weight_decay", dict(rows=[tensor(0, weight_decay=float("nan"))])),
    (-1, "copy", dict(rows=[tensor(0, copy=0x900)])), (-1, "NULL", dict(rows=[tensor(0, m=None)])),
    (-1, "NULL", dict(rows=[tensor(0, m_scale=None)], bits=8)), (-1, "misaligned", dict(rows=[tensor(0, param=0x1001)])),
    (-1, "misaligned", dict(rows=[tensor(0, v=0x1002)])), (-1, "share memory", dict(rows=[tensor(0), tensor(0)])),
    (-1, "share memory", dict(rows=[tensor(0), tensor(1, param=0x10000000 + 996 * 4)])),
    (-1, "share memory", dict(rows=[tensor(0), tensor(1, grad=0x10000000)])),
    (-1, "share memory", dict(rows=[tensor(0, 1000, grad=0x12000000 - 8)]))])
def test_adamw_refusals(code, words, kw):
    refused(lambda: adamw(**kw), code, words)


def test_adamw_rows_with_unknown_fields_are_refused():
    with pytest.raises(ValueError):
        row_ops.adamw_tensors([dict(params=1)])
    with pytest.raises(ValueError):
        calls.block_norm_spec(2, 8, gains=1)


def test_fused_specs_refuse_bf16():
    sb = FusedSpecBuilder([16])
    a, b = sb.tensor(0x1000, [1], NGH_BF16), sb.tensor(0x2000, [1], NGH_F32)
    sb.store(b, sb.load(a))
    refused(lambda: _check(calls.lib, calls.lib.ngh_validate_fused(ctypes.byref(sb.build()))), -1, "dtype")
