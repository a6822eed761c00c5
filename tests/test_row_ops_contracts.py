"""What the header says of the operators over rows and parameters beyond single arguments: several operands that share
memory, calls over nothing, counters, without a device where that is possible."""
import ctypes

import numpy as np
import pytest

from ngraph_hip.runtime import HipLibraryError, load_library, row_ops
from ngraph_hip.runtime.hiplib import NGH_ABI_VERSION, _check
from row_helpers import DTYPES, Pool


class Calls(row_ops.OperatorCalls):
    """The spec builders without a device."""
    abi_version = NGH_ABI_VERSION

    def __init__(self):
        self.lib, self.ctx = load_library(), None

    def _check(self, rc):
        _check(self.lib, rc)


calls = Calls()
AT = {k: 0x1000000 * (i + 1) for i, k in enumerate(("x", "b", "h", "y", "gain", "post_gain", "dy", "dh", "dx", "db", "dgain", "dpost_gain"))}


def norm(gradient, rows=12, **same):
    """Validates a spec in which the operands named are at the addresses of others."""
    names = ("b", "h", "gain", "post_gain") + (("dy", "dh", "dx", "db", "dgain", "dpost_gain") if gradient else ("x", "y"))
    at = {n: AT[same.get(n, n)] for n in names}
    s = calls.block_norm_spec(rows, 64, post_norm=True, **at)
    calls._check(calls.lib.ngh_validate_block_norm(ctypes.byref(s), 1 if gradient else 0))


def test_the_stream_and_its_gradient_may_be_updated_in_place():
    for rows in (1, 12):
        norm(False, rows, h="x")
        norm(True, rows, dx="dh")


@pytest.mark.parametrize("rows", [1, 12])
@pytest.mark.parametrize("gradient,same", [
    (False, dict(h="x", y="x")), (False, dict(h="x", b="x")), (False, dict(h="x", gain="x")), (False, dict(h="x", post_gain="x")), (False, dict(y="h")),
    (True, dict(dx="dh", db="dh")), (True, dict(dx="dh", dgain="dh")), (True, dict(dx="dh", dpost_gain="dh")), (True, dict(dx="dh", post_gain="dh")),
    (True, dict(dx="dh", gain="dh")), (True, dict(dx="dh", b="dh"))])
def test_nothing_else_may_share_what_is_updated_in_place(gradient, same, rows):
    with pytest.raises(HipLibraryError) as e:
        norm(gradient, rows, **same)
    assert e.value.code == -1 and "overlaps" in str(e.value)


@pytest.mark.gpu
@pytest.mark.parametrize("types", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")], ids="-".join)
@pytest.mark.parametrize("width,gate_rows", [(1, 0), (64, 7), (4096, 0), (16384, 3)])
def test_gradients_of_no_rows_are_zeros(hip_runtime, width, gate_rows, types):
    """(an empty batch: with the workspace that the query asks for)"""
    rt = hip_runtime
    with Pool(rt) as pool:
        rows = pool.rows((1, width), types[0], np.zeros((1, width)))
        outs = {n: pool.rows((1, width), types[1]) for n in ("dgain", "dbias", "dpost_gain", "dpost_bias")}
        untouched = {n: pool.rows((1, width), t, np.full((1, width), 3.0)) for n, t in (("dx", types[0]), ("db", types[0]), ("dgate", types[1]))}
        gate = {"gate": rows.ptr, "dgate": untouched["dgate"].ptr, "gate_rows": gate_rows} if gate_rows else {}
        spec = rt.block_norm_spec(0, width, "layer", DTYPES[types[0]], DTYPES[types[1]], True, h=rows.ptr, b=rows.ptr, dy=rows.ptr,
                                  dx=untouched["dx"].ptr, db=untouched["db"].ptr, **dict({n: t.ptr for n, t in outs.items()}, **gate))
        spec.workspace_bytes = rt.block_norm_grad_workspace(spec)
        spec.workspace = pool.bytes(spec.workspace_bytes).ptr
        rt.block_norm_grad(spec)
        for n, t in outs.items():
            assert not t.get().any(), n
        for n, t in untouched.items():
            assert (t.get() == 3.0).all(), n


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[], [0, 0]])
def test_an_update_of_nothing_counts(hip_runtime, lengths):
    rt = hip_runtime
    with Pool(rt) as pool:
        count, lr = pool.array(np.array([4], np.int32)), pool.array(np.array([1e-3], np.float32))
        plan = rt.adamw_plan([dict(n=n) for n in lengths])
        for k in range(3):
            rt.adamw_step(plan, dev_step=count.ptr, dev_lr=lr.ptr)
            assert count.get()[0] == 5 + k
        rt.graph_begin()
        rt.adamw_step(plan, dev_step=count.ptr)
        graph = rt.graph_end()
        for k in range(2):
            rt.graph_launch(graph)
            assert count.get()[0] == 8 + k
        rt.graph_free(graph)
        rt.adamw_plan_free(plan)
