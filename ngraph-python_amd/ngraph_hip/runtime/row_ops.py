"""ctypes side of the operators over rows and parameters (include/ngraph_hip.h): embedding lookup and
gradient, the norms around a block, AdamW over many tensors.  `OperatorCalls` is what `HipRuntime`
mixes in; specs are filled once and used for every call, as the fused specs are.  The reference has
the lookup table (op_graph/lookuptable.py:55-115) and composes the others of elementwise kernels
(frontends/neon/layer.py:1242-1257, optimizer.py:446-470).
"""
from __future__ import division
import ctypes

_vp, _i32, _i64, _f32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float

NGH_NORM_RMS, NGH_NORM_LAYER = 0, 1
NGH_BLOCK_NORM_MAX_WIDTH = 16384
NGH_ADAMW_BLOCK = 256
NORM_KINDS = {"rms": NGH_NORM_RMS, "layer": NGH_NORM_LAYER}


class ngh_embedding_spec(ctypes.Structure):
    _fields_ = [("abi_version", _i32), ("table_dtype", _i32), ("y_dtype", _i32), ("pad_idx", _i32),
                ("rows", _i64), ("vocab", _i64), ("width", _i64),
                ("tokens", _vp), ("table", _vp), ("table_stride", _i64), ("y", _vp), ("y_stride", _i64),
                ("scale", _f32), ("accumulate", _i32), ("workspace", _vp), ("workspace_bytes", ctypes.c_size_t)]


class ngh_block_norm_spec(ctypes.Structure):
    _fields_ = [("abi_version", _i32), ("kind", _i32), ("dtype", _i32), ("param_dtype", _i32), ("post_norm", _i32),
                ("eps", _f32), ("residual_scale", _f32), ("reserved", _i32),
                ("rows", _i64), ("width", _i64), ("gate_rows", _i64),
                ("x", _vp), ("b", _vp), ("x_stride", _i64), ("b_stride", _i64),
                ("gain", _vp), ("bias", _vp), ("post_gain", _vp), ("post_bias", _vp), ("gate", _vp), ("gate_stride", _i64),
                ("h", _vp), ("y", _vp), ("h_stride", _i64), ("y_stride", _i64),
                ("dy", _vp), ("dh", _vp), ("dy_stride", _i64), ("dh_stride", _i64),
                ("dx", _vp), ("db", _vp), ("dx_stride", _i64), ("db_stride", _i64),
                ("dgain", _vp), ("dbias", _vp), ("dpost_gain", _vp), ("dpost_bias", _vp), ("dgate", _vp), ("dgate_stride", _i64),
                ("workspace", _vp), ("workspace_bytes", ctypes.c_size_t)]


class ngh_adamw_tensor(ctypes.Structure):
    _fields_ = [("param", _vp), ("grad", _vp), ("m", _vp), ("v", _vp), ("m_scale", _vp), ("v_scale", _vp), ("copy", _vp),
                ("n", _i64), ("weight_decay", _f32), ("reserved", _i32)]


class ngh_adamw_hyper(ctypes.Structure):
    _fields_ = [("lr", ctypes.c_double), ("beta1", ctypes.c_double), ("beta2", ctypes.c_double), ("eps", ctypes.c_double),
                ("grad_scale", _f32), ("step", _i32), ("dev_step", _vp), ("dev_lr", _vp), ("dev_grad_scale", _vp)]


_emb, _norm, _tensors = (ctypes.POINTER(t) for t in (ngh_embedding_spec, ngh_block_norm_spec, ngh_adamw_tensor))
SYMBOLS = {
    "ngh_validate_embedding": [_emb, _i32],
    "ngh_embedding": [_vp, _emb],
    "ngh_embedding_grad": [_vp, _emb],
    "ngh_embedding_grad_workspace": [_emb, ctypes.POINTER(ctypes.c_size_t)],
    "ngh_validate_block_norm": [_norm, _i32],
    "ngh_block_norm": [_vp, _norm],
    "ngh_block_norm_grad": [_vp, _norm],
    "ngh_block_norm_grad_workspace": [_norm, ctypes.POINTER(ctypes.c_size_t)],
    "ngh_validate_adamw": [_tensors, _i32, _i32, _i32, _i32, _i32],
    "ngh_adamw_plan_create": [_vp, _tensors, _i32, _i32, _i32, _i32, _i32, ctypes.POINTER(_vp)],
    "ngh_adamw_step": [_vp, _vp, ctypes.POINTER(ngh_adamw_hyper)],
    "ngh_adamw_plan_free": [_vp, _vp],
    "ngh_adamw_decode": [_vp, _vp, _vp, _vp, _i64, _i32],
    "ngh_adamw_encode": [_vp, _vp, _vp, _vp, _i64, _i32],
}


def adamw_tensors(rows):
    """An array of ngh_adamw_tensor from dicts with param, grad, m, v, n and, where they apply, m_scale,
    v_scale, copy (device addresses) and weight_decay."""
    known = set(name for name, _ in ngh_adamw_tensor._fields_)
    out = (ngh_adamw_tensor * max(len(rows), 1))()
    for t, row in zip(out, rows):
        unknown = set(row) - known
        if unknown:
            raise ValueError("adamw tensor: unknown fields %s" % ", ".join(sorted(unknown)))
        for k, v in row.items():
            setattr(t, k, v)
    return out


class AdamWPlan(object):
    """Handle of ngh_adamw_plan_create; freed by `adamw_plan_free` or with its runtime."""

    def __init__(self, handle, n_tensors, state_bits):
        self.handle, self.n_tensors, self.state_bits = handle, n_tensors, state_bits


class DryRunOperatorCalls(object):
    """The same calls where no device exists: specs are checked by the library and recorded."""

    def embedding(self, spec):
        self._check(self.lib.ngh_validate_embedding(ctypes.byref(spec), 0))
        self.launched.append(spec)

    def embedding_grad(self, spec):
        self._check(self.lib.ngh_validate_embedding(ctypes.byref(spec), 1))
        self.launched.append(spec)

    def block_norm(self, spec):
        self._check(self.lib.ngh_validate_block_norm(ctypes.byref(spec), 0))
        self.launched.append(spec)

    def block_norm_grad(self, spec):
        self._check(self.lib.ngh_validate_block_norm(ctypes.byref(spec), 1))
        self.launched.append(spec)

    def adamw_plan(self, tensors, param_dtype=0, grad_dtype=0, copy_dtype=-1, state_bits=32):
        self._check(self.lib.ngh_validate_adamw(adamw_tensors(tensors), len(tensors), param_dtype, grad_dtype, copy_dtype, state_bits))
        return AdamWPlan(None, len(tensors), state_bits)

    def adamw_step(self, plan, **hyper):
        self.launched.append(("adamw", plan, hyper))

    def adamw_plan_free(self, plan):
        pass


class OperatorCalls(object):
    """The calls of these operators on a runtime: needs self.lib, self.ctx and self._check(rc)."""

    abi_version = None           # set by the class that mixes this in

    # -- embedding ---------------------------------------------------------
    def embedding_spec(self, rows, vocab, width, tokens, table, y, table_dtype=0, y_dtype=None, scale=1.0, pad_idx=-1,
                       table_stride=None, y_stride=None):
        """The spec of y[n, :] = scale * table[tokens[n], :]; strides default to the width."""
        if not -2 ** 31 <= pad_idx < 2 ** 31:
            raise ValueError("embedding: pad_idx %r is no int32" % (pad_idx,))
        s = ngh_embedding_spec()
        s.abi_version = self.abi_version
        s.rows, s.vocab, s.width = int(rows), int(vocab), int(width)
        s.tokens, s.table, s.y = tokens, table, y
        s.table_dtype, s.y_dtype = table_dtype, table_dtype if y_dtype is None else y_dtype
        s.table_stride = width if table_stride is None else table_stride
        s.y_stride = width if y_stride is None else y_stride
        s.scale, s.pad_idx = scale, pad_idx
        return s

    def embedding_grad_spec(self, rows, vocab, width, tokens, dy, dtable, y_dtype=0, table_dtype=None, scale=1.0, pad_idx=-1,
                            accumulate=False, table_stride=None, y_stride=None, workspace=None, workspace_bytes=0):
        """The spec of dtable[v, :] (+)= scale * sum of dy[n, :] over tokens[n] == v."""
        s = self.embedding_spec(rows, vocab, width, tokens, dtable, dy, y_dtype if table_dtype is None else table_dtype, y_dtype,
                                scale, pad_idx, table_stride, y_stride)
        s.accumulate = 1 if accumulate else 0
        s.workspace, s.workspace_bytes = workspace, int(workspace_bytes)
        return s

    def embedding(self, spec):
        rc = self.lib.ngh_embedding(self.ctx, spec)
        if rc:
            self._check(rc)

    def embedding_grad(self, spec):
        rc = self.lib.ngh_embedding_grad(self.ctx, spec)
        if rc:
            self._check(rc)

    def embedding_grad_workspace(self, spec):
        """Bytes of device memory embedding_grad(spec) works in."""
        n = ctypes.c_size_t()
        self._check(self.lib.ngh_embedding_grad_workspace(ctypes.byref(spec), ctypes.byref(n)))
        return n.value

    # -- block norm ----------------------------------------------------------
    _NORM_VIEWS = ("x", "b", "h", "y", "dy", "dh", "dx", "db", "gate", "dgate")

    def block_norm_spec(self, rows, width, kind="rms", dtype=0, param_dtype=None, post_norm=False, gate_rows=0, residual_scale=1.0,
                        eps=1e-5, **operands):
        """The spec of ngh_block_norm / ngh_block_norm_grad; `operands`: device addresses by field name, strides as
        x_stride, ... (default: the width) and workspace / workspace_bytes."""
        s = ngh_block_norm_spec()
        s.abi_version = self.abi_version
        if kind not in NORM_KINDS:
            raise ValueError("norm kind %r (rms or layer)" % (kind,))
        s.kind = NORM_KINDS[kind]
        s.dtype, s.param_dtype = dtype, dtype if param_dtype is None else param_dtype
        s.post_norm, s.gate_rows = 1 if post_norm else 0, int(gate_rows)
        s.eps, s.residual_scale = eps, residual_scale
        s.rows, s.width = int(rows), int(width)
        for name in self._NORM_VIEWS:
            setattr(s, name + "_stride", int(width))
        known = set(name for name, _ in ngh_block_norm_spec._fields_)
        for k, v in operands.items():
            if k not in known:
                raise ValueError("block norm has no operand %r" % (k,))
            setattr(s, k, v)
        return s

    def block_norm(self, spec):
        rc = self.lib.ngh_block_norm(self.ctx, spec)
        if rc:
            self._check(rc)

    def block_norm_grad(self, spec):
        rc = self.lib.ngh_block_norm_grad(self.ctx, spec)
        if rc:
            self._check(rc)

    def block_norm_grad_workspace(self, spec):
        """Bytes of device memory block_norm_grad(spec) works in."""
        n = ctypes.c_size_t()
        self._check(self.lib.ngh_block_norm_grad_workspace(ctypes.byref(spec), ctypes.byref(n)))
        return n.value

    # -- AdamW -----------------------------------------------------------------
    def adamw_plan(self, tensors, param_dtype=0, grad_dtype=0, copy_dtype=-1, state_bits=32):
        """A plan for the tensors (dicts, see adamw_tensors)."""
        handle = _vp()
        self._check(self.lib.ngh_adamw_plan_create(self.ctx, adamw_tensors(tensors), len(tensors), param_dtype, grad_dtype,
                                                   copy_dtype, state_bits, ctypes.byref(handle)))
        plan = AdamWPlan(handle, len(tensors), state_bits)
        self._adamw_plans.append(plan)
        return plan

    def adamw_step(self, plan, step=0, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, grad_scale=1.0, dev_step=None, dev_lr=None,
                   dev_grad_scale=None):
        """One update of every tensor of the plan; `step` counts from 1 (or dev_step: an int32 on the device)."""
        if not -2 ** 31 <= int(step) < 2 ** 31:
            raise ValueError("adamw: step %r is no int32" % (step,))
        h = ngh_adamw_hyper(lr, beta1, beta2, eps, grad_scale, int(step), dev_step, dev_lr, dev_grad_scale)
        self._check(self.lib.ngh_adamw_step(self.ctx, plan.handle, ctypes.byref(h)))

    def adamw_plan_free(self, plan):
        self._check(self.lib.ngh_adamw_plan_free(self.ctx, plan.handle))
        plan.handle = None
        if plan in self._adamw_plans:
            self._adamw_plans.remove(plan)

    def adamw_decode(self, out, codes, scales, n, second=False):
        """n first (second) moments held in 8 bits as fp32."""
        self._check(self.lib.ngh_adamw_decode(self.ctx, out, codes, scales, int(n), 1 if second else 0))

    def adamw_encode(self, codes, scales, values, n, second=False):
        self._check(self.lib.ngh_adamw_encode(self.ctx, codes, scales, values, int(n), 1 if second else 0))
