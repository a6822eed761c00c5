"""The operators over rows and parameters as graph ops: embedding lookup with scaling and its gradient
by sorted tokens, the norms around a block with its gate and residual, AdamW over many variables; and
the kernels that run them through the C ABI (`ngh_embedding`, `ngh_block_norm`, `ngh_adamw_step` and
their gradients).

The reference has the lookup table with its own gradient kernel (op_graph/lookuptable.py:55-160) and
composes norms and optimisers of elementwise ops (frontends/neon/layer.py:1242-1257,
optimizer.py:446-470); those compositions stay as they are, these ops stand beside them.

An op here has one tensor as its result like any other; what its kernel writes besides (the stream
after a block, the gradients of gains) are `RowResultOp`s that depend on it: their buffers are
filled by that kernel, and one that nothing uses is not computed.

The kernels take an operand as an address and at most one stride.  What an operand's description is
shows only behind the graph passes, which turn 1 * x, x + 0 and folded constants into views: an
operand that they may replace stands behind a `RowLayoutOp`, which `RowLayoutPass`, the last pass,
resolves to the operand itself or to a copy of it.  Every kernel checks what it is bound to.
"""
from __future__ import division

import numpy as np

from ngraph_hip.op_graph import op_graph as og
from ngraph_hip.transformers.hipdevice import _td
from ngraph_hip.transformers.hiplowering import HipKernel, og_unsupported
from ngraph_hip.transformers.passes.passes import PeepholeGraphPass

F32, F16, I32 = np.dtype(np.float32), np.dtype(np.float16), np.dtype(np.int32)
STATE_BLOCK = 256                       # elements that share a scale in 8-bit optimiser states


# ------------------------------------------------------------------------------------- layouts
def _merged(td, axes):
    """(length, stride) of `axes` of the description walked as one axis; None if they do not."""
    dims = [(a.length, td.full_strides[td.axes.index(a)]) for a in axes if a.length != 1]
    for (_, s0), (n1, s1) in zip(dims[:-1], dims[1:]):
        if s0 != s1 * n1:
            return None
    n = int(np.prod([n for n, _ in dims], dtype=np.int64)) if dims else 1
    return n, (dims[-1][1] if dims else 0)


def rows_of(td, width_axis):
    """(rows, width, row stride) of a tensor whose last axis is width_axis, when the elements of a row are
    consecutive and the rows evenly spaced without overlap; None otherwise."""
    if len(td.axes) == 0 or td.axes[len(td.axes) - 1] != width_axis:
        return None
    stride = td.full_strides[len(td.axes) - 1]
    if width_axis.length != 1 and stride != 1:
        return None
    merged = _merged(td, list(td.axes)[:-1])
    if merged is None:
        return None
    rows, row_stride = merged
    if rows > 1 and row_stride < width_axis.length:
        return None
    return rows, width_axis.length, row_stride if rows > 1 else width_axis.length


def _fits(td, dtype, width_axis):
    """Whether a row kernel can take a tensor of this description as `dtype` operand: rows along width_axis, or
    with None elements in C order."""
    return td.dtype == dtype and (td.c_contiguous if width_axis is None else rows_of(td, width_axis) is not None)


class RowLayoutOp(og.TensorOp):
    """x as a row kernel takes it (`_fits`), in other memory than the tensors `apart`, which the kernel writes; in
    the graph until RowLayoutPass has seen what the other passes made of x."""

    def __init__(self, x, width_axis, apart=(), **kwargs):
        super(RowLayoutOp, self).__init__(args=(x,), axes=x.axes, dtype=x.dtype, **kwargs)
        self.width_axis, self.apart = width_axis, apart
        self.deriv_handler = _Adjoint(lambda add_delta, adjoints, delta: add_delta(adjoints, self.args[0], delta))


class RowLayoutPass(PeepholeGraphPass):
    """Resolves every RowLayoutOp; has to be the last pass."""

    def visit(self, op, *args):
        if isinstance(op, RowLayoutOp):
            x, = args
            td = _td(x)
            if _fits(td, op.dtype, op.width_axis) and not any(t.tensor_description().base == td.base for t in op.apart):
                self.replace_op(op, x)
            elif td.dtype == op.dtype:
                self.replace_op(op, og.ContiguousOp(x))
            else:
                # (x16 * 1.0 has dtype float32 and becomes x16)
                self.replace_op(op, _copied(x, op.axes, op.dtype))


def _laid_out(x, width_axis):
    # (no pass replaces the read of a tensor with storage of its own)
    x = og.as_op(x)
    return x if isinstance(x, og.TensorValueOp) and _fits(_td(x), x.dtype, width_axis) else RowLayoutOp(x, width_axis)


def _as_rows(x, width_axis):
    """x with width_axis last and rows as rows_of wants them, by a device copy if there is no other way."""
    x = og.as_op(x)
    if x.axes[len(x.axes) - 1] != width_axis:
        others = [a for a in x.axes if a != width_axis]
        x = og.axes_with_order(x, og.make_axes(others + [width_axis]))
    return _laid_out(x, width_axis)


def _dense(x):
    """x in C order, by a device copy if its view is not."""
    return _laid_out(x, None)


def _check_dtype(op, allowed, what):
    if not isinstance(op.dtype, np.dtype) or op.dtype not in allowed:
        raise ValueError("%s: dtype %s (%s)" % (what, op.dtype, ", ".join(str(d) for d in allowed)))


def _cast(x, dtype):
    """x as `dtype` (a device copy where it is another)."""
    x = og.as_op(x)
    return x if x.dtype == dtype else _copied(x, x.axes, dtype)


def _copied(x, axes, dtype):
    copy = og.temporary(axes=axes, dtype=dtype)
    return og.sequential([og.AssignOp(copy, x), copy])


class RowResultOp(og.TensorOp):
    """A further result `name` of `main`, written by main's kernel: storage of its own, nothing to run."""

    def __init__(self, main, name, axes, dtype, **kwargs):
        super(RowResultOp, self).__init__(args=(main,), axes=axes, dtype=dtype, **kwargs)
        self.result_name = name
        main.results[name] = self

    @property
    def is_device_op(self):
        return False


class _Adjoint(object):
    """Differentiates an op or one of its results (the graph's `deriv_handler`)."""

    def __init__(self, generate):
        self.generate_adjoints = generate


# ------------------------------------------------------------------------------------- embedding
class EmbeddingOp(og.TensorOp):
    """scale * table[tokens[...], :]; axes: those of the tokens, then the table's second."""

    def __init__(self, table, tokens, scale=1.0, pad_idx=None, **kwargs):
        table, tokens = og.as_op(table), og.as_op(tokens)
        if len(table.axes) != 2:
            raise ValueError("embedding: a table of 2 axes, got {}".format(table.axes))
        _check_dtype(table, (F32, F16), "embedding: table")
        _check_dtype(tokens, (I32,), "embedding: tokens")
        vocab_axis, width_axis = table.axes[0], table.axes[1]
        if len(tokens.axes) == 0 or width_axis in tokens.axes or vocab_axis in tokens.axes:
            raise ValueError("embedding: token axes {} with table axes {}".format(tokens.axes, table.axes))
        table = _as_rows(table, width_axis)
        tokens = _dense(tokens)
        self.scale_factor, self.pad_idx = float(scale), -1 if pad_idx is None else int(pad_idx)
        if not -2 ** 31 <= self.pad_idx < 2 ** 31:
            raise ValueError("embedding: pad_idx {} is no int32".format(pad_idx))
        self.results = {}
        super(EmbeddingOp, self).__init__(args=(table, tokens), axes=tokens.axes + og.make_axes([width_axis]), dtype=table.dtype, **kwargs)
        self.deriv_handler = _Adjoint(self._adjoints)

    def _adjoints(self, add_delta, adjoints, delta):
        table, tokens = self.args
        delta = og.axes_with_order(og.broadcast(delta, self.axes), self.axes)
        add_delta(adjoints, table.forwarded, EmbeddingGradOp(table.axes, tokens, delta, self.scale_factor, self.pad_idx, table.dtype))


class EmbeddingGradOp(og.TensorOp):
    """The gradient of an EmbeddingOp's table: the scaled rows of `delta` added up by token."""

    def __init__(self, table_axes, tokens, delta, scale, pad_idx, dtype, **kwargs):
        delta = _as_rows(_cast(delta, dtype), table_axes[1])
        self.scale_factor, self.pad_idx = scale, pad_idx
        self.results = {}
        super(EmbeddingGradOp, self).__init__(args=(tokens, delta), axes=table_axes, dtype=dtype, **kwargs)


def embedding(table, tokens, scale=1.0, pad_idx=None):
    """Rows of `table` [V, F] (float32 or float16) by int32 `tokens`, times `scale`; zeros for tokens equal to
    pad_idx or outside [0, V).  Its derivative adds up a token's rows in order of their places."""
    return EmbeddingOp(table, tokens, scale, pad_idx)


# ------------------------------------------------------------------------------------- block norm
class BlockNormOp(og.TensorOp):
    """y = N(h) * gain + bias with h = residual_scale * x + gate * (N(b) * post_gain + post_bias), rows along
    x's last axis.  `stream` is h."""

    def __init__(self, x, b, gain, bias, post_gain, post_bias, gate, kind, post_norm, residual_scale, eps, **kwargs):
        x = og.as_op(x)
        width = x.axes[len(x.axes) - 1]
        _check_dtype(x, (F32, F16), "block_norm: x")
        if kind not in ("rms", "layer"):
            raise ValueError("block_norm: kind %r (rms or layer)" % (kind,))
        if b is None and (post_norm or post_gain is not None or post_bias is not None or gate is not None):
            raise ValueError("block_norm: a norm, gain, bias or gate after the block, and no block output")
        if not post_norm and (post_gain is not None or post_bias is not None):
            raise ValueError("block_norm: a gain or bias after the block without post_norm")
        x = _as_rows(x, width)
        self.width_axis, self.kind, self.post_norm = width, kind, bool(post_norm)
        self.residual_scale, self.eps = float(residual_scale), float(eps)
        operands = [("x", x)]
        if b is not None:
            b = og.as_op(b)
            if not b.axes.is_equal_set(x.axes) or b.dtype != x.dtype:
                raise ValueError("block_norm: block output {} {} beside the stream {} {}".format(b.axes, b.dtype, x.axes, x.dtype))
            operands.append(("b", _as_rows(og.axes_with_order(b, x.axes), width)))
        param_dtypes = set()
        for name, p in (("gain", gain), ("bias", bias), ("post_gain", post_gain), ("post_bias", post_bias)):
            if p is None:
                continue
            p = og.as_op(p)
            if list(p.axes) != [width]:
                raise ValueError("block_norm: {} has axes {}, not {}".format(name, p.axes, width))
            param_dtypes.add(p.dtype)
            operands.append((name, _dense(p)))
        self.gate_rows = 0
        if gate is not None:
            gate = og.as_op(gate)
            lead = [a for a in gate.axes if a != width]
            if width not in gate.axes or lead != list(x.axes)[:len(lead)]:
                raise ValueError("block_norm: gate axes {} are not the first axes of {} and {}".format(gate.axes, x.axes, width))
            param_dtypes.add(gate.dtype)
            operands.append(("gate", _as_rows(gate, width)))
            self.gate_rows = x.axes.size // width.length // int(np.prod([a.length for a in lead], dtype=np.int64))
        if len(param_dtypes) > 1 or any(d not in (F32, x.dtype) for d in param_dtypes):
            raise ValueError("block_norm: gains, biases and gate share a dtype, float32 or the stream's; got {}".format(sorted(map(str, param_dtypes))))
        self.param_dtype = param_dtypes.pop() if param_dtypes else x.dtype
        self.operand_names = [n for n, _ in operands]
        self.results = {}
        super(BlockNormOp, self).__init__(args=tuple(o for _, o in operands), axes=x.axes, dtype=x.dtype, **kwargs)
        self.stream = RowResultOp(self, "h", x.axes, x.dtype)
        self.deriv_handler = _Adjoint(self._adjoints)
        self.stream.deriv_handler = _Adjoint(self._stream_adjoints)

    def operand(self, name):
        return self.args[self.operand_names.index(name)].forwarded if name in self.operand_names else None

    # The adjoint of the stream arrives first (it depends on this op): it is kept until this op's own turn, for
    # which there has to be an entry; a zero stands for "no gradient of y".
    def _stream_adjoints(self, add_delta, adjoints, delta):
        adjoints[("stream", self)] = delta
        if self.forwarded not in adjoints:
            zero = og.broadcast(og.constant(0.0, dtype=self.dtype), self.axes)
            adjoints[("no y", self)] = zero
            adjoints[self.forwarded] = zero

    def _adjoints(self, add_delta, adjoints, delta):
        dh, dy = adjoints.pop(("stream", self), None), delta
        if adjoints.pop(("no y", self), None) is delta:
            dy = None
        grad = BlockNormGradOp(self, dy, dh)
        add_delta(adjoints, self.operand("x"), grad)
        for name in self.operand_names[1:]:
            if "d" + name in grad.results:
                add_delta(adjoints, self.operand(name), grad.results["d" + name])


class BlockNormGradOp(og.TensorOp):
    """The gradient of a BlockNormOp's x; results: those of its other operands by name ("db", "dgain", ...)."""

    def __init__(self, norm, dy, dh, **kwargs):
        self.norm = norm
        width = norm.width_axis
        operands = [("h", norm.stream)]
        if norm.operand("b") is not None:
            operands.append(("b", norm.operand("b")))
        for name, d in (("dy", dy), ("dh", dh)):
            if d is not None:
                d = og.axes_with_order(og.broadcast(og.as_op(d), norm.axes), norm.axes)
                operands.append((name, _as_rows(_cast(d, norm.dtype), width)))
        vectors = [n for n in norm.operand_names if n not in ("x", "b")]
        if dy is None:
            vectors = [n for n in vectors if n not in ("gain", "bias")]
        operands += [(n, norm.operand(n)) for n in vectors if n != "bias"]
        self.operand_names = [n for n, _ in operands]
        self.results = {}
        super(BlockNormGradOp, self).__init__(args=tuple(o for _, o in operands), axes=norm.axes, dtype=norm.dtype, **kwargs)
        if norm.operand("b") is not None:
            RowResultOp(self, "db", norm.axes, norm.dtype)
        for n in vectors:
            RowResultOp(self, "d" + n, norm.operand(n).axes, norm.param_dtype)


def block_norm(x, b=None, gain=None, bias=None, post_gain=None, post_bias=None, gate=None, kind="rms", post_norm=None, residual_scale=1.0,
               eps=1e-5):
    """(y, h): the stream h = residual_scale * x + gate * u after a block with output b, u = N(b) * post_gain +
    post_bias with post_norm and b without, and the next block's input y = N(h) * gain + bias.

    N is the rms or the layer norm over x's last axis.  post_norm defaults to whether a post gain or bias is
    given; gate's axes are the last axis alone, or the first ones of x's and the last.  b None: only the norm
    before the first block, h = residual_scale * x."""
    if post_norm is None:
        post_norm = post_gain is not None or post_bias is not None
    op = BlockNormOp(x, b, gain, bias, post_gain, post_bias, gate, kind, post_norm, residual_scale, eps)
    return op, op.stream


# ------------------------------------------------------------------------------------- AdamW
class AdamWOp(og.Op):
    """One AdamW update of `variables` by `grads`; states: persistent tensors made here (m, v and, with 8
    bits, their scales) and `step`, an int32 that counts the updates."""

    def __init__(self, variables, grads, lr=1e-3, beta_1=0.9, beta_2=0.999, epsilon=1e-8, weight_decay=(), state_bits=32, grad_scale=1.0,
                 clip_factor=None, **kwargs):
        if state_bits not in (8, 32):
            raise ValueError("AdamW: states of %r bits (8 or 32)" % (state_bits,))
        if len(variables) != len(grads) or len(weight_decay) != len(variables):
            raise ValueError("AdamW: %d variables, %d gradients, %d decays" % (len(variables), len(grads), len(weight_decay)))
        if not all(isinstance(v, og.AssignableTensorOp) for v in variables):
            raise ValueError("AdamW updates variables, got {}".format([v for v in variables if not isinstance(v, og.AssignableTensorOp)]))
        if len(set(variables)) != len(variables):
            raise ValueError("AdamW: a variable is given twice")
        args = []
        for v, g in zip(variables, grads):
            _check_dtype(v, (F32, F16), "AdamW: variable")
            g = og.as_op(g)
            if not g.axes.is_equal_set(v.axes):
                raise ValueError("AdamW: a gradient with axes {} for a variable with {}".format(g.axes, v.axes))
            _check_dtype(g, (F32, F16), "AdamW: gradient")
            # (the gradient of sum(v * w) in v is w itself)
            args.append(RowLayoutOp(og.axes_with_order(g, v.axes), None, apart=variables))
        for what, kinds in (("variables", set(v.dtype for v in variables)), ("gradients", set(a.dtype for a in args))):
            if len(kinds) > 1:
                raise ValueError("AdamW: %s of several dtypes; use an op for each (neon's AdamW does)" % what)
        self.variables, self.n = list(variables), len(variables)
        self.grad_dtype = args[0].dtype if args else F32
        self.beta_1, self.beta_2, self.epsilon = float(beta_1), float(beta_2), float(epsilon)
        self.weight_decay, self.state_bits, self.grad_scale = [float(w) for w in weight_decay], state_bits, float(grad_scale)
        self.lr = lr if isinstance(lr, og.Op) else float(lr)
        self.scalar_names = []
        for name, s in (("lr", self.lr if isinstance(self.lr, og.Op) else None), ("clip", clip_factor)):
            if s is not None:
                s = og.as_op(s)
                if not s.is_scalar or s.dtype != F32:
                    raise ValueError("AdamW: %s is a float32 scalar, got %s %s" % (name, s.axes, s.dtype))
                self.scalar_names.append(name)
                args.append(_dense(s))
        self.step = og.persistent_tensor(axes=(), dtype=I32, initial_value=0)
        self.m, self.v, self.m_scale, self.v_scale = [], [], [], []
        for var in variables:
            if state_bits == 8:
                blocks = og.make_axis((var.axes.size + STATE_BLOCK - 1) // STATE_BLOCK)
                self.m.append(og.persistent_tensor(axes=var.axes, dtype=np.dtype(np.int8), initial_value=0))
                self.v.append(og.persistent_tensor(axes=var.axes, dtype=np.dtype(np.uint8), initial_value=0))
                self.m_scale.append(og.persistent_tensor(axes=[blocks], initial_value=0.))
                self.v_scale.append(og.persistent_tensor(axes=[blocks], initial_value=0.))
            else:
                self.m.append(og.persistent_tensor(axes=var.axes, initial_value=0.))
                self.v.append(og.persistent_tensor(axes=var.axes, initial_value=0.))
        super(AdamWOp, self).__init__(args=tuple(args), **kwargs)

    @property
    def written_tensors(self):
        """Tensors the op changes in place (the planner moves no read of them across it)."""
        return self.variables + self.m + self.v + self.m_scale + self.v_scale + [self.step]

    @property
    def states_written(self):
        return og.OrderedSet(self.written_tensors)

    @property
    def states_read(self):
        return super(AdamWOp, self).states_read | og.OrderedSet(self.written_tensors)

    @property
    def has_side_effects(self):
        return True


# ------------------------------------------------------------------------------------- kernels
class RowKernel(HipKernel):
    """A kernel of this module: `spec` filled when the buffers are bound, one call to run it."""

    def __init__(self, transformer, op):
        super(RowKernel, self).__init__(transformer)
        self.op = op
        self.spec = None

    def view(self, op):
        return self.transformer.get_tensor_description_tensor_view(_td(op.forwarded))

    def code(self, dtype):
        return self.transformer.ngh_dtype(dtype)

    def checked(self, op, axes, dtype, width_axis=None):
        """The description of an operand, after checking that the kernel can take it."""
        td = _td(op.forwarded)
        if not _fits(td, dtype, width_axis) or td.axes.lengths != og.make_axes(axes).lengths:
            raise og_unsupported("%s: operand %s is %s with strides %s, %s" % (type(self.op).__name__, op, td.axes, tuple(td.full_strides), td.dtype))
        return td

    def rows(self, op, axes, dtype):
        """(address, rows, row stride) of a row operand."""
        width_axis = axes[len(axes) - 1]
        layout = rows_of(self.checked(op, axes, dtype, width_axis), width_axis)
        return self.view(op).ptr, layout[0], layout[2]

    def dense(self, op, axes, dtype):
        """The address of an operand whose elements follow one another."""
        self.checked(op, axes, dtype)
        return self.view(op).ptr

    def results(self):
        """The op's further results that the transformer's computations hold: {name: op}."""
        held = set(o.forwarded for o in self.transformer.ops)
        return {n: r for n, r in getattr(self.op, "results", {}).items() if r.forwarded in held}

    def buffer_uses(self):
        uses = [(_td(a.forwarded).base, True, False) for a in self.op.args]
        uses.append((_td(self.op).base, False, True))
        return uses + [(_td(r).base, False, True) for r in self.results().values()]

    def workspace(self, n):
        """Device memory of this kernel's own (the runtime frees it when it closes)."""
        return self.transformer.runtime.malloc(n)

    def describe(self):
        return [[self.name]]


class EmbeddingKernel(RowKernel):
    name = "embedding"

    def bind_buffers(self):
        table, tokens = (a.forwarded for a in self.op.args)
        width = self.op.axes[len(self.op.axes) - 1]
        at, vocab, stride = self.rows(table, table.axes, self.op.dtype)
        y, n, y_stride = self.rows(self.op, self.op.axes, self.op.dtype)
        self.spec = self.transformer.runtime.embedding_spec(
            n, vocab, width.length, self.dense(tokens, list(self.op.axes)[:-1], I32), at, y, self.code(self.op.dtype), None,
            self.op.scale_factor, self.op.pad_idx, stride, y_stride)
        super(EmbeddingKernel, self).bind_buffers()

    def execute(self):
        self.transformer.runtime.embedding(self.spec)


class EmbeddingGradKernel(RowKernel):
    name = "embedding_grad"

    def bind_buffers(self):
        rt = self.transformer.runtime
        tokens, delta = (a.forwarded for a in self.op.args)
        width = self.op.axes[1]
        at, vocab, stride = self.rows(self.op, self.op.axes, self.op.dtype)
        dy, n, dy_stride = self.rows(delta, list(tokens.axes) + [width], self.op.dtype)
        s = rt.embedding_grad_spec(n, vocab, width.length, self.dense(tokens, tokens.axes, I32), dy, at, self.code(self.op.dtype), None,
                                   self.op.scale_factor, self.op.pad_idx, False, stride, dy_stride)
        s.workspace_bytes = rt.embedding_grad_workspace(s)
        s.workspace = self.workspace(s.workspace_bytes)
        self.spec = s
        super(EmbeddingGradKernel, self).bind_buffers()

    def execute(self):
        self.transformer.runtime.embedding_grad(self.spec)


def _norm_spec(kernel, norm, operands):
    """The block norm spec with the addresses and strides of `operands` ({field: op})."""
    width = norm.width_axis
    fields = {}
    for name, op in operands.items():
        if name in ("gain", "bias", "post_gain", "post_bias", "dgain", "dbias", "dpost_gain", "dpost_bias"):
            fields[name] = kernel.dense(op, [width], norm.param_dtype)
        elif name in ("gate", "dgate"):
            fields[name], _, fields[name + "_stride"] = kernel.rows(op, norm.operand("gate").axes, norm.param_dtype)
        else:
            fields[name], _, fields[name + "_stride"] = kernel.rows(op, norm.axes, norm.dtype)
    return kernel.transformer.runtime.block_norm_spec(
        norm.axes.size // width.length, width.length, norm.kind, kernel.code(norm.dtype), kernel.code(norm.param_dtype), norm.post_norm,
        norm.gate_rows if "gate" in operands else 0, norm.residual_scale, norm.eps, **fields)


class BlockNormKernel(RowKernel):
    name = "block_norm"

    def bind_buffers(self):
        op = self.op
        operands = dict(zip(op.operand_names, op.args))
        operands["y"] = op
        operands.update(self.results())
        self.spec = _norm_spec(self, op, operands)
        super(BlockNormKernel, self).bind_buffers()

    def execute(self):
        self.transformer.runtime.block_norm(self.spec)


class BlockNormGradKernel(RowKernel):
    name = "block_norm_grad"

    def bind_buffers(self):
        op, rt = self.op, self.transformer.runtime
        operands = dict(zip(op.operand_names, op.args))
        results = self.results()
        operands["dx"] = op
        operands.update(results)
        if "db" not in results and "b" in operands:
            # nothing asks for the block's gradient: with those of the norm behind it, its rows are written aside
            if any(n in results for n in ("dgate", "dpost_gain", "dpost_bias")):
                operands["db"] = op.results["db"]
            else:
                for n in ("b", "post_gain", "post_bias", "gate"):
                    operands.pop(n, None)
        aside = operands.get("db") is not None and "db" not in results
        if aside:
            del operands["db"]
        spec = _norm_spec(self, op.norm, operands)
        if "b" not in operands:
            spec.post_norm = 0
        if aside:
            width = op.norm.width_axis.length
            spec.db = self.workspace(op.norm.axes.size * op.dtype.itemsize)
            spec.db_stride = width
        spec.workspace_bytes = rt.block_norm_grad_workspace(spec)
        spec.workspace = self.workspace(spec.workspace_bytes)
        self.spec = spec
        super(BlockNormGradKernel, self).bind_buffers()

    def execute(self):
        self.transformer.runtime.block_norm_grad(self.spec)


class AdamWKernel(RowKernel):
    name = "adamw"
    plan = None

    def buffer_uses(self):
        return [(_td(a.forwarded).base, True, False) for a in self.op.args] + \
            [(t.tensor_description().base, True, True) for t in self.op.written_tensors]

    def bind_buffers(self):
        op, rt = self.op, self.transformer.runtime
        at = lambda t: self.dense(t, t.axes, t.dtype)                                                 # noqa: E731
        rows = []
        for i, var in enumerate(op.variables):
            row = dict(param=at(var), grad=self.dense(op.args[i], var.axes, op.grad_dtype), m=at(op.m[i]), v=at(op.v[i]), n=var.axes.size,
                       weight_decay=op.weight_decay[i])
            if op.state_bits == 8:
                row.update(m_scale=at(op.m_scale[i]), v_scale=at(op.v_scale[i]))
            rows.append(row)
        kinds = dict(param_dtype=self.code(op.variables[0].dtype), grad_dtype=self.code(op.grad_dtype)) if rows else {}
        self.plan = rt.adamw_plan(rows, state_bits=op.state_bits, **kinds)
        scalars = dict(zip(op.scalar_names, op.args[op.n:]))
        self.hyper = dict(lr=0.0 if "lr" in scalars else op.lr, beta1=op.beta_1, beta2=op.beta_2, eps=op.epsilon, grad_scale=op.grad_scale,
                          dev_step=at(op.step), dev_lr=self.dense(scalars["lr"], (), F32) if "lr" in scalars else None,
                          dev_grad_scale=self.dense(scalars["clip"], (), F32) if "clip" in scalars else None)
        super(AdamWKernel, self).bind_buffers()

    def execute(self):
        self.transformer.runtime.adamw_step(self.plan, **self.hyper)


KERNELS = ((EmbeddingOp, EmbeddingKernel), (EmbeddingGradOp, EmbeddingGradKernel), (BlockNormOp, BlockNormKernel),
           (BlockNormGradOp, BlockNormGradKernel), (AdamWOp, AdamWKernel))


def row_kernel(transformer, op):
    """The kernel of one of this module's ops, else None."""
    for cls, kernel in KERNELS:
        if isinstance(op, cls):
            if any(not isinstance(o.dtype, np.dtype) for o in [op] + list(op.args) if o.is_tensor_op):
                raise og_unsupported("%s takes no flex tensors" % cls.__name__)
            return kernel(transformer, op)
    return None
