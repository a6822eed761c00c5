"""A training step of the operators over rows and parameters through the C ABI: embedding, the norm before a
block (whose output is the stream's own copy), their gradients and AdamW; eager, recorded with eager work
between the replays, and on two contexts at once.  Every sum has a fixed order: all of them give the same bits.
"""
import threading

import numpy as np
import pytest

from ngraph_hip.runtime import HipRuntime
from row_helpers import DTYPES, Pool, rounded

pytestmark = pytest.mark.gpu
f32 = np.float32


class Step(object):
    """Buffers and specs of a step over n tokens; `launch` enqueues it, `state` is all it changes."""

    def __init__(self, rt, pool, n=3000, vocab=700, width=200, dtype="bf16", bits=8, seed=0):
        self.rt, self.n, self.vocab = rt, n, vocab
        rs = np.random.RandomState(seed)
        act = lambda: pool.rows((n, width), dtype)                                                       # noqa: E731
        new = lambda rows, mean, std: pool.rows((rows, width), "f32", rs.normal(mean, std, (rows, width)).astype(f32))   # noqa: E731
        self.tokens = pool.array(np.zeros(n, np.int32))
        self.target = pool.rows((n, width), dtype, rounded(rs.normal(0, 1, (n, width)), dtype))
        self.table, self.gain, self.post, self.gate = new(vocab, 0, 1), new(1, 1, 0.1), new(1, 1, 0.1), new(1, 0.5, 0.1)
        self.grads = [new(r.rows, 0, 0) for r in (self.table, self.gain, self.post, self.gate)]
        x, h, y, dx, db = act(), act(), act(), act(), act()
        d = DTYPES[dtype]
        self.lookup = rt.embedding_spec(n, vocab, width, self.tokens.ptr, self.table.ptr, x.ptr, 0, d, scale=2.0, pad_idx=3)
        common = dict(gain=self.gain.ptr, post_gain=self.post.ptr, gate=self.gate.ptr, b=self.target.ptr)
        self.norm = rt.block_norm_spec(n, width, "rms", d, 0, True, n, 0.5, x=x.ptr, h=h.ptr, y=y.ptr, **common)
        self.back = rt.block_norm_spec(n, width, "rms", d, 0, True, n, 0.5, h=h.ptr, dy=y.ptr, dh=x.ptr, dx=dx.ptr, db=db.ptr,
                                       dgain=self.grads[1].ptr, dpost_gain=self.grads[2].ptr, dgate=self.grads[3].ptr, **common)
        self.scatter = rt.embedding_grad_spec(n, vocab, width, self.tokens.ptr, dx.ptr, self.grads[0].ptr, d, 0, 2.0, 3)
        for spec, size in ((self.back, rt.block_norm_grad_workspace), (self.scatter, rt.embedding_grad_workspace)):
            spec.workspace_bytes = size(spec)
            spec.workspace = pool.bytes(spec.workspace_bytes).ptr
        self.count = pool.array(np.zeros(1, np.int32))
        rows, self.moments = [], []
        for p, g in zip((self.table, self.gain, self.post, self.gate), self.grads):
            size = p.rows * width
            held = [pool.array(np.zeros(size, np.uint8 if bits == 8 else f32)) for _ in range(2)]
            scales = [pool.array(np.zeros((size + 255) // 256, f32)) for _ in range(2)] if bits == 8 else []
            self.moments += held + scales
            rows.append(dict(param=p.ptr, grad=g.ptr, n=size, m=held[0].ptr, v=held[1].ptr, weight_decay=0.01,
                             **(dict(m_scale=scales[0].ptr, v_scale=scales[1].ptr) if scales else {})))
        self.plan = rt.adamw_plan(rows, state_bits=bits)

    def launch(self):
        rt = self.rt
        rt.embedding(self.lookup)
        rt.block_norm(self.norm)
        rt.block_norm_grad(self.back)
        rt.embedding_grad(self.scatter)
        rt.adamw_step(self.plan, lr=1e-2, dev_step=self.count.ptr)

    def feed(self, k):
        t = np.random.RandomState(100 + k).randint(-1, self.vocab + 1, self.n).astype(np.int32)
        t[::3] = 7
        self.tokens.set(t)

    def state(self):
        return [p.get() for p in [self.table, self.gain, self.post, self.gate] + self.grads] + [m.get() for m in self.moments]


def same(a, b):
    for x, y in zip(a, b):
        np.testing.assert_array_equal(x, y)


@pytest.mark.parametrize("n,bits", [(3000, 8), (700, 32), (20000, 8)])
def test_recorded_steps_equal_eager_ones(hip_runtime, n, bits):
    rt = hip_runtime
    with Pool(rt) as pool:
        eager, recorded = Step(rt, pool, n, bits=bits), Step(rt, pool, n, bits=bits)
        rt.graph_begin()
        recorded.launch()
        graph = rt.graph_end()
        try:
            for k in range(4):
                eager.feed(k)
                recorded.feed(k)
                eager.launch()
                rt.graph_launch(graph)
                assert recorded.count.get()[0] == eager.count.get()[0] == k + 1
                same(eager.state(), recorded.state())
        finally:
            rt.graph_free(graph)
        assert np.isfinite(recorded.table.get()).all() and recorded.grads[0].get().any()
        for s in (eager, recorded):
            rt.adamw_plan_free(s.plan)


def test_two_contexts_at_once(hip_runtime):
    """Threads with a context each, their launches interleaved; against the session's context alone."""
    with Pool(hip_runtime) as pool:
        alone = Step(hip_runtime, pool, 5000)
        for k in range(6):
            alone.feed(k)
            alone.launch()
        want = alone.state()
        hip_runtime.adamw_plan_free(alone.plan)
    got, failed, start = {}, [], threading.Barrier(2, timeout=60)

    def work(i):
        try:
            rt = HipRuntime(0)
            try:
                with Pool(rt) as pool:
                    step = Step(rt, pool, 5000)
                    start.wait()
                    for k in range(6):
                        step.feed(k)
                        step.launch()
                    got[i] = step.state()
                    rt.adamw_plan_free(step.plan)
            finally:
                rt.close()
        except Exception as e:                           # (seen by the test's own thread)
            failed.append(e)
            start.abort()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not failed and len(got) == 2, failed
    for i in got:
        same(got[i], want)
