"""The memory-bound operators of a language model's training step, as cases that can be timed: the embedding lookup and its
gradient, the norms around a block with its gate and residual, and AdamW over many tensors.

With `own` false every operator is computed in its plain form (elementary torch operations in 32 bits, rounded once at the
end); with `own` true through libngraph_hip, the way a program that keeps its buffers on the device calls it.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 256                      # elements that share a scale in the 8-bit states, and the alignment of a parameter's start

_runtime = None


def runtime():
    """The process's device context of the framework."""
    global _runtime
    if _runtime is None:
        import os
        import sys
        path = os.path.join(os.getcwd(), "ngraph-python_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        from ngraph_hip.runtime import HipRuntime
        _runtime = HipRuntime(0)
    return _runtime


def code(dtype):
    from ngraph_hip.runtime import hiplib
    return {"f32": hiplib.NGH_F32, "bf16": hiplib.NGH_BF16, "f16": hiplib.NGH_F16}[dtype]


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one new token of a generating program: a row of a large table, all latency
        dict(name="embedding_one_token", op="embedding", n=1, vocab=32768, width=2048, dtype="bf16", out="bf16", scale=45.25, pad=False),
        # the tokens of a large training batch, fp32 table read into bf16 activations
        dict(name="embedding_batch", op="embedding", n=65536, vocab=131072, width=2048, dtype="f32", out="bf16", scale=1.0, pad=True),
        # a small fp32 model with an odd width and vocabulary, padded batch: the whole gradient table is written
        dict(name="embedding_grad_odd", op="embedding_grad", n=1999, vocab=20011, width=301, dtype="f32", out="f32", scale=17.35, pad=True,
             accumulate=False),
        # an ordinary step: bf16 gradients into an fp32 table
        dict(name="embedding_grad_step", op="embedding_grad", n=16384, vocab=65536, width=1024, dtype="bf16", out="f32", scale=32.0, pad=False,
             accumulate=False),
        # a large batch added to the gradient that the output layer left in a shared table
        dict(name="embedding_grad_tied", op="embedding_grad", n=131072, vocab=131072, width=2048, dtype="bf16", out="bf16", scale=1.0, pad=True,
             accumulate=True),
        # one new token through a block's end and the next block's beginning
        dict(name="block_norm_one_token", op="block_norm", rows=1, width=4096, kind="rms", dtype="bf16", params="bf16", post=True, gate_rows=0,
             bias=False, alpha=1.0),
        # a long batch: norm after the block, channel gate, residual, norm before the next block
        dict(name="block_norm_batch", op="block_norm", rows=16384, width=4096, kind="rms", dtype="bf16", params="f32", post=True, gate_rows=16384,
             bias=False, alpha=1.0),
        # its backward pass, with the gradients of both gains and of the gate
        dict(name="block_norm_grad_batch", op="block_norm_grad", rows=16384, width=4096, kind="rms", dtype="bf16", params="f32", post=True,
             gate_rows=16384, bias=False, alpha=1.0),
        # layer norms with gains and biases in fp32, an odd width, a gate for each sequence of 250 rows, a scaled residual
        dict(name="block_norm_grad_odd", op="block_norm_grad", rows=3000, width=1027, kind="layer", dtype="f32", params="f32", post=True,
             gate_rows=250, bias=True, alpha=1.5),
        # a small model's step: 69 small tensors, all launches
        dict(name="adamw_small", op="adamw", layers=6, width=128, vocab=1000, params="f32", grads="f32", bits=32),
        # 25 million parameters with states in 32 bits, as many as the framework's own optimiser benchmark has
        dict(name="adamw_25m", op="adamw", layers=6, width=512, vocab=13135, params="f32", grads="f32", bits=32),
        # a larger model with bf16 gradients and states in 8 bits
        dict(name="adamw_8bit", op="adamw", layers=8, width=1024, vocab=50001, params="f32", grads="bf16", bits=8),
    ]


def spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm; odd more often than not."""
    n = int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))
    if rng.random() < 0.3:
        n = n // 64 * 64
    return max(low, min(high, n))


def draw(rng):
    op = rng.choice(["embedding", "embedding_grad", "block_norm", "block_norm_grad", "adamw"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op in ("embedding", "embedding_grad"):
        width = spread(rng, 64, 4096)
        case = dict(op=op, vocab=spread(rng, 1000, min(131072, (1 << 27) // width)), width=width, n=spread(rng, 1, min(131072, (1 << 27) // width)), dtype=dtype,
                    out=rng.choice(["f32", "same"] if op == "embedding_grad" else ["same", "same", "bf16", "f16"] if dtype == "f32" else ["same"]),
                    scale=rng.choice([1.0, round(math.sqrt(width), 3)]), pad=rng.random() < 0.5)
        case["out"] = dtype if case["out"] == "same" else case["out"]
        if op == "embedding_grad":
            case["accumulate"] = rng.random() < 0.3
        return case
    if op in ("block_norm", "block_norm_grad"):
        width = spread(rng, 64, 8192)
        group = rng.choice([0, 1, 2, 3])                   # no gate, a gate for each row, for each sequence, one for all
        sequences = rng.randint(2, 9)
        rows = spread(rng, 1, min(65536, (1 << 25) // width))
        if group == 2:
            rows = max(1, rows // sequences) * sequences
        return dict(op=op, rows=rows, width=width, kind=rng.choice(["rms", "layer"]), dtype=dtype, params=rng.choice(["f32", dtype]),
                    post=rng.random() < 0.7, gate_rows=(0, 1, max(1, rows // sequences), rows)[group], bias=rng.random() < 0.4,
                    alpha=rng.choice([1.0, round(rng.uniform(0.5, 2.0), 3)]))
    return dict(op=op, layers=rng.randint(1, 8), width=spread(rng, 32, 700), vocab=spread(rng, 500, 32768),
                params=rng.choice(["f32", "f32", "bf16"]), grads=rng.choice(["f32", "bf16"]), bits=rng.choice([8, 32]))


def parameter_sizes(case):
    """Element counts of the parameters of a model with this many layers: matrices, gains and biases, the table last."""
    w = case["width"]
    layer = [w, w * w, w * w, w * w, w * w, w, w, 4 * w * w, 4 * w, 4 * w * w, w]
    return layer * case["layers"] + [w, w, case["vocab"] * w]


def parameter_starts(case):
    """Where each parameter starts in one allocation that keeps every start on a multiple of 256 elements; and its length."""
    lengths = np.array(parameter_sizes(case), dtype=np.int64)
    room = (lengths + BLOCK - 1) // BLOCK * BLOCK
    return np.concatenate([[0], np.cumsum(room)[:-1]]), lengths, int(room.sum())


def distinct(n, vocab):
    """How many different tokens n draws hold on average where the k-th most frequent one has a share of 1/k."""
    p = np.log1p(1.0 / np.arange(1, vocab + 1)) / math.log(vocab + 1)
    return float((1 - np.exp(n * np.log1p(-p))).sum())


def work(case):
    op = case["op"]
    if op == "embedding":
        n, d = case["n"], case["width"]
        rows = distinct(n, case["vocab"])
        return {"bytes": 4 * n + rows * d * SIZE[case["dtype"]] + n * d * SIZE[case["out"]], "flops": n * d}
    if op == "embedding_grad":
        n, d = case["n"], case["width"]
        rows = 2 * distinct(n, case["vocab"]) if case["accumulate"] else case["vocab"]
        return {"bytes": 4 * n + n * d * SIZE[case["dtype"]] + rows * d * SIZE[case["out"]], "flops": n * d}
    if op in ("block_norm", "block_norm_grad"):
        n, d, e, q = case["rows"], case["width"], SIZE[case["dtype"]], SIZE[case["params"]]
        gates = 0 if not case["gate_rows"] else n // case["gate_rows"]
        vectors = (1 + case["post"]) * (1 + case["bias"]) + gates
        back = op == "block_norm_grad"
        return {"bytes": n * d * e * (6 if back else 4) + vectors * d * q * (2 if back else 1), "flops": n * d * (30 if back else 14)}
    starts, lengths, total = parameter_starts(case)
    n = int(lengths.sum())
    state = 16 if case["bits"] == 32 else 4 + 16.0 / BLOCK + 8          # 8 bits: codes and scales both ways, and the values they stand for
    return {"bytes": n * (2 * SIZE[case["params"]] + SIZE[case["grads"]] + state), "flops": n * (14 if case["bits"] == 32 else 40)}


# ------------------------------------------------------------------------------------------------ inputs
def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, shape, dtype="f32", std=1.0, mean=0.0):
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    return (x * std + mean).to(DTYPES[dtype])


def draw_tokens(g, n, vocab, pad):
    """Token numbers with the frequencies of a text: the k-th most frequent has a share of 1/k, frequent ones anywhere in the table."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    rank = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).long().clamp_(0, vocab - 1)
    t = torch.randperm(vocab, generator=g, device="cuda")[rank].to(torch.int32)
    if pad:                      # the ends of short sequences in a batch
        t[torch.rand(n, generator=g, device="cuda") < 0.06] = 0
    return t


def prepare(case, seed):
    g = generator(seed)
    op, s = case["op"], {"case": case}
    if op == "embedding":
        n, v, d = case["n"], case["vocab"], case["width"]
        s["pad"] = 0 if case["pad"] else -1
        s["table"] = normal(g, (v, d), case["dtype"], 0.02)
        s["tokens"] = draw_tokens(g, n, v, case["pad"])
        s["y"] = torch.empty((n, d), device="cuda", dtype=DTYPES[case["out"]])
        if own:
            s["spec"] = runtime().embedding_spec(
                n, v, d, s["tokens"].data_ptr(), s["table"].data_ptr(), s["y"].data_ptr(), table_dtype=code(case["dtype"]),
                y_dtype=code(case["out"]), scale=case["scale"], pad_idx=s["pad"])
    elif op == "embedding_grad":
        n, v, d = case["n"], case["vocab"], case["width"]
        s["pad"] = 0 if case["pad"] else -1
        s["dy"] = normal(g, (n, d), case["dtype"], 1e-2)
        s["tokens"] = draw_tokens(g, n, v, case["pad"])
        s["dtable"] = normal(g, (v, d), case["out"], 1e-2) if case["accumulate"] else torch.empty((v, d), device="cuda", dtype=DTYPES[case["out"]])
        if own:
            rt = runtime()
            s["spec"] = rt.embedding_grad_spec(
                n, v, d, s["tokens"].data_ptr(), s["dy"].data_ptr(), s["dtable"].data_ptr(), y_dtype=code(case["dtype"]),
                table_dtype=code(case["out"]), scale=case["scale"], pad_idx=s["pad"], accumulate=case["accumulate"])
            s["workspace"] = torch.empty(rt.embedding_grad_workspace(s["spec"]), device="cuda", dtype=torch.uint8)
            s["spec"].workspace, s["spec"].workspace_bytes = s["workspace"].data_ptr(), s["workspace"].numel()
    elif op in ("block_norm", "block_norm_grad"):
        prepare_norm(case, s, g)
    else:
        prepare_adamw(case, s, g)
    return s


def prepare_norm(case, s, g):
    n, d, dt, pt = case["rows"], case["width"], case["dtype"], case["params"]
    s["x"] = normal(g, (n, d), dt, 1.5, 0.1)
    s["b"] = normal(g, (n, d), dt, 0.7, -0.05)
    s["gain"] = normal(g, (d,), pt, 0.1, 1.0)
    s["bias"] = normal(g, (d,), pt, 0.1) if case["bias"] else None
    s["post_gain"] = normal(g, (d,), pt, 0.1, 1.0) if case["post"] else None
    s["post_bias"] = normal(g, (d,), pt, 0.1) if case["post"] and case["bias"] else None
    s["gate"] = normal(g, (n // case["gate_rows"], d), pt, 0.2, 0.5) if case["gate_rows"] else None
    like = {"gain": s["gain"], "bias": s["bias"], "post_gain": s["post_gain"], "post_bias": s["post_bias"], "gate": s["gate"]}
    if case["op"] == "block_norm":
        s["h"], s["y"] = torch.empty_like(s["x"]), torch.empty_like(s["x"])
        outs = dict(x=s["x"], b=s["b"], h=s["h"], y=s["y"])
    else:
        # the forward pass left the stream after the block; gradients arrive for it and for the norm's result
        s["h"] = plain_norm(case, s)["h"]
        s["dy"], s["dh"] = normal(g, (n, d), dt, 1e-2), normal(g, (n, d), dt, 1e-2)
        s["dx"], s["db"] = torch.empty_like(s["x"]), torch.empty_like(s["x"])
        s["grads"] = {k: torch.empty_like(t) for k, t in like.items() if t is not None}
        outs = dict(b=s["b"], h=s["h"], dy=s["dy"], dh=s["dh"], dx=s["dx"], db=s["db"], **{"d" + k: t for k, t in s["grads"].items()})
    if own:
        rt = runtime()
        s["spec"] = rt.block_norm_spec(n, d, kind=case["kind"], dtype=code(dt), param_dtype=code(pt), post_norm=case["post"],
                                       gate_rows=case["gate_rows"], residual_scale=case["alpha"], eps=1e-5,
                                       **{k: t.data_ptr() for k, t in {**like, **outs}.items() if t is not None})
        if case["op"] == "block_norm_grad":
            s["workspace"] = torch.empty(rt.block_norm_grad_workspace(s["spec"]), device="cuda", dtype=torch.uint8)
            s["spec"].workspace, s["spec"].workspace_bytes = s["workspace"].data_ptr(), s["workspace"].numel()


def encode(x, second):
    """8-bit codes and scales of blocks of 256 values: the value's share of the block's largest, under a root of order 2 (signed, the first
    moments) or 4 (the second), in 127 or 255 equal steps."""
    rows = x.reshape(-1, BLOCK)
    scale = rows.abs().amax(1, keepdim=True)
    share = torch.where(scale > 0, rows.abs() / scale, torch.zeros_like(rows))
    if second:
        return torch.round(torch.sqrt(torch.sqrt(share)) * 255.0).to(torch.uint8).reshape(-1), scale.reshape(-1)
    return (torch.round(torch.sqrt(share) * 127.0) * torch.sign(rows)).to(torch.int8).reshape(-1), scale.reshape(-1)


def decode(codes, scale, second):
    t = codes.reshape(-1, BLOCK).to(torch.float32) * (np.float32(1.0 / 255.0) if second else np.float32(1.0 / 127.0)).item()
    return (((t * t) * (t * t) if second else t * t.abs()) * scale.reshape(-1, 1)).reshape(-1)


def prepare_adamw(case, s, g):
    starts, lengths, total = parameter_starts(case)
    # one number for each element, nothing between the parameters
    inside = torch.zeros(total + 1, device="cuda", dtype=torch.int32)
    inside[torch.from_numpy(starts).cuda()] += 1
    inside.index_add_(0, torch.from_numpy(starts + lengths).cuda(), torch.full((len(starts),), -1, device="cuda", dtype=torch.int32))
    inside = (torch.cumsum(inside, 0)[:total] > 0).float()
    s["p"] = (normal(g, (total,), "f32", 0.02) * inside).to(DTYPES[case["params"]])
    # gradients of very different sizes from block to block, as layers have them
    size = torch.exp(normal(g, (total // BLOCK, 1), "f32", 1.5, -7.0))
    s["g"] = ((normal(g, (total // BLOCK, BLOCK), "f32") * size).reshape(-1) * inside).to(DTYPES[case["grads"]])
    m = (normal(g, (total // BLOCK, BLOCK), "f32", 0.3) * size).reshape(-1) * inside
    v = ((normal(g, (total // BLOCK, BLOCK), "f32", 0.3, 1.0) * size).square().reshape(-1)) * inside
    if case["bits"] == 8:
        s["m"], s["m_scale"] = encode(m, False)
        s["v"], s["v_scale"] = encode(v, True)
        s["m_out"], s["v_out"] = torch.empty_like(m), torch.empty_like(v)
    else:
        s["m"], s["v"] = m, v
    s["step"] = 100
    # no decay for gains and biases: those are the short ones
    decayed = np.where(lengths > 8 * case["width"], 0.1, 0.0)
    change = torch.zeros(total + 1, device="cuda", dtype=torch.float32)
    change.index_add_(0, torch.from_numpy(starts).cuda(), torch.from_numpy(decayed).float().cuda())
    change.index_add_(0, torch.from_numpy(starts + lengths).cuda(), torch.from_numpy(-decayed).float().cuda())
    s["decay"] = (torch.cumsum(change, 0)[:total] > 0.05).float() * 0.1
    if own:
        e, q = SIZE[case["params"]], SIZE[case["grads"]]
        w = 1 if case["bits"] == 8 else 4
        rows = [dict(param=s["p"].data_ptr() + int(a) * e, grad=s["g"].data_ptr() + int(a) * q, m=s["m"].data_ptr() + int(a) * w,
                     v=s["v"].data_ptr() + int(a) * w, n=int(n), weight_decay=float(z),
                     m_scale=s["m_scale"].data_ptr() + int(a) // BLOCK * 4 if w == 1 else None,
                     v_scale=s["v_scale"].data_ptr() + int(a) // BLOCK * 4 if w == 1 else None) for a, n, z in zip(starts, lengths, decayed)]
        s["plan"] = runtime().adamw_plan(rows, param_dtype=code(case["params"]), grad_dtype=code(case["grads"]), state_bits=case["bits"])


HYPER = dict(lr=3e-4, beta1=0.9, beta2=0.95, eps=1e-8)


# ------------------------------------------------------------------------------------------------ plain forms
def plain_embedding(case, s):
    t = s["tokens"].long()
    y = s["table"][t].float() * case["scale"]
    if case["pad"]:
        y = torch.where((t == s["pad"])[:, None], torch.zeros_like(y), y)
    return {"y": y.to(DTYPES[case["out"]])}


def plain_embedding_grad(case, s):
    t, dy = s["tokens"].long(), s["dy"].float()
    if case["pad"]:
        dy = torch.where((t == s["pad"])[:, None], torch.zeros_like(dy), dy)
    total = torch.zeros((case["vocab"], case["width"]), device="cuda", dtype=torch.float32).index_add_(0, t, dy) * case["scale"]
    if case["accumulate"]:
        total += s["dtable"].float()
    s["dtable"].copy_(total)
    return {"dtable": s["dtable"]}


def normalise(case, x):
    """The normalised rows and the reciprocal root by which they were scaled."""
    if case["kind"] == "layer":
        x = x - x.mean(1, keepdim=True)
    r = 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-5)
    return x * r, r


def through(case, xh, r, t):
    """The gradient of the rows that `normalise` was given, for the gradient t of what it returned."""
    inner = t - xh * (t * xh).mean(1, keepdim=True)
    return r * (inner - t.mean(1, keepdim=True) if case["kind"] == "layer" else inner)


def gate_of(case, s):
    return s["gate"].float().repeat_interleave(case["gate_rows"], 0) if case["gate_rows"] not in (1, case["rows"]) else s["gate"].float()


def branch(case, s):
    """The block's output normalised, with its gain and bias; all before the gate."""
    bh, r = normalise(case, s["b"].float()) if case["post"] else (s["b"].float(), None)
    u = bh * s["post_gain"].float() if case["post"] else bh
    return bh, r, u if s["post_bias"] is None else u + s["post_bias"].float()


def plain_norm(case, s):
    u = branch(case, s)[2]
    h = case["alpha"] * s["x"].float() + (u * gate_of(case, s) if case["gate_rows"] else u)
    y = normalise(case, h)[0] * s["gain"].float()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return {"h": h.to(DTYPES[case["dtype"]]), "y": y.to(DTYPES[case["dtype"]])}


def plain_norm_grad(case, s):
    dt, pt = DTYPES[case["dtype"]], DTYPES[case["params"]]
    hh, r = normalise(case, s["h"].float())
    dy, out = s["dy"].float(), {}
    d = s["dh"].float() + through(case, hh, r, dy * s["gain"].float())
    out["dx"], out["dgain"] = (case["alpha"] * d).to(dt), (dy * hh).sum(0).to(pt)
    if s["bias"] is not None:
        out["dbias"] = dy.sum(0).to(pt)
    bh, rb, u = branch(case, s)
    if case["gate_rows"]:
        out["dgate"] = (d * u).reshape(-1, case["gate_rows"], case["width"]).sum(1).to(pt)
        d = d * gate_of(case, s)
    if case["post"]:
        out["dpost_gain"] = (d * bh).sum(0).to(pt)
        if s["post_bias"] is not None:
            out["dpost_bias"] = d.sum(0).to(pt)
        d = through(case, bh, rb, d * s["post_gain"].float())
    out["db"] = d.to(dt)
    return out


def plain_adamw(case, s):
    k, t = HYPER, s["step"]
    eight = case["bits"] == 8
    g = s["g"].float()
    m = decode(s["m"], s["m_scale"], False) if eight else s["m"]
    v = decode(s["v"], s["v_scale"], True) if eight else s["v"]
    m = m * k["beta1"] + g * (1.0 - k["beta1"])
    v = v * k["beta2"] + (g * g) * (1.0 - k["beta2"])
    root = torch.sqrt(v) * (1.0 / math.sqrt(1.0 - k["beta2"] ** t)) + k["eps"]
    p = s["p"].float() * (1.0 - s["decay"] * k["lr"]) - m / root * (k["lr"] / (1.0 - k["beta1"] ** t))
    s["p"].copy_(p)
    if eight:
        for name, x in (("m", m), ("v", v)):
            codes, scale = encode(x, name == "v")
            s[name].copy_(codes)
            s[name + "_scale"].copy_(scale)
            s[name + "_out"].copy_(decode(codes, scale, name == "v"))
        return {"p": s["p"], "m": s["m_out"], "v": s["v_out"]}
    s["m"].copy_(m)
    s["v"].copy_(v)
    return {"p": s["p"], "m": s["m"], "v": s["v"]}


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    op = case["op"]
    if op == "adamw":
        s["step"] += 1
    if not own:
        return {"embedding": plain_embedding, "embedding_grad": plain_embedding_grad, "block_norm": plain_norm,
                "block_norm_grad": plain_norm_grad, "adamw": plain_adamw}[op](case, s)
    rt = runtime()
    if op == "embedding":
        rt.embedding(s["spec"])
        return {"y": s["y"]}
    if op == "embedding_grad":
        rt.embedding_grad(s["spec"])
        return {"dtable": s["dtable"]}
    if op == "block_norm":
        rt.block_norm(s["spec"])
        return {"h": s["h"], "y": s["y"]}
    if op == "block_norm_grad":
        rt.block_norm_grad(s["spec"])
        return {"dx": s["dx"], "db": s["db"], **{"d" + k: t for k, t in s["grads"].items()}}
    rt.adamw_step(s["plan"], step=s["step"], **HYPER)
    if case["bits"] == 32:
        return {"p": s["p"], "m": s["m"], "v": s["v"]}
    n = s["m"].numel()
    rt.adamw_decode(s["m_out"].data_ptr(), s["m"].data_ptr(), s["m_scale"].data_ptr(), n, second=False)
    rt.adamw_decode(s["v_out"].data_ptr(), s["v"].data_ptr(), s["v_scale"].data_ptr(), n, second=True)
    return {"p": s["p"], "m": s["m_out"], "v": s["v_out"]}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """What one pass returns for the inputs of this seed, from the operators' definitions in 64 bits.

    The states in 8 bits have no such value: their codes are defined by arithmetic in 32 bits, and a moment that lies within its
    rounding of the border of two codes gets the one or the other."""
    global own
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    wide = {k: t.double() for k, t in s.items() if isinstance(t, torch.Tensor) and t.is_floating_point()}
    return {"embedding": exact_embedding, "embedding_grad": exact_embedding_grad, "block_norm": exact_norm, "block_norm_grad": exact_norm_grad,
            "adamw": exact_adamw}[case["op"]](case, s, wide)


def exact_embedding(case, s, w):
    t = s["tokens"].long()
    y = w["table"].index_select(0, t).mul(case["scale"])
    return {"y": y.masked_fill_((t == s["pad"]).unsqueeze(1), 0.0)}


def exact_embedding_grad(case, s, w):
    # a column at a time would do; sums over tokens in order, by the differences of running sums over the sorted positions
    t = s["tokens"].long()
    keep = (t != s["pad"]).nonzero().reshape(-1)
    order = keep[torch.sort(t[keep], stable=True).indices]
    count = torch.bincount(t[keep], minlength=case["vocab"])
    ends = torch.cumsum(count, 0)
    out = torch.empty((case["vocab"], case["width"]), device="cuda", dtype=torch.float64)
    step = max(1, (1 << 26) // max(1, len(order)))
    for a in range(0, case["width"], step):
        part = w["dy"][:, a:a + step].index_select(0, order).cumsum(0)
        part = torch.cat([torch.zeros((1, part.shape[1]), device="cuda", dtype=torch.float64), part])
        out[:, a:a + step] = part[ends] - part[ends - count]
    out *= case["scale"]
    if case["accumulate"]:
        out += w["dtable"]
    return {"dtable": out}


def exact_stats(case, x):
    mean = x.mean(1, keepdim=True) if case["kind"] == "layer" else 0.0
    return mean, ((x - mean).square().mean(1, keepdim=True) + 1e-5).sqrt()


def exact_norm(case, s, w):
    n, d = case["rows"], case["width"]
    u = w["b"]
    if case["post"]:
        mean, dev = exact_stats(case, u)
        u = (u - mean) / dev * w["post_gain"] + w.get("post_bias", 0.0)
    if case["gate_rows"]:
        u = (u.reshape(n // case["gate_rows"], case["gate_rows"], d) * w["gate"][:, None, :]).reshape(n, d)
    h = w["x"] * case["alpha"] + u
    mean, dev = exact_stats(case, h)
    return {"h": h, "y": (h - mean) / dev * w["gain"] + w.get("bias", 0.0)}


def exact_back(case, x, dz):
    """d sum(dz * z) / dx for z = (x - mean) / dev with dev = sqrt(var + eps), from the derivative of dev alone."""
    mean, dev = exact_stats(case, x)
    c = x - mean
    dx = dz / dev - c * (dz * c).sum(1, keepdim=True) / (x.shape[1] * dev ** 3)
    return dx - (dz / dev).mean(1, keepdim=True) if case["kind"] == "layer" else dx


def exact_norm_grad(case, s, w):
    n, d, out = case["rows"], case["width"], {}
    mean, dev = exact_stats(case, w["h"])
    out["dgain"] = ((w["h"] - mean) / dev * w["dy"]).sum(0)
    if case["bias"]:
        out["dbias"] = w["dy"].sum(0)
    dh = exact_back(case, w["h"], w["dy"] * w["gain"]) + w["dh"]
    out["dx"] = dh * case["alpha"]
    z = w["b"]
    if case["post"]:
        mean, dev = exact_stats(case, w["b"])
        z = (w["b"] - mean) / dev
    if case["gate_rows"]:
        u = z * w["post_gain"] + w.get("post_bias", 0.0) if case["post"] else z
        shape = (n // case["gate_rows"], case["gate_rows"], d)
        out["dgate"] = (dh * u).reshape(shape).sum(1)
        dh = (dh.reshape(shape) * w["gate"][:, None, :]).reshape(n, d)
    if case["post"]:
        out["dpost_gain"] = (dh * z).sum(0)
        if case["bias"]:
            out["dpost_bias"] = dh.sum(0)
        dh = exact_back(case, w["b"], dh * w["post_gain"])
    out["db"] = dh
    return out


def exact_adamw(case, s, w):
    t, b1, b2 = s["step"] + 1, HYPER["beta1"], HYPER["beta2"]
    if case["bits"] == 8:
        m = (torch.sign(s["m"].double()) * (s["m"].double() / 127.0) ** 2).reshape(-1, BLOCK).mul(w["m_scale"][:, None]).reshape(-1)
        v = ((s["v"].double() / 255.0) ** 4).reshape(-1, BLOCK).mul(w["v_scale"][:, None]).reshape(-1)
    else:
        m, v = w["m"], w["v"]
    m = b1 * m + (1.0 - b1) * w["g"]
    v = b2 * v + (1.0 - b2) * w["g"] ** 2
    p = w["p"] - HYPER["lr"] * ((m / (1.0 - b1 ** t)) / ((v / (1.0 - b2 ** t)).sqrt() + HYPER["eps"]) + s["decay"].double() * w["p"])
    if case["bits"] == 8:
        return {"p": p, "m": None, "v": None}
    return {"p": p, "m": m, "v": v}
