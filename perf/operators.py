"""The 8-bit linear layer and the gradient norm / clipping: cases, plain forms and exact values.

Two paths of a sparse language model are covered. Training: the global norm of all gradients and their
clipping, between the backward pass and the optimizer. Inference: a finalised (2:4 pruned) linear layer whose
weight is held in 8-bit integers with a scale per output channel, and whose input rows are quantised on the fly
with a scale per token.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}
# [out, in] of the seven matrices of one decoder layer of the benchmark's layer set
LAYER = [(4096, 4096)] * 4 + [(11008, 4096)] * 2 + [(4096, 11008)]
LARGEST_PRODUCT = 8192 * 4096 * 11008
LARGEST_SET = 4


# ---------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------
def listed():
    def linear(name, rows, k, n, dtype="bf16", bias=False):
        return {"name": name, "op": "linear", "rows": rows, "in": k, "out": n, "dtype": dtype, "bias": bias}

    def grads(name, op, layout, count, dtype="bf16", out="bf16", p="2", clips=True):
        return {"name": name, "op": op, "layout": layout, "count": count, "dtype": dtype, "out": out, "p": p,
                "clips": clips}

    return [
        # one token of one sequence through an attention projection: the latency of a decode step
        linear("decode_1_attn", 1, 4096, 4096),
        # the same through the longest reduction of the layer set
        linear("decode_1_down", 1, 11008, 4096),
        # a small decode batch through the widest matrix
        linear("decode_16_gate", 16, 4096, 11008),
        # full precision activations, a bias, no size a multiple of anything: a small model's odd projection
        linear("odd_37_f32", 37, 1003, 1111, "f32", True),
        # a short prompt (or a large decode batch)
        linear("prompt_512_attn", 512, 4096, 4096, "bf16", True),
        # the benchmark's token batch through the widest matrix
        linear("prefill_8192_gate", 8192, 4096, 11008),
        # norm of the gradients of one decoder layer (bf16), and of many odd small fp32 tensors
        grads("norm_layer", "norm", "layers", 1),
        grads("norm_small_f32", "norm", "ragged", 150, "f32"),
        # clipping one decoder layer's gradients
        grads("clip_layer", "clip", "layers", 1),
        # biases, norms, small matrices of odd sizes: launch latency
        grads("clip_small", "clip", "ragged", 60, "bf16", "bf16"),
        # fp32 accumulators of several micro-steps, clipped into bf16 gradients
        grads("clip_f32_to_bf16", "clip", "layers", 1, "f32", "bf16"),
        # four decoder layers
        grads("clip_4_layers", "clip", "layers", LARGEST_SET),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "norm", "clip", "clip"])
    if kind == "linear":
        while True:
            rows, k, n = _log_int(rng, 1, 8192), _log_int(rng, 64, 12288), _log_int(rng, 64, 12288)
            if rng.random() < 0.5:
                k, n = (k + 15) // 16 * 16, (n + 15) // 16 * 16
            if rows * k * n <= LARGEST_PRODUCT:
                break
        return {"op": "linear", "rows": rows, "in": k, "out": n, "dtype": rng.choice(["bf16", "bf16", "bf16", "f32"]),
                "bias": rng.random() < 0.5}
    layout = rng.choice(["layers", "ragged", "ragged"])
    # a norm takes hundreds of tensors; clipping hands every one of them back, so its sets stay small
    count = rng.randint(1, LARGEST_SET - 1) if layout == "layers" else _log_int(rng, 1, 400 if kind == "norm" else 60)
    dtype = rng.choice(["bf16", "f32", "mixed"]) if layout == "ragged" else "bf16"
    return {"op": kind, "layout": layout, "count": count, "dtype": dtype, "out": rng.choice(["same", "bf16"]),
            "p": rng.choice(["2", "2", "inf"]), "clips": rng.random() < 0.75, "shape_seed": rng.randint(0, 1 << 30)}


def _shapes(case):
    """The tensors' shapes: whole decoder layers with their norm weights, or small tensors of odd sizes."""
    if case["layout"] == "layers":
        return (LAYER + [(4096,)] * 2) * case["count"]
    g = torch.Generator().manual_seed(int(case.get("shape_seed", 7)))
    logs = torch.rand(case["count"], generator=g) * math.log(200000.0)
    return [(max(1, int(math.exp(float(v)))),) for v in logs]


def _dtypes(case, count):
    if case["dtype"] == "mixed":
        ins = [torch.bfloat16 if i % 3 else torch.float32 for i in range(count)]
    else:
        ins = [DTYPES[case["dtype"]]] * count
    outs = ins if case["out"] == "same" else [DTYPES[case["out"]]] * count
    return ins, outs


# ---------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------
def _linear_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, k, n, dt = case["rows"], case["in"], case["out"], DTYPES[case["dtype"]]
    x = torch.randn(rows, k, device="cuda", generator=g)
    # a few input channels carry most of the range, as hidden states of language models do
    wide = torch.randint(0, k, (max(1, k // 512),), device="cuda", generator=g)
    x[:, wide] *= 12.0
    if rows > 8:
        x[rows // 2] = 0.0  # a padded position
    w = torch.randn(n, k, device="cuda", generator=g) * 0.02
    # finalised 2:4: the two smaller magnitudes of every whole group of four are zero
    whole = k // 4 * 4
    groups = w[:, :whole].reshape(n, whole // 4, 4)
    order = groups.abs().argsort(dim=2, descending=True, stable=True)
    groups.scatter_(2, order[:, :, 2:], 0.0)
    w[:, :whole] = groups.reshape(n, whole)
    bias = torch.randn(n, device="cuda", generator=g) * 0.1 if case["bias"] else None
    return x.to(dt), w.to(torch.bfloat16), None if bias is None else bias.to(dt)


def _grad_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shapes = _shapes(case)
    ins, outs = _dtypes(case, len(shapes))
    total = sum(math.prod(s) for s in shapes)
    grads = []
    for i, (shape, dt) in enumerate(zip(shapes, ins)):
        # layers' gradients differ in scale
        grads.append((torch.randn(shape, device="cuda", generator=g) * (1e-3 * (1 + i % 5))).to(dt))
    size = 3e-3 * math.sqrt(total) if case["p"] == "2" else 1.5e-2
    return grads, outs, size * (0.1 if case["clips"] else 4.0)


def prepare(case, seed):
    if case["op"] == "linear":
        x, w, bias = _linear_inputs(case, seed)
        # the layer's weight is quantised once, when the model is loaded
        if own:
            from sparseforge_b200 import ops

            wq, ws = ops.int8_quantize_rows(w)
        else:
            wq, ws = _quantize_plain(w)
        return {"op": "linear", "x": x, "wq": wq, "ws": ws, "bias": bias}
    grads, outs, max_norm = _grad_inputs(case, seed)
    # the clipped gradients go to buffers of their own: the raw ones stay for the next pass
    out = [torch.empty_like(g, dtype=dt) for g, dt in zip(grads, outs)] if case["op"] == "clip" else None
    return {"op": case["op"], "grads": grads, "out": out, "max_norm": max_norm,
            "p": math.inf if case["p"] == "inf" else 2.0}


# ---------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------
def _quantize_plain(x):
    """Symmetric 8-bit rows: scale max|x| / 127, values 127 x / max|x| rounded half to even. Values beside a
    half need more than 32 bits where x itself has 24."""
    wide = torch.float32 if x.dtype == torch.bfloat16 else torch.float64
    amax = x.abs().amax(dim=1)
    q = torch.round(x.to(wide) * 127.0 / torch.where(amax == 0, torch.ones_like(amax), amax).to(wide)[:, None])
    scale = amax.float() / torch.full_like(amax, 127.0, dtype=torch.float32)
    pad = -x.shape[1] % 16  # rows of whole 16-byte pieces
    return torch.nn.functional.pad(q.to(torch.int8), (0, pad)), scale


def _linear_plain(x, wq, ws, bias):
    xq, xs = _quantize_plain(x)
    y = (xq.float() @ wq.float().t()) * xs[:, None] * ws
    if bias is not None:
        y = y + bias.float()
    return y.to(x.dtype)


def _norm_plain(grads, p):
    if p == math.inf:
        return torch.stack([g.float().abs().amax() for g in grads]).amax()
    return torch.stack([(g.float() * g.float()).sum() for g in grads]).sum().sqrt()


def run(state):
    if state["op"] == "linear":
        if own:
            from sparseforge_b200 import ops

            return ops.int8_linear(state["x"], state["wq"], state["ws"], state["bias"])
        return _linear_plain(state["x"], state["wq"], state["ws"], state["bias"])
    if own:
        from sparseforge_b200 import ops

        if state["op"] == "norm":
            return ops.grad_norm(state["grads"], state["p"])
        return [ops.clip_grad_norm(state["grads"], state["max_norm"], state["p"], out=state["out"])] + state["out"]
    norm = _norm_plain(state["grads"], state["p"])
    if state["op"] == "norm":
        return norm
    coef = torch.clamp(state["max_norm"] / (norm + 1e-6), max=1.0)
    for g, o in zip(state["grads"], state["out"]):
        o.copy_(g.float() * coef)
    return [norm] + state["out"]


# ---------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "linear":
        rows, k, n, b = case["rows"], case["in"], case["out"], BYTES[case["dtype"]]
        return {"bytes": rows * k * b + n * k + 4 * n + rows * n * b + (n * b if case["bias"] else 0),
                "flops": 2 * rows * k * n}
    shapes = _shapes(case)
    ins, outs = _dtypes(case, len(shapes))
    sizes = [math.prod(s) for s in shapes]
    read = sum(n * (2 if d == torch.bfloat16 else 4) for n, d in zip(sizes, ins))
    if case["op"] == "norm":
        return {"bytes": read + 4, "flops": 2 * sum(sizes)}
    return {"bytes": read + 4 + sum(n * (2 if d == torch.bfloat16 else 4) for n, d in zip(sizes, outs)),
            "flops": 3 * sum(sizes)}


# ---------------------------------------------------------------------------------------------------------
# from the definition, in 64 bits
# ---------------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "linear":
        x, w, bias = _linear_inputs(case, seed)

        def rows_in_8_bits(t):
            t = t.double()
            top = t.abs().max(dim=1, keepdim=True).values
            steps = torch.where(top > 0, t * 127.0 / top, torch.zeros_like(t)).round()
            return steps, top / 127.0

        xi, xs = rows_in_8_bits(x)
        wi, ws = rows_in_8_bits(w)
        y = torch.matmul(xi, wi.t()).mul_(xs).mul_(ws.t())
        return y if bias is None else y.add_(bias.double())
    grads, _, max_norm = _grad_inputs(case, seed)
    if case["p"] == "inf":
        norm = max(float(g.double().abs().max()) for g in grads)
    else:
        norm = math.sqrt(math.fsum(float(g.double().pow(2).sum()) for g in grads))
    value = torch.tensor(norm, dtype=torch.float64, device="cuda")
    if case["op"] == "norm":
        return value
    factor = min(1.0, max_norm / (norm + 1e-6))
    return [value] + [g.double() * factor for g in grads]
