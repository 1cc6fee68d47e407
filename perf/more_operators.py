"""Measured cases of the operators on 8-bit integers.

Four operators: quantising a matrix to 8-bit integers with a scale for each row
and reading it back, the same with a scale for each column of each run of 128
rows (a checkpoint of activations), the product of 8-bit matrices with scales
for each token and channel, and the weight gradient from a checkpoint.  `run`
computes a case in plain torch operations, or, with `own` set, by the calls of
this package that a user makes.
"""
import math

import torch

own = False

DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "i32": torch.int32}
SIZE = {"i8": 1, "f16": 2, "bf16": 2, "f32": 4, "i32": 4}
RUN = 128  # rows that share a column's scale
LEAST = 2.0 ** -119  # what is smaller throughout stands for zeros


def listed():
    return [
        # One new token's activations: a single row.
        quant("rows_token", "bf16", 1, 4096),
        # The weight of a wide layer in the optimizer's type, a scale for each output channel.
        quant("rows_weight", "f32", 8192, 4096),
        # The activations that a small layer keeps, odd sizes in padded rows.
        quant("checkpoint_ragged", "f16", 1000, 1531, columns=True, pad=5),
        # The activations that a training step keeps for its backward pass.
        quant("checkpoint_batch", "bf16", 8192, 4096, columns=True),
        # One new token through a projection.
        matmul("matmul_token", "bf16", 1, 4096, 4096, "bf16"),
        # One new token each of 48 sequences, up to a wide layer.
        matmul("matmul_decode", "bf16", 48, 16384, 4096, "bf16"),
        # A small product of whole numbers, as a module of 8-bit constants holds it.
        matmul("matmul_sums", "i8", 500, 512, 1024, "i32"),
        # A prompt of odd length through a layer of odd sizes.
        matmul("matmul_ragged", "f16", 1001, 2047, 1531, "f32"),
        # A long prompt whose activations were quantised before.
        matmul("matmul_prompt", "i8", 4096, 4096, 4096, "bf16", bias=True),
        # A first small fine-tuning batch.
        grad("grad_small", "bf16", 200, 256, 512, "f32"),
        # A ragged batch of a small layer.
        grad("grad_ragged", "f16", 4001, 1000, 1531, "f16", pad=5),
        # A training step's tokens and a square projection.
        grad("grad_batch", "bf16", 8192, 4096, 4096, "f32"),
    ]


def quant(name, dtype, rows, cols, columns=False, pad=0):
    return {"name": name, "op": "quant", "dtype": dtype, "rows": rows, "cols": cols, "columns": columns, "pad": pad}


def matmul(name, dtype, tokens, channels, depth, out, bias=False, pad=0):
    return {"name": name, "op": "matmul", "dtype": dtype, "tokens": tokens, "channels": channels, "depth": depth,
            "out": out, "bias": bias, "pad": pad}


def grad(name, dtype, tokens, channels, depth, out, pad=0):
    return {"name": name, "op": "grad", "dtype": dtype, "tokens": tokens, "channels": channels, "depth": depth,
            "out": out, "pad": pad}


def draw(rng):
    def size(low, high):
        return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))

    def whole(n):
        # Half of the sizes are whole vectors, as most layers' are.
        return n if n < 64 or rng.random() < 0.5 else n // 64 * 64

    op = rng.choice(["quant", "matmul", "grad"])
    pad = rng.choice([0, 0, 0, 3, 16])
    if op == "quant":
        rows, cols = size(1, 16384), whole(size(16, 16384))
        rows = max(1, min(rows, (1 << 25) // cols))
        case = quant("", rng.choice(["f16", "bf16", "f32"]), rows, cols, rng.random() < 0.5, pad)
    elif op == "matmul":
        tokens, channels, depth = size(1, 4096), whole(size(16, 16384)), whole(size(16, 8192))
        tokens = max(1, min(tokens, (1 << 36) // (channels * depth)))
        out = rng.choice(["f16", "bf16", "f32", "i32"])
        dtype = "i8" if out == "i32" else rng.choice(["i8", "f16", "bf16", "f32"])
        case = matmul("", dtype, tokens, channels, depth, out, out != "i32" and rng.random() < 0.3, pad)
    else:
        tokens, channels, depth = size(1, 8192), whole(size(16, 4096)), whole(size(16, 4096))
        case = grad("", rng.choice(["f16", "bf16"]), tokens, channels, depth, rng.choice(["f16", "bf16", "f32", "f32"]), pad)
    del case["name"]
    return case


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    def activations(rows, cols):
        # Some channels carry more than others; tokens that pad a batch are zeros.
        x = normal(rows, cols) * (0.7 * normal(cols)).exp()
        if rows > 8:
            x[rows * 2 // 3:rows * 2 // 3 + rows // 50 + 1] = 0
        return x

    def padded(x, dtype):
        room = torch.zeros(x.shape[0], x.shape[1] + case["pad"], device="cuda", dtype=dtype)
        room[:, :x.shape[1]] = x
        return room[:, :x.shape[1]]

    def empty(rows, cols, dtype):
        return torch.empty(rows, cols + case["pad"], device="cuda", dtype=dtype)[:, :cols]

    if own:
        import mlirpass_b200 as dcf
        state["status"] = torch.empty(2, dtype=torch.int64, device="cuda")
        dcf.status_reset(state["status"])
    if case["op"] == "quant":
        rows, cols = case["rows"], case["cols"]
        x = activations(rows, cols) if case["columns"] or rows < 64 else 0.02 * normal(rows, cols) * (
            0.3 * normal(rows, 1)).exp()
        state["x"] = padded(x, DTYPE[case["dtype"]])
        if own:
            stride = cols + case["pad"]
            state["plan"] = dcf.quantize_plan(case["dtype"], rows, cols, along="columns" if case["columns"] else "rows",
                                              row_stride=stride, q_row_stride=stride)
            state["q"] = empty(rows, cols, torch.int8)
            state["scale"] = torch.empty(*((-(-rows // RUN), cols) if case["columns"] else (rows,)), device="cuda")
            state["values"] = empty(rows, cols, DTYPE[case["dtype"]])
        return state
    tokens, channels, depth = case["tokens"], case["channels"], case["depth"]
    if case["op"] == "matmul":
        # Weights and their scales as a program holds them.
        state["b"] = padded((40 * normal(channels, depth)).round().clamp(-127, 127), torch.int8)
        state["bias"] = 0.1 * normal(channels) if case["bias"] else None
        if case["out"] != "i32":
            state["b_scale"] = 5e-4 * (0.3 * normal(channels)).exp()
        if case["dtype"] == "i8":
            state["a"] = padded((30 * normal(tokens, depth)).round().clamp(-127, 127), torch.int8)
            if case["out"] != "i32":
                state["a_scale"] = 0.03 * (0.5 * normal(tokens)).exp()
        else:
            state["a"] = padded(activations(tokens, depth), DTYPE[case["dtype"]])
        if own:
            stride = depth + case["pad"]
            plan = dcf.int8_matmul_plan(tokens, channels, depth, a_dtype=case["dtype"], out_dtype=case["out"],
                                        a_row_stride=stride, b_row_stride=stride, out_row_stride=channels + case["pad"])
            state["plan"] = plan
            state["work"] = torch.empty(dcf.int8_matmul_workspace(plan), dtype=torch.uint8, device="cuda")
            state["out"] = empty(tokens, channels, DTYPE[case["out"]])
        return state
    # The checkpoint of a layer's input, and the gradient of its output: small, with a few strong tokens.
    rows = -(-tokens // RUN)
    state["q"] = padded((40 * normal(tokens, depth)).round().clamp(-127, 127), torch.int8)
    state["scale"] = 0.02 * (0.7 * normal(depth)).exp() * (0.2 * normal(rows, depth)).exp()
    state["grad"] = padded(1e-2 * normal(tokens, channels) * normal(tokens, 1).exp(), DTYPE[case["dtype"]])
    if own:
        plan = dcf.checkpoint_grad_plan(case["dtype"], tokens, channels, depth, out_dtype=case["out"],
                                        grad_row_stride=channels + case["pad"], q_row_stride=depth + case["pad"],
                                        out_row_stride=depth + case["pad"])
        state["plan"] = plan
        state["work"] = torch.empty(dcf.checkpoint_grad_workspace(plan), dtype=torch.uint8, device="cuda")
        state["out"] = empty(channels, depth, DTYPE[case["out"]])
    return state


def run(state):
    case = state["case"]
    if own:
        import mlirpass_b200 as dcf
        if case["op"] == "quant":
            dcf.quantize_async(state["plan"], state["x"], state["q"], state["scale"])
            dcf.dequantize_async(state["plan"], state["q"], state["scale"], state["values"])
            return {"values": state["values"], "scale": state["scale"]}
        if case["op"] == "matmul":
            dcf.int8_matmul_async(state["plan"], state["a"], state["b"], state["out"], state["work"], state["status"],
                                  a_scale=state.get("a_scale"), b_scale=state.get("b_scale"), bias=state["bias"])
        else:
            dcf.checkpoint_grad_async(state["plan"], state["grad"], state["q"], state["scale"], state["out"],
                                      state["work"], state["status"])
        return state["out"]
    if case["op"] == "quant":
        x = state["x"].float()
        rows, cols = x.shape
        runs = -(-rows // RUN)
        if case["columns"]:
            x = torch.nn.functional.pad(x, (0, 0, 0, runs * RUN - rows)).reshape(runs, RUN, cols)
        q, scale = _quantize_plain(x, 1)
        values = (q * scale).reshape(-1, cols)[:rows].to(DTYPE[case["dtype"]])
        return {"values": values, "scale": scale.reshape(runs, cols) if case["columns"] else scale.reshape(rows)}
    if case["op"] == "matmul":
        if case["dtype"] == "i8":
            a, a_scale = state["a"].float(), state.get("a_scale")
        else:
            a, a_scale = _quantize_plain(state["a"].float(), 1)
        if case["out"] == "i32":
            # Whole numbers past 24 bits need the longer sums.
            return (a.double() @ state["b"].double().T).to(torch.int32)
        out = (a @ state["b"].float().T) * a_scale.reshape(-1, 1) * state["b_scale"]
        if state["bias"] is not None:
            out = out + state["bias"]
        return out.to(DTYPE[case["out"]])
    scale = state["scale"].repeat_interleave(RUN, 0)[:case["tokens"]]
    return (state["grad"].float().T @ (state["q"].float() * scale)).to(DTYPE[case["out"]])


def work(case):
    if case["op"] == "quant":
        rows, cols = case["rows"], case["cols"]
        scales = -(-rows // RUN) * cols if case["columns"] else rows
        # Values read, whole numbers written and read, values written; the scales the same.
        return {"bytes": 2 * rows * cols * (SIZE[case["dtype"]] + 1) + 8 * scales, "flops": 3 * rows * cols}
    t, c, d = case["tokens"], case["channels"], case["depth"]
    if case["op"] == "matmul":
        scales = 0 if case["out"] == "i32" else 4 * (c + (t if case["dtype"] == "i8" else 0) + (c if case["bias"] else 0))
        return {"bytes": t * d * SIZE[case["dtype"]] + c * d + t * c * SIZE[case["out"]] + scales, "flops": 2 * t * c * d}
    return {"bytes": 2 * t * c + t * d + 4 * d * -(-t // RUN) + c * d * SIZE[case["out"]], "flops": 2 * t * c * d}


def exact(case, seed):
    state = prepare(case, seed)

    def levels(x, top):
        """Whole numbers of each value, where `top` is the largest magnitude beside it."""
        seen = (top >= LEAST) & torch.isfinite(top)
        factor = torch.where(seen, (127 / top).float().double(), torch.zeros_like(top))
        return torch.special.round(x * factor), torch.where(torch.isfinite(top), seen * (top / 127).float().double(), math.nan)

    if case["op"] == "quant":
        x = state["x"].double()
        if not case["columns"]:
            q, scale = levels(x, x.abs().amax(1, keepdim=True))
            return {"values": q * scale, "scale": scale[:, 0]}
        parts = [levels(part, part.abs().amax(0, keepdim=True)) for part in x.split(RUN)]
        return {"values": torch.cat([q * scale for q, scale in parts]), "scale": torch.cat([scale for _, scale in parts])}
    if case["op"] == "matmul":
        a = state["a"].double()
        if case["dtype"] != "i8":
            q, scale = levels(a, a.abs().amax(1, keepdim=True))
            a = q * scale
        elif case["out"] == "i32":
            return torch.mm(a, state["b"].double().t()).long()
        else:
            a = a * state["a_scale"].double()[:, None]
        out = torch.mm(a, (state["b"].double() * state["b_scale"].double()[:, None]).t())
        return out if state["bias"] is None else out + state["bias"].double()
    out = torch.zeros(case["channels"], case["depth"], device="cuda", dtype=torch.float64)
    for i, (g, q) in enumerate(zip(state["grad"].split(RUN), state["q"].split(RUN))):
        out.addmm_(g.double().t(), q.double() * state["scale"][i].double())
    return out


def _quantize_plain(x, dim):
    """Whole numbers and scales along a dim."""
    top = x.abs().amax(dim, keepdim=True)
    most = torch.full_like(top, 127)
    some, fine = top >= LEAST, torch.isfinite(top)
    factor = torch.where(some & fine, most / top, torch.zeros_like(top))
    scale = torch.where(some, top / most, torch.zeros_like(top))
    # 64 bits: the product of two 32-bit values is exact, and rounded once.
    q = torch.where(fine, (x.double() * factor.double()).round().float(), torch.zeros_like(x))
    return q, torch.where(fine, scale, torch.full_like(scale, math.nan))
