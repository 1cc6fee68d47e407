"""Measured cases of the operators on learned tensors.

Three operators: the relative position bias expanded from a learned table of
buckets, the gradient of that table, and the orthogonalisation of a dense
matrix by Newton-Schulz products.  `run` computes a case in plain torch
operations, or, with `own` set, by the calls of this package that a user makes.
"""
import math

import torch

own = False

DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "f64": torch.float64}
SIZE = {"f16": 2, "bf16": 2, "f32": 4, "f64": 8}
# The quintic iteration whose singular values settle around one in five steps.
COEF = (3.4445, -4.7750, 2.0315)
EPS = 1e-7


def listed():
    return [
        # One new token of one sequence: a single row of the bias, the keys behind it.
        bias("bias_one_token", "bf16", 32, 1, 2048, first=2047, both=False, causal=True),
        # An encoder's bias at a training length, in the table's own type.
        bias("bias_encoder", "f32", 12, 512, 512, both=True),
        # One new token each of many sequences at positions of their own.
        bias("bias_tokens_of_many", "bf16", 32, 250, 8192, both=False, causal=True, scattered=True),
        # A decoder's whole prompt with the causal mask written into the bias, odd length in padded rows.
        bias("bias_prompt", "bf16", 32, 4001, 4001, both=False, causal=True, pad=7),
        # A first small fine-tuning batch.
        grad("grad_small", "f32", 8, 1, 128, 128, both=True),
        # An encoder's training batch: the bias is shared by the batch, its gradient is the sum.
        grad("grad_encoder_batch", "bf16", 12, 8, 512, 512, both=True),
        # A decoder trained on long sequences.
        grad("grad_decoder_long", "f16", 16, 2, 4001, 4001, both=False, causal=True),
        # One small square weight: latency.
        orth("orth_small", "f32", 1, 96, 96),
        # The heads' slices of one projection, taken one by one.
        orth("orth_heads", "bf16", 32, 128, 1000),
        # A projection of a wide layer.
        orth("orth_wide", "bf16", 1, 1024, 4096),
        # A tall matrix in f32.
        orth("orth_tall", "f32", 1, 8192, 2048),
        # A large square weight.
        orth("orth_square", "bf16", 1, 4096, 4096),
    ]


def bias(name, dtype, heads, queries, keys, first=0, both=True, causal=False, scattered=False, pad=0, buckets=32,
         distance=128):
    return {"name": name, "op": "bias", "dtype": dtype, "heads": heads, "batch": 1, "queries": queries, "keys": keys,
            "first": first, "both": both, "causal": causal, "scattered": scattered, "pad": pad, "buckets": buckets,
            "distance": distance}


def grad(name, dtype, heads, batch, queries, keys, first=0, both=True, causal=False, scattered=False, pad=0, buckets=32,
         distance=128):
    return {"name": name, "op": "grad", "dtype": dtype, "heads": heads, "batch": batch, "queries": queries,
            "keys": keys, "first": first, "both": both, "causal": causal, "scattered": scattered, "pad": pad,
            "buckets": buckets, "distance": distance}


def orth(name, dtype, batch, rows, cols, steps=5):
    return {"name": name, "op": "orth", "dtype": dtype, "batch": batch, "rows": rows, "cols": cols, "steps": steps}


def draw(rng):
    def size(low, high):
        return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))

    op = rng.choice(["bias", "grad", "orth"])
    if op == "orth":
        rows, cols = size(16, 4096), size(16, 4096)
        m, n = min(rows, cols), max(rows, cols)
        batch = min(size(1, 32), max(1, (1 << 33) // (m * m * n)))
        case = orth("", rng.choice(["f16", "bf16", "f32"]), batch, rows, cols, rng.randint(3, 6) if m < 3500 else 5)
    else:
        heads, batch = size(1, 32), 1 if op == "bias" else size(1, 8)
        keys = size(16, 8192)
        queries = 1 if op == "bias" and rng.random() < 0.2 else size(2, 4096)
        while heads * batch * queries * keys > 1 << 28:
            heads, batch, queries = max(1, heads // 2), max(1, batch // 2), max(1, queries * 2 // 3)
        both = rng.random() < 0.5
        scattered = rng.random() < 0.3
        first = 0 if scattered or rng.random() < 0.5 else max(0, keys - queries)
        case = (bias if op == "bias" else grad)(
            "", rng.choice(["f16", "bf16", "f32"]), heads, *([] if op == "bias" else [batch]), queries, keys,
            first=first, both=both, causal=not both or rng.random() < 0.2, scattered=scattered,
            pad=rng.choice([0, 0, 3, 8]), buckets=rng.choice([8, 16, 32, 64]), distance=rng.choice([64, 128, 200, 1000]))
    del case["name"]
    return case


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    dtype = DTYPE[case["dtype"]]
    if case["op"] == "orth":
        batch, rows, cols = case["batch"], case["rows"], case["cols"]
        # A gradient: a few strong directions over noise.
        few = min(8, rows, cols)
        x = torch.randn(batch, rows, cols, device="cuda", generator=gen)
        x += 0.5 * torch.randn(batch, rows, few, device="cuda", generator=gen) @ torch.randn(
            batch, few, cols, device="cuda", generator=gen)
        state["x"] = (x * 1e-3).to(dtype)
        state["out"] = torch.empty_like(state["x"])
        if own:
            import mlirpass_b200 as dcf
            plan = dcf.orthogonalize_plan(case["dtype"], rows, cols, batch=batch, steps=case["steps"], coef=COEF, eps=EPS)
            state["plan"] = plan
            state["work"] = torch.empty(dcf.orthogonalize_workspace(plan), dtype=torch.uint8, device="cuda")
            state["status"] = torch.empty(2, dtype=torch.int64, device="cuda")
            dcf.status_reset(state["status"])
        return state
    heads, queries, keys, width = case["heads"], case["queries"], case["keys"], case["keys"] + case["pad"]
    positions = None
    if case["scattered"]:
        positions = torch.randint(0, keys, (queries,), device="cuda", generator=gen, dtype=torch.int32)
    state["positions"] = positions
    if case["op"] == "bias":
        state["table"] = (0.5 * torch.randn(case["buckets"], heads, device="cuda", generator=gen)).to(dtype)
        state["out"] = torch.empty(heads, queries, width, device="cuda", dtype=dtype)[:, :, :keys]
    else:
        g = torch.randn(case["batch"], heads, queries, width, device="cuda", generator=gen, dtype=torch.float32)
        state["grad"] = (g * 1e-2).to(dtype)[..., :keys]
        # The loss falls off along a direction of its own: sums that do not cancel to nothing.
        state["grad"] += 1e-3
        if case["causal"]:
            state["grad"].masked_fill_(_distance(case, positions) > 0, 0)
        state["out"] = torch.empty(case["buckets"], heads, device="cuda", dtype=torch.float32)
    if own:
        import mlirpass_b200 as dcf
        plan = dcf.position_bias_plan(
            case["dtype"], heads, queries, keys, num_buckets=case["buckets"], max_distance=case["distance"],
            bidirectional=case["both"], causal=case["causal"], first_query=case["first"], batch=case["batch"],
            row_stride=width, head_stride=queries * width, batch_stride=heads * queries * width)
        state["plan"] = plan
        if case["op"] == "grad":
            state["work"] = torch.empty(dcf.position_bias_grad_workspace(plan), dtype=torch.uint8, device="cuda")
    return state


def run(state):
    case = state["case"]
    if own:
        import mlirpass_b200 as dcf
        if case["op"] == "orth":
            dcf.orthogonalize_async(state["plan"], state["x"], state["out"], state["work"], state["status"])
        elif case["op"] == "bias":
            dcf.position_bias_async(state["plan"], state["table"], state["out"], positions=state["positions"])
        else:
            dcf.position_bias_grad_async(state["plan"], state["grad"], state["out"], state["work"],
                                         positions=state["positions"])
        return state["out"]
    if case["op"] == "orth":
        return _orth_plain(case, state["x"])
    distance = _distance(case, state["positions"])
    bucket = _bucket_plain(case, distance)
    if case["op"] == "bias":
        out = state["table"][bucket].permute(2, 0, 1)
        if case["causal"]:
            out = out.masked_fill(distance > 0, -math.inf)
        return out.contiguous()
    g = state["grad"].float()
    if case["causal"]:
        g = torch.where(distance > 0, torch.zeros((), device="cuda"), g)
    g = g.sum(0).reshape(case["heads"], -1)
    hot = (bucket.reshape(-1, 1) == torch.arange(case["buckets"], device="cuda")).float()
    return hot.T @ g.T


def work(case):
    if case["op"] == "orth":
        m, n = min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
        # X X^T and A A are symmetric: half of each is the work; then B X.
        flops = case["batch"] * case["steps"] * (m * m * n + m * m * m + 2 * m * m * n)
        return {"bytes": 2 * case["batch"] * m * n * SIZE[case["dtype"]], "flops": flops}
    q, k, first = case["queries"], case["keys"], case["first"]
    seen = q * k
    if case["op"] == "grad" and case["causal"]:
        # What lies after the query is not read.
        seen = q * (k + 1) // 2 if case["scattered"] else sum(min(k, first + i + 1) for i in range(q))
    table = case["buckets"] * case["heads"] * (SIZE[case["dtype"]] if case["op"] == "bias" else 4)
    moved = seen * case["heads"] * case["batch"] * SIZE[case["dtype"]]
    return {"bytes": moved + table + (4 * q if case["scattered"] else 0),
            "flops": 0 if case["op"] == "bias" else seen * case["heads"] * case["batch"]}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "orth":
        x = state["x"].double()
        wide = x if case["rows"] <= case["cols"] else x.transpose(1, 2)
        a, b, c = COEF
        y = wide / (torch.linalg.vector_norm(wide, dim=(1, 2), keepdim=True) + EPS)
        for _ in range(case["steps"]):
            gram = torch.bmm(y, y.transpose(1, 2))
            square = torch.bmm(gram, gram)
            y = torch.baddbmm(y, gram.mul(b).add_(square, alpha=c), y, beta=a)
        return y if case["rows"] <= case["cols"] else y.transpose(1, 2)
    # Buckets from whole numbers: the first distance of each far bucket, by integer powers.
    half = case["buckets"] // 2 if case["both"] else case["buckets"]
    near, last = half // 2, case["distance"]
    starts, n, far = [], near, half - near
    for k in range(1, far):
        while n ** far * near ** k < last ** k * near ** far:
            n += 1
        starts.append(n)
    edges = torch.tensor(list(range(1, near + 1)) + starts, device="cuda")
    rows = case["first"] + torch.arange(case["queries"], device="cuda")
    if state["positions"] is not None:
        rows = state["positions"].long()
    ahead = torch.arange(case["keys"], device="cuda")[None, :] - rows[:, None]
    length = ahead.abs() if case["both"] else (-ahead).clamp(min=0)
    bucket = torch.searchsorted(edges, length, right=True) + (half * (ahead > 0) if case["both"] else 0)
    if case["op"] == "bias":
        out = torch.stack([column[bucket] for column in state["table"].double().T])
        return out.masked_fill_(ahead > 0, -math.inf) if case["causal"] else out
    out = torch.zeros(case["buckets"], case["heads"], device="cuda", dtype=torch.float64)
    seen = (ahead <= 0) if case["causal"] else torch.ones_like(ahead, dtype=torch.bool)
    for h in range(case["heads"]):
        g = state["grad"][:, h].double().sum(0)
        for v in range(case["buckets"]):
            out[v, h] = g[(bucket == v) & seen].sum() if v < 2 * half else 0
    return out


def _distance(case, positions):
    """Key position minus query position, [queries, keys]."""
    rows = case["first"] + torch.arange(case["queries"], device="cuda")
    if positions is not None:
        rows = positions.long()
    return torch.arange(case["keys"], device="cuda") - rows[:, None]


def _bucket_plain(case, distance):
    if case["both"]:
        half = case["buckets"] // 2
        base = torch.where(distance > 0, half, 0)
        length = distance.abs()
    else:
        half, base = case["buckets"], 0
        length = (-distance).clamp(min=0)
    near = half // 2
    # 64 bits, and a nudge of a few roundings: a distance that starts a bucket belongs to it.
    steps = (length.clamp(min=1).double() / near).log() * ((half - near) / math.log(case["distance"] / near))
    far = (near + (steps * (1 + 1e-14)).floor().long()).clamp(max=half - 1)
    return base + torch.where(length < near, length, far)


def _orth_plain(case, x):
    a, b, c = COEF
    y = x.float()
    if case["rows"] > case["cols"]:
        y = y.transpose(1, 2)
    y = y / (y.square().sum((1, 2), keepdim=True).sqrt() + EPS)
    for _ in range(case["steps"]):
        gram = y @ y.transpose(1, 2)
        y = a * y + (b * gram + c * (gram @ gram)) @ y
    if case["rows"] > case["cols"]:
        y = y.transpose(1, 2)
    return y.to(x.dtype).contiguous()
