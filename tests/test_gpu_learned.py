"""The operators on learned tensors on the GPU against 64-bit statements."""
import numpy as np
import pytest

import learned_oracle as lo

pytestmark = pytest.mark.gpu

WIDE = {"f16": np.float16, "f32": np.float32, "f64": np.float64}


def tdtype(name):
    import torch
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "f64": torch.float64}[name]


def values(t) -> np.ndarray:
    return t.double().cpu().numpy()


def randn(shape, dtype, seed, scale=1.0):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=gen, dtype=torch.float64) * scale).to(tdtype(dtype))


# ------------------------------------------------------------------ bias


def bias_want(table, ids, hidden):
    want = table.T[:, ids]
    return np.where(hidden, -np.inf, want) if hidden is not None else want


def run_bias(dcf, table, dtype, heads, queries, keys, *, given=None, table_dtype=None, fill=7.0, **kw):
    import torch
    plan = dcf.position_bias_plan(dtype, heads, queries, keys, table_dtype=table_dtype, **kw)
    flat = torch.full((plan.out_elements + 3,), fill, dtype=tdtype(dtype), device="cuda")
    pos = torch.tensor(given, dtype=torch.int32, device="cuda") if given is not None else None
    dcf.position_bias_async(plan, table, flat, positions=pos)
    torch.cuda.synchronize()
    d = plan.desc
    row = d.row_stride or keys
    head = d.head_stride or queries * row
    assert (flat[plan.out_elements:] == fill).all()      # nothing behind the last row
    return flat.as_strided((heads, queries, keys), (head, row, 1)), flat


SIZES = [(1, 1), (1, 7), (1, 300), (2, 1), (5, 8), (9, 31), (33, 64), (64, 129), (130, 257)]


@pytest.mark.parametrize("queries,keys", SIZES)
@pytest.mark.parametrize("both,causal", [(True, False), (False, True), (False, False), (True, True)])
@pytest.mark.parametrize("dtype", ["bf16", "f32", "f16", "f64"])
def test_bias_sizes(dcf, queries, keys, both, causal, dtype):
    heads = 3
    table = randn((32, heads), dtype, 1)
    first = keys - queries if causal else 0
    got, _ = run_bias(dcf, table, dtype, heads, queries, keys, bidirectional=both, causal=causal, first_query=first)
    q = lo.positions(queries, first)
    ids = lo.buckets(q, keys, 32, 128, both)
    want = bias_want(values(table), ids, lo.masked(q, keys) if causal else None)
    assert np.array_equal(values(got), want)


@pytest.mark.parametrize("num_buckets,max_distance,both", [
    (1, 1, False), (2, 2, False), (2, 1, True), (3, 2, False), (4, 2, True), (5, 3, False), (7, 5, True),
    (8, 64, True), (16, 1000, False), (32, 128, True), (32, 128, False), (33, 200, True), (64, 33, True),
    (128, 1 << 20, False), (256, 2000, False), (256, (1 << 31) - 1, False), (255, 128, False), (32, 256, True),
    (32, 512, False), (48, 4096, True)])
def test_bias_every_border(dcf, num_buckets, max_distance, both):
    """A table of its own row numbers returns the buckets themselves."""
    import torch
    table = torch.arange(num_buckets, dtype=torch.float32, device="cuda").reshape(-1, 1)
    keys, mid = 5000, 2500
    far = [mid, 0, keys - 1, -1, -(1 << 30), (1 << 31) - 1, -(1 << 31), max_distance, max_distance - mid]
    far = [min(max(f, -(1 << 31)), (1 << 31) - 1) for f in far]
    got, _ = run_bias(dcf, table, "f32", 1, len(far), keys, given=far, num_buckets=num_buckets,
                      max_distance=max_distance, bidirectional=both)
    assert np.array_equal(values(got)[0], lo.buckets(far, keys, num_buckets, max_distance, both))


@pytest.mark.parametrize("dtype", ["bf16", "f64"])
@pytest.mark.parametrize("row,head,off", [(40, 0, 0), (37, 0, 0), (38, 5 * 38 + 3, 0), (3 * 37, 37, 0), (131, 41, 1),
                                          (64, 1024, 5)])
def test_bias_strides_alignments_and_what_lies_between(dcf, dtype, row, head, off):
    import torch
    heads, queries, keys = 3, 5, 37
    table = randn((32, heads), dtype, 2)
    plan = dcf.position_bias_plan(dtype, heads, queries, keys, row_stride=row, head_stride=head, bidirectional=False,
                                  causal=True, first_query=20)
    h = head or queries * row
    flat = torch.full((plan.out_elements + off + 9,), 3.0, dtype=tdtype(dtype), device="cuda")
    dcf.position_bias_async(plan, table, flat[off:])
    got = flat[off:].as_strided((heads, queries, keys), (h, row, 1))
    q = lo.positions(queries, 20)
    want = bias_want(values(table), lo.buckets(q, keys, 32, 128, False), lo.masked(q, keys))
    assert np.array_equal(values(got), want)
    got.fill_(3.0)
    assert (flat == 3.0).all()


def test_bias_positions_of_their_own_and_rows_with_no_key(dcf):
    heads, keys = 4, 100
    given = [0, 99, 50, 50, -1, 1000, -(1 << 31), 7]
    table = randn((32, heads), "bf16", 3)
    got, _ = run_bias(dcf, table, "bf16", heads, len(given), keys, given=given, bidirectional=False, causal=True)
    ids = lo.buckets(given, keys, 32, 128, False)
    hidden = lo.masked(given, keys)
    assert hidden[4].all() and hidden[6].all()
    assert np.array_equal(values(got), bias_want(values(table), ids, hidden))


def test_bias_far_first_query(dcf):
    table = randn((32, 2), "f32", 4)
    for first in (1 << 40, -(1 << 40), (1 << 31) + 5):
        got, _ = run_bias(dcf, table, "f32", 2, 3, 20, first_query=first)
        q = lo.positions(3, first)
        assert np.array_equal(values(got), bias_want(values(table), lo.buckets(q, 20, 32, 128, True), None))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_bias_from_a_f32_table_rounds_once(dcf, dtype):
    import torch
    table = randn((32, 5), "f32", 5)
    table[0, 0], table[1, 0], table[2, 1], table[3, 2] = float("nan"), float("inf"), 1e-40, 70000.0
    got, _ = run_bias(dcf, table, dtype, 5, 40, 50, table_dtype="f32")
    ids = torch.from_numpy(lo.buckets(lo.positions(40, 0), 50, 32, 128, True)).cuda()
    want = table.to(tdtype(dtype))[ids].permute(2, 0, 1)
    assert torch.equal(got.nan_to_num(123.0), want.nan_to_num(123.0))
    assert torch.equal(got.isnan(), want.isnan())


def test_bias_keeps_the_bits_of_a_table(dcf):
    import torch
    bits = torch.randint(-(1 << 15), 1 << 15, (32, 6), dtype=torch.int32, device="cuda").to(torch.int16)
    got, _ = run_bias(dcf, bits.view(torch.bfloat16), "bf16", 6, 70, 90)
    ids = torch.from_numpy(lo.buckets(lo.positions(70, 0), 90, 32, 128, True)).cuda()
    assert torch.equal(got.contiguous().view(torch.int16), bits[ids].permute(2, 0, 1).contiguous())


def test_bias_many_heads_and_buckets(dcf):
    """More heads than one block's table holds."""
    table = randn((256, 70), "f32", 6)
    got, _ = run_bias(dcf, table, "f32", 70, 6, 700, num_buckets=256, max_distance=600, first_query=300)
    ids = lo.buckets(lo.positions(6, 300), 700, 256, 600, True)
    assert np.array_equal(values(got), bias_want(values(table), ids, None))


def test_bias_past_32_bits_of_elements(dcf):
    """Row offsets beyond 2^32 elements, through a stride."""
    import torch
    keys, row = 19, (1 << 32) + 40
    plan = dcf.position_bias_plan("f16", 1, 2, keys, row_stride=row)
    flat = torch.zeros(plan.out_elements, dtype=torch.float16, device="cuda")
    table = randn((32, 1), "f16", 7)
    dcf.position_bias_async(plan, table, flat)
    ids = lo.buckets(lo.positions(2, 0), keys, 32, 128, True)
    got = torch.stack([flat[:keys], flat[row:row + keys]])
    assert np.array_equal(values(got)[None], bias_want(values(table), ids, None))
    assert int(flat[keys:row].count_nonzero()) == 0


def test_bias_of_the_longest_row(dcf):
    """Columns up to the largest count that is taken: offsets of columns near 2^31."""
    import torch
    keys = (1 << 31) - 65536
    plan = dcf.position_bias_plan("f16", 1, 1, keys, first_query=keys - 200)
    flat = torch.zeros(keys + 8, dtype=torch.float16, device="cuda")
    table = randn((32, 1), "f16", 8)
    dcf.position_bias_async(plan, table, flat)
    ids = lo.buckets(lo.positions(1, 500), 700, 32, 128, True)
    assert np.array_equal(values(flat[keys - 700:keys])[None, None], bias_want(values(table), ids, None))
    assert (flat[:keys - 700] == table[15, 0]).all() and (flat[keys:] == 0).all()


# -------------------------------------------------------------- gradient


def run_grad(dcf, g, dtype, *, given=None, out=None, **kw):
    import torch
    batch, heads, queries, keys = g.shape
    strides = dict(batch_stride=g.stride(0), head_stride=g.stride(1), row_stride=g.stride(2)) if g.numel() else {}
    plan = dcf.position_bias_plan(dtype, heads, queries, keys, batch=batch, accumulate=out is not None, **strides,
                                  **kw)
    wide = torch.float64 if dtype == "f64" else torch.float32
    if out is None:
        out = torch.full((kw.get("num_buckets", 32), heads), float("nan"), dtype=wide, device="cuda")
    work = torch.full((dcf.position_bias_grad_workspace(plan) + 256,), 255, dtype=torch.uint8, device="cuda")
    pos = torch.tensor(given, dtype=torch.int32, device="cuda") if given is not None else None
    dcf.position_bias_grad_async(plan, g, out, work[:plan.workspace], positions=pos)
    torch.cuda.synchronize()
    assert (work[plan.workspace:] == 255).all()
    return out


def check_grad(got, g, dtype, ids, hidden, num_buckets=32, start=0.0):
    batch, heads, queries, keys = g.shape
    want, mag = lo.bias_grad(values(g), ids, num_buckets, hidden)
    step = lo.HALF_STEP["f64" if dtype == "f64" else "f32"]
    bound = lo.bias_grad_bound(mag + abs(start), batch, queries, keys, 16 // g.element_size(), step)
    err = np.abs(values(got) - (want + start))
    assert (err <= bound).all(), (err / bound).max()


@pytest.mark.parametrize("batch,queries,keys", [(1, 1, 1), (2, 1, 9), (1, 3, 40), (3, 17, 33), (1, 64, 64),
                                                (9, 50, 131), (2, 257, 513)])
@pytest.mark.parametrize("both,causal", [(True, False), (False, True)])
@pytest.mark.parametrize("dtype", ["bf16", "f32", "f16", "f64"])
def test_grad_sizes(dcf, batch, queries, keys, both, causal, dtype):
    g = randn((batch, 3, queries, keys), dtype, 11)
    first = max(0, keys - queries)
    got = run_grad(dcf, g, dtype, bidirectional=both, causal=causal, first_query=first)
    q = lo.positions(queries, first)
    check_grad(got, g, dtype, lo.buckets(q, keys, 32, 128, both), lo.masked(q, keys) if causal else None)


@pytest.mark.parametrize("num_buckets,max_distance,both", [(1, 1, False), (2, 1, True), (5, 3, False), (64, 300, True),
                                                           (100, 300, False), (128, 70, True), (256, 400, False)])
@pytest.mark.parametrize("dtype", ["f16", "f64"])
def test_grad_buckets(dcf, num_buckets, max_distance, both, dtype):
    g = randn((2, 2, 90, 210), dtype, 12)
    got = run_grad(dcf, g, dtype, num_buckets=num_buckets, max_distance=max_distance, bidirectional=both,
                   first_query=60)
    ids = lo.buckets(lo.positions(90, 60), 210, num_buckets, max_distance, both)
    check_grad(got, g, dtype, ids, None, num_buckets)


def test_grad_does_not_read_masked_places(dcf):
    """NaN and infinities after the query, and rows that see nothing."""
    import torch
    given = [5, -1, 63, 0, 200, -(1 << 31)]
    g = randn((2, 3, len(given), 64), "bf16", 13)
    hidden = lo.masked(given, 64)
    g[:, :, torch.from_numpy(hidden).cuda()] = float("nan")
    got = run_grad(dcf, g, "bf16", given=given, bidirectional=False, causal=True)
    check_grad(got, g.nan_to_num(0.0), "bf16", lo.buckets(given, 64, 32, 128, False), hidden)


def test_grad_passes_on_what_is_not_finite(dcf):
    g = randn((1, 2, 20, 20), "f32", 14)
    g[0, 1, 3, 3] = float("inf")
    got = values(run_grad(dcf, g, "f32"))
    assert got[0, 1] == np.inf and np.isfinite(np.delete(got.reshape(-1), 1)).all()


@pytest.mark.parametrize("shape,strides,off", [((2, 3, 20, 45), (8000, 2000, 50, 1), 0), ((2, 3, 20, 45), (3 * 20 * 45 + 1, 45, 135, 1), 0),
                                               ((1, 2, 30, 70), (9999, 2101, 70, 1), 3)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_grad_strides(dcf, shape, strides, off, dtype):
    n = sum((s - 1) * t for s, t in zip(shape, strides)) + 1
    flat = randn((n + off,), dtype, 15)
    g = flat[off:].as_strided(shape, strides, off)
    got = run_grad(dcf, g, dtype, first_query=3)
    check_grad(got, g, dtype, lo.buckets(lo.positions(shape[2], 3), shape[3], 32, 128, True), None)


@pytest.mark.parametrize("off", [0, 1, 7])
@pytest.mark.parametrize("batch,queries,keys,first", [(2, 20, 512, 100), (8, 40, 512, -600), (5, 3, 1024, 900),
                                                      (6, 700, 256, 0)])
@pytest.mark.parametrize("dtype,causal", [("bf16", False), ("f16", True), ("f64", False)])
def test_grad_whole_steps_from_any_start(dcf, off, batch, queries, keys, first, dtype, causal):
    """Rows of whole steps, whose first element is off the boundary: the last
    part of a row has a step more."""
    n = batch * 2 * queries * keys
    flat = randn((n + 8,), dtype, 19)
    g = flat[off:off + n].view(batch, 2, queries, keys)
    got = run_grad(dcf, g, dtype, first_query=first, bidirectional=not causal, causal=causal)
    at = lo.positions(queries, first)
    check_grad(got, g, dtype, lo.buckets(at, keys, 32, 128, not causal), lo.masked(at, keys) if causal else None)


def test_grad_accumulates_and_overwrites(dcf):
    import torch
    g = randn((1, 2, 300, 300), "bf16", 16)
    ids = lo.buckets(lo.positions(300, 0), 300, 32, 128, True)
    out = torch.full((32, 2), 5.0, device="cuda")
    got = run_grad(dcf, g, "bf16", out=out)
    assert got is out
    check_grad(got, g, "bf16", ids, None, start=5.0)
    small = g[:, :, :1, :3].contiguous()      # one split: written by the first kernel
    out = torch.full((32, 2), 5.0, device="cuda")
    check_grad(run_grad(dcf, small, "bf16", out=out), small, "bf16", ids[:1, :3], None, start=5.0)


@pytest.mark.parametrize("shape", [(0, 2, 3, 4), (1, 2, 0, 4), (1, 2, 3, 0)])
def test_grad_of_nothing_is_zero(dcf, shape):
    import torch
    g = torch.empty(shape, dtype=torch.float32, device="cuda")
    assert (run_grad(dcf, g, "f32") == 0).all()
    out = torch.full((32, 2), 2.0, device="cuda")
    assert (run_grad(dcf, g, "f32", out=out) == 2.0).all()


@pytest.mark.parametrize("keys,strides", [(19, (20, 20, (1 << 32) + 40)), (24, ((1 << 32) + 40, 48, 24)),
                                          ((1 << 31) - 65536, ((1 << 31) - 65536,) * 3)])
def test_grad_past_32_bits_of_elements(dcf, keys, strides):
    """Offsets beyond 2^32 elements, and the longest row.  Powers of two: every sum is exact."""
    import torch
    rows = 1 if keys > 24 else 2
    batch = 2 if keys == 24 else 1
    n = (batch - 1) * strides[0] + (rows - 1) * strides[2] + keys
    flat = torch.zeros(n, dtype=torch.float16, device="cuda")
    g = flat.as_strided((batch, 1, rows, keys), strides + (1,))
    want, ids = np.zeros((32, 1)), lo.buckets([10], 20, 32, 128, True)
    first = keys - 10
    for k in range(batch * rows):
        for d, v in ((-9, 1.0), (-3, 2.0), (0, 4.0), (2, 8.0), (8, 16.0)):
            b, r = divmod(k, rows)
            place = first + r + d
            if place >= keys:
                continue
            g[b, 0, r, place] = v * 8.0 ** k
            want[ids[0, 10 + d], 0] += v * 8.0 ** k
    if keys > 24:
        g[0, 0, 0, 0] = 0.5
        want[15, 0] += 0.5
    got = run_grad(dcf, g, "f16", first_query=first)
    assert np.array_equal(values(got), want)


def test_grad_same_bits_every_time(dcf):
    import torch
    g = randn((2, 4, 500, 700), "bf16", 17)
    first = run_grad(dcf, g, "bf16")
    for _ in range(3):
        assert torch.equal(run_grad(dcf, g, "bf16"), first)


def test_grad_against_differences(dcf):
    """d/dt sum(g * bias(t)) by differences in 64 bits: the bias is linear in
    its table, so a difference of any width is exact up to rounding."""
    import torch
    heads, queries, keys = 2, 40, 55
    g = randn((1, heads, queries, keys), "f64", 18)
    table = randn((32, heads), "f64", 19)
    grad = values(run_grad(dcf, g, "f64"))
    mag = lo.bias_grad(values(g), lo.buckets(lo.positions(queries, 0), keys, 32, 128, True), 32)[1]
    for v, h in ((0, 0), (3, 1), (8, 0), (17, 1), (24, 0)):
        sums = []
        for sign in (1, -1):
            t = table.clone()
            t[v, h] += sign
            got, _ = run_bias(dcf, t, "f64", heads, queries, keys)
            sums.append(float((got * g[0]).sum()))
        scale = float((g.abs() * 5).sum()) + mag[v, h]
        assert abs((sums[0] - sums[1]) / 2 - grad[v, h]) <= 4400 * 2 * lo.HALF_STEP["f64"] * scale


# ---------------------------------------------------------- orthogonalize

COEF = (3.4445, -4.7750, 2.0315)


def run_orth(dcf, x, dtype, *, out=None, **kw):
    import torch
    batch, rows, cols = x.shape
    plan = dcf.orthogonalize_plan(dtype, rows, cols, batch=batch, **kw)
    if out is None:
        out = torch.full((batch, rows, cols), float("nan"), dtype=tdtype(plan.out_dtype), device="cuda")
    # A workspace full of NaN: what is read has been written.
    work = torch.full((dcf.orthogonalize_workspace(plan) + 256,), 255, dtype=torch.uint8, device="cuda")
    status = torch.empty(2, dtype=torch.int64, device="cuda")
    dcf.status_reset(status)
    dcf.orthogonalize_async(plan, x, out, work[:plan.workspace], status)
    assert dcf.status_read(status).folded
    assert (work[plan.workspace:] == 255).all()
    return out


def check_orth(got, x, out_dtype, coef, eps=1e-7):
    got, x = values(got), values(x)
    for k in range(x.shape[0]):
        want = lo.newton_schulz(x[k], coef, eps)
        tol = lo.orth_tolerance(x[k], coef, eps) + lo.HALF_STEP[out_dtype]
        # fp16 results below its normal range round to half of 2^-24
        small = 2.0 ** -25 * np.sqrt(want.size) if out_dtype == "f16" else 0.0
        err = np.linalg.norm(got[k] - want)
        assert err <= tol * np.linalg.norm(want) + small, (err / np.linalg.norm(want), tol)


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (7, 1), (3, 5), (16, 16), (31, 65), (64, 64), (96, 96),
                                       (65, 31), (127, 129), (128, 128), (129, 128), (128, 500), (200, 333), (333, 200),
                                       (257, 257), (1, 1000), (300, 2), (100, 2048), (2048, 100), (9, 2049),
                                       (2049, 9), (128, 257), (600, 128), (513, 65), (40, 256)])
def test_orth_sizes(dcf, rows, cols):
    x = randn((1, rows, cols), "f32", 21)
    check_orth(run_orth(dcf, x, "f32"), x, "f32", [COEF] * 5)


@pytest.mark.parametrize("dtype,out_dtype", [("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("bf16", "f32"),
                                             ("f16", "f32"), ("f32", "f16")])
@pytest.mark.parametrize("rows,cols", [(40, 72), (150, 90)])
def test_orth_types(dcf, dtype, out_dtype, rows, cols):
    x = randn((3, rows, cols), dtype, 22)
    check_orth(run_orth(dcf, x, dtype, out_dtype=out_dtype), x, out_dtype, [COEF] * 5)


@pytest.mark.parametrize("steps", [0, 1, 2, 7])
def test_orth_steps(dcf, steps):
    for shape in ((2, 50, 80), (1, 150, 140)):
        x = randn(shape, "f32", 23)
        check_orth(run_orth(dcf, x, "f32", steps=steps), x, "f32", [COEF] * steps)


def test_orth_coefficients_of_each_step(dcf):
    coef = [(4.0, -6.0, 2.9), (3.0, -3.2, 1.2), (1.875, -1.25, 0.375), (1.5, -0.5, 0.0)]
    x = randn((1, 70, 180), "f32", 24)
    check_orth(run_orth(dcf, x, "f32", steps=4, coef=coef), x, "f32", coef)


@pytest.mark.parametrize("rows,cols", [(100, 120), (260, 200)])
def test_orth_low_rank(dcf, rows, cols):
    """What rounding leaves in the null space is amplified the most."""
    import torch
    x = randn((1, rows, 4), "f32", 25) @ randn((1, 4, cols), "f32", 26)
    # the f32 product itself is the input: its own noise is part of it
    check_orth(run_orth(dcf, x, "f32"), x, "f32", [COEF] * 5)


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e30])
def test_orth_scales(dcf, scale):
    x = randn((1, 60, 50), "f32", 27, scale)
    check_orth(run_orth(dcf, x, "f32", eps=0.0), x, "f32", [COEF] * 5, eps=0.0)


def test_orth_small_coefficients(dcf):
    """Results far below the input's scale keep their precision."""
    for shape in ((1, 40, 60), (1, 150, 170)):
        x = randn(shape, "f32", 34)
        coef = [(1e-12, 1e-13, -2e-13)] * 2
        check_orth(run_orth(dcf, x, "f32", steps=2, coef=coef), x, "f32", coef)


def test_orth_zero_and_not_finite(dcf):
    import torch
    x = randn((4, 33, 40), "f32", 28)
    x[0] = 0
    x[2, 3, 3] = float("nan")
    got = run_orth(dcf, x, "f32")
    assert (got[0] == 0).all()
    assert got[2].isnan().all()
    check_orth(got[[1, 3]], x[[1, 3]], "f32", [COEF] * 5)


@pytest.mark.parametrize("rows,cols", [(45, 61), (150, 131)])
def test_orth_strides_and_what_lies_between(dcf, rows, cols):
    import torch
    for dtype in ("bf16", "f32"):
        flat = randn((3 * 200 * 200 + 7,), dtype, 29)
        x = flat[5:].as_strided((2, rows, cols), (rows * 183 + 11, 183, 1), 5)
        out = torch.full((2 * 200 * 200,), 9.0, dtype=tdtype(dtype), device="cuda")
        view = out.as_strided((2, rows, cols), (rows * 171 + 1, 171, 1), 3)
        run_orth(dcf, x, dtype, out=view, row_stride=183, batch_stride=rows * 183 + 11, out_row_stride=171,
                 out_batch_stride=rows * 171 + 1)
        check_orth(view, x, dtype, [COEF] * 5)
        view.fill_(9.0)
        assert (out == 9.0).all()


@pytest.mark.parametrize("steps", [0, 5])
def test_orth_in_place(dcf, steps):
    import torch
    for shape in ((2, 40, 30), (1, 200, 140)):
        x = randn(shape, "f32", 30)
        want = run_orth(dcf, x, "f32", steps=steps)
        run_orth(dcf, x, "f32", steps=steps, out=x)
        assert torch.equal(x, want)


@pytest.mark.parametrize("batch", [1, 7, 40, 80, 160])
@pytest.mark.parametrize("rows,cols", [(30, 600), (600, 30)])
def test_orth_clusters_of_every_size(dcf, batch, rows, cols):
    """The number of CTAs to a matrix depends on how many matrices there are."""
    x = randn((batch, rows, cols), "f32", 33)
    got = run_orth(dcf, x, "f32", steps=3)
    some = sorted({0, batch // 2, batch - 1})
    check_orth(got[some], x[some], "f32", [COEF] * 3)


def test_orth_same_bits_every_time_and_in_any_place_of_a_batch(dcf):
    import torch
    for rows, cols in ((50, 60), (140, 300)):
        x = randn((5, rows, cols), "bf16", 31)
        first = run_orth(dcf, x, "bf16")
        assert torch.equal(run_orth(dcf, x, "bf16"), first)
        assert torch.equal(run_orth(dcf, x[[3] * 5].contiguous(), "bf16"), first[[3] * 5])


# ------------------------------------------------------------- together


def test_device_pointer_checks(dcf):
    import torch
    plan = dcf.position_bias_plan("f32", 2, 4, 8)
    out = torch.zeros(64, device="cuda")
    table = torch.zeros(32, 2)                     # host memory
    with pytest.raises(dcf.DcfError):
        dcf.position_bias_async(plan, table, out)
    with pytest.raises(ValueError):
        dcf.position_bias_async(plan, table.cuda(), out[1:])
    with pytest.raises(ValueError):
        dcf.position_bias_async(plan, table.cuda().double(), out)
    with pytest.raises(ValueError):
        dcf.position_bias_async(plan, table.cuda(), out, positions=torch.zeros(4, device="cuda"))
    with pytest.raises(ValueError):          # one element shown many times is not room for many
        dcf.position_bias_async(plan, table.cuda(), torch.zeros(1, device="cuda").expand(64))
    odd = torch.zeros(300, dtype=torch.uint8, device="cuda")[1:257].view(torch.uint8)
    with pytest.raises(dcf.DcfError):
        dcf._check(dcf.lib().dcf_position_bias_async(plan.ref, table.cuda().data_ptr(), None, odd.data_ptr(), None))


def test_host_forms(dcf):
    rng = np.random.default_rng(41)
    plan = dcf.position_bias_plan("f32", 3, 20, 30, bidirectional=False, causal=True, first_query=10, batch=2)
    table = rng.standard_normal((32, 3)).astype(np.float32)
    q = lo.positions(20, 10)
    ids, hidden = lo.buckets(q, 30, 32, 128, False), lo.masked(q, 30)
    f = dcf.position_bias(plan, table)
    assert f.folded and not f.is_splat
    assert np.array_equal(f.out.view(np.float32), bias_want(table, ids, hidden).astype(np.float32))
    assert dcf.position_bias(dcf.position_bias_plan("f32", 3, 20, 30), np.full((32, 3), 2.5, np.float32)).is_splat
    g = rng.standard_normal((2, 3, 20, 30)).astype(np.float32)
    want, mag = lo.bias_grad(g, ids, 32, hidden)
    got = dcf.position_bias_grad(plan, g)
    assert (np.abs(got.out - want) <= lo.bias_grad_bound(mag, 2, 20, 30, 4, lo.U32)).all()
    given = rng.integers(0, 30, 20).astype(np.int32)
    f = dcf.position_bias(plan, table, positions=given)
    assert np.array_equal(f.out.view(np.float32),
                          bias_want(table, lo.buckets(given, 30, 32, 128, False), lo.masked(given, 30)).astype(np.float32))
    x = rng.standard_normal((2, 30, 25)).astype(np.float32)
    o = dcf.orthogonalize(dcf.orthogonalize_plan("f32", 30, 25, batch=2), x)
    for k in range(2):
        want = lo.newton_schulz(x[k], [COEF] * 5, 1e-7)
        tol = lo.orth_tolerance(x[k], [COEF] * 5, 1e-7) + lo.U32
        assert np.linalg.norm(o.out[k].view(np.float32) - want) <= tol * np.linalg.norm(want)


def test_another_stream_and_captured_graph(dcf):
    """Bias, its gradient and the orthogonalised gradient as one captured step,
    replayed on new inputs."""
    import torch
    heads, queries, keys = 4, 100, 120
    bias = dcf.position_bias_plan("f32", heads, queries, keys)
    orth = dcf.orthogonalize_plan("f32", 32, heads)
    table = randn((32, heads), "f32", 51)
    g = torch.empty(1, heads, queries, keys, device="cuda")
    dtable, step = torch.empty(32, heads, device="cuda"), torch.empty(32, heads, device="cuda")
    out = torch.empty(heads, queries, keys, device="cuda")
    w1 = torch.empty(dcf.position_bias_grad_workspace(bias) + 1, dtype=torch.uint8, device="cuda")
    w2 = torch.empty(dcf.orthogonalize_workspace(orth), dtype=torch.uint8, device="cuda")
    status = torch.empty(2, dtype=torch.int64, device="cuda")
    dcf.status_reset(status)

    def run():
        dcf.position_bias_async(bias, table, out)
        g.copy_(out[None] - 1.0)                # the gradient of |bias - 1|^2 / 2
        dcf.position_bias_grad_async(bias, g, dtable, w1)
        dcf.orthogonalize_async(orth, dtable, step, w2, status)
        table.sub_(step, alpha=0.1)

    start = table.clone()
    eager = []
    for _ in range(3):
        run()
        eager.append((table.clone(), dtable.clone(), out.clone()))
    table.copy_(start)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(table, eager[0][0])
    table.copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    assert torch.equal(table, start)
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((table, dtable, out), eager[k]):
            assert torch.equal(a, b)
    assert dcf.status_read(status).folded
    # and the step means what it says: the table's rows move against the gradient
    ids = lo.buckets(lo.positions(queries, 0), keys, 32, 128, True)
    check_grad(dtable, g, "f32", ids, None)


def test_two_streams_at_once_and_graphs_that_share_a_workspace(dcf):
    import torch
    xs = [randn((3, 200, 333), "f32", 71), randn((12, 150, 140), "f32", 72)]
    gs = [randn((2, 4, 300, 257), "bf16", 73), randn((1, 4, 300, 257), "bf16", 74)]
    orth = [dcf.orthogonalize_plan("f32", *x.shape[1:], batch=x.shape[0]) for x in xs]
    grad = [dcf.position_bias_plan("bf16", 4, 300, 257, batch=g.shape[0]) for g in gs]
    want = [run_orth(dcf, x, "f32") for x in xs], [run_grad(dcf, g, "bf16") for g in gs]
    got = [torch.empty_like(x) for x in xs], [torch.empty(32, 4, device="cuda") for _ in gs]
    size = [dcf.orthogonalize_workspace(o) for o in orth], [dcf.position_bias_grad_workspace(p) for p in grad]
    status = torch.empty(2, 2, dtype=torch.int64, device="cuda")
    for k in range(2):
        dcf.status_reset(status[k])

    def run(k, w1, w2):
        dcf.orthogonalize_async(orth[k], xs[k], got[0][k], w1, status[k])
        dcf.position_bias_grad_async(grad[k], gs[k], got[1][k], w2)

    def same():
        torch.cuda.synchronize()
        for a, b in zip(want[0] + want[1], got[0] + got[1]):
            assert torch.equal(a, b)
        for t in got[0] + got[1]:
            t.fill_(float("nan"))

    own = [[torch.empty(n[k] + 1, dtype=torch.uint8, device="cuda") for n in size] for k in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                run(k, *own[k])
    same()
    shared = [torch.empty(max(n) + 1, dtype=torch.uint8, device="cuda") for n in size]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for k in range(2):
        with torch.cuda.graph(graphs[k]):
            run(k, *shared)
    for order in ((0, 1), (1, 0), (0, 0, 1, 1)):
        for k in order:
            graphs[k].replay()
        same()
    assert all(dcf.status_read(status[k]).folded for k in range(2))


@pytest.mark.parametrize("batch,rows,cols", [(65535, 3, 5), (70, 130, 150), (300, 20, 2100)])
def test_orth_many_matrices(dcf, batch, rows, cols):
    x = randn((batch, rows, cols), "f32", 81)
    got = run_orth(dcf, x, "f32")
    at = [0, 1, batch // 2, batch - 2, batch - 1]
    check_orth(got[at], x[at], "f32", [COEF] * 5)
    assert bool(got.isfinite().all())


@pytest.mark.parametrize("rows,cols,dtype", [(1601, 1550, "f32"), (1540, 1603, "bf16"), (1536, 2100, "f32")])
def test_orth_large(dcf, rows, cols, dtype):
    """Sizes that pairs of CTAs take."""
    x = randn((1, rows, cols), dtype, 61)
    check_orth(run_orth(dcf, x, dtype, steps=2), x, dtype, [COEF] * 2)


def fp32_form(x, steps):
    """The iteration with products of fp32 values, rounded once to x's type."""
    y = x.float() if x.shape[1] <= x.shape[2] else x.float().transpose(1, 2)
    y = y / (y.square().sum((1, 2), keepdim=True).sqrt() + 1e-7)
    a, b, c = COEF
    for _ in range(steps):
        gram = y @ y.transpose(1, 2)
        y = a * y + (b * gram + c * (gram @ gram)) @ y
    return (y if x.shape[1] <= x.shape[2] else y.transpose(1, 2)).to(x.dtype)


def exact_form(x, steps):
    import torch
    y = x.double() if x.shape[1] <= x.shape[2] else x.double().transpose(1, 2)
    y = y / (torch.linalg.vector_norm(y, dim=(1, 2), keepdim=True) + 1e-7)
    a, b, c = COEF
    for _ in range(steps):
        gram = y @ y.transpose(1, 2)
        y = a * y + (b * gram + c * (gram @ gram)) @ y
    return y if x.shape[1] <= x.shape[2] else y.transpose(1, 2)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("batch,rows,cols", [(8, 96, 96), (8, 128, 128), (8, 128, 1000), (8, 1000, 60), (8, 70, 900), (8, 150, 180),
                                             (8, 258, 131), (8, 260, 300), (1, 512, 2048), (1, 520, 530),
                                             (1, 800, 810), (1, 1300, 1100), (1, 1024, 4096), (1, 4096, 300)])
def test_orth_rounds_what_fp32_products_would(dcf, dtype, batch, rows, cols):
    """Results of 16 bits come from sums as exact as those of fp32 products: a
    result that is not the 64-bit value rounded lies within the sums' error of
    a border, so the share of these is proportional to that error.  Half as many
    again are allowed, and four times what counting them varies by."""
    import torch
    assert not torch.backends.cuda.matmul.allow_tf32
    x = randn((batch, rows, cols), dtype, 91)
    want = exact_form(x, 5).to(tdtype(dtype))
    plain = float((fp32_form(x, 5) != want).double().mean())
    here = float((run_orth(dcf, x, dtype) != want).double().mean())
    assert here <= 1.5 * plain + 4 * (plain / want.numel()) ** 0.5, (here, plain)


@pytest.mark.parametrize("shape", [(2, 30, 40), (2, 150, 140)])
@pytest.mark.parametrize("steps", [0, 5])
def test_orth_zeros_stay_zeros_beside_the_smallest_eps(dcf, shape, steps):
    import torch
    x = torch.zeros(shape, device="cuda")
    for eps in (1e-7, 1e-300, 1e-306, 5e-324):
        assert (run_orth(dcf, x, "f32", steps=steps, eps=eps) == 0).all(), eps
    assert run_orth(dcf, x, "f32", steps=steps, eps=0.0).isnan().all()      # 0 / 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(60, 90), (500, 100), (150, 170), (300, 131)])
def test_orth_norms_far_below_eps(dcf, rows, cols, dtype):
    """The norm's share of norm + eps scales the planes: nothing is lost to a
    fixed scale.  One batch of very different matrices, the first and last of usual norm."""
    norms = [1.0, 1e-9, 1e-12, 1e-15, 1e-30, 0.0, 5e-8, 1e-7, 3.0]
    x = randn((len(norms), rows, cols), "f32", 95)
    for k, norm in enumerate(norms):
        x[k] *= norm / float(x[k].double().norm())
    x = x.to(tdtype(dtype))
    got = run_orth(dcf, x, dtype)
    assert (got[5] == 0).all()
    some = [k for k in range(len(norms)) if k != 5]
    check_orth(got[some], x[some], dtype, [COEF] * 5)


def check_orth_f32(got, x, coef, eps):
    """One f32 matrix whose results may be far smaller than the planes' bounds (odd powers
    alone shrink what is below one), or lie below f32's normal range: there they round to
    half of 2^-149 (and below that to zero), so a 2-norm is off by 2^-150 for each; as much
    again is allowed."""
    got, x = values(got)[0], values(x)[0]
    want = lo.newton_schulz(x, coef, eps)
    tol = lo.orth_tolerance(x, coef, eps) + lo.U32
    err = np.linalg.norm(got - want)
    assert err <= tol * np.linalg.norm(want) + lo.orth_quantum(x, coef, eps) + 2.0 ** -149 * np.sqrt(want.size), \
        (err, np.linalg.norm(want), tol)


@pytest.mark.parametrize("rows,cols", [(60, 90), (150, 170)])
@pytest.mark.parametrize("coef", [(3.4445, -4.7750, 2.0315), (1.5, -0.5, 0.0), (0.0, 1.0, 0.0), (1e-3, 0.5, 0.25),
                                  (2.0, 0.0, -1.0)])
def test_orth_small_norms_with_other_coefficients(dcf, rows, cols, coef):
    """Odd powers alone (a = 0) make results far smaller than X; eps beyond 1."""
    for norm, eps, steps in ((1e-3, 1e-1, 2), (1e-5, 2.0, 3), (1e-2, 1e-2, 2)):
        x = randn((1, rows, cols), "f32", 96)
        x *= norm / float(x.double().norm())
        check_orth_f32(run_orth(dcf, x, "f32", steps=steps, coef=coef, eps=eps), x, [coef] * steps, eps)


@pytest.mark.parametrize("shape", [(1, 60, 90), (1, 150, 170)])
def test_orth_results_at_the_end_of_f32(dcf, shape):
    """norm / (norm + eps) of 2^-133, and a value that no f32 has."""
    x = randn(shape, "f32", 97)
    x *= 1e-30 / float(x.double().norm())
    for eps in (1e10, 1e300):
        check_orth_f32(run_orth(dcf, x, "f32", eps=eps), x, [COEF] * 5, eps)


@pytest.mark.parametrize("rows,cols", [(2, 2), (150, 170), (170, 150)])
@pytest.mark.parametrize("c", [0.0, 5.5e-17, -5.5e-17])
def test_orth_largest_value_inside_the_interval(dcf, rows, cols, c):
    """2.6 s - 2.5 s^3 is 0.1 at 1 and 1.02 at 0.589: planes scaled for the first overflow."""
    import torch
    x = torch.zeros(1, rows, cols, device="cuda")
    x[0, 0, 0], x[0, 1, 1] = 0.589, 0.808
    coef = [(2.6, -2.5, c)] * 2
    check_orth(run_orth(dcf, x, "f32", steps=2, coef=coef), x, "f32", coef)


PROGRAMMATIC_EDGES = """
import ctypes, sys
import torch
import mlirpass_b200 as dcf
cu = ctypes.CDLL("libcuda.so.1")
def check(rc):
    assert rc == 0, rc
torch.manual_seed(1)
stream = torch.cuda.Stream()
orth = dcf.orthogonalize_plan("f32", 150, 170)
grad = dcf.position_bias_plan("f32", 8, 500, 500)
x, g = torch.randn(150, 170, device="cuda"), torch.randn(1, 8, 500, 500, device="cuda")
out, table = torch.empty_like(x), torch.empty(32, 8, device="cuda")
work = torch.empty(orth.workspace + grad.workspace, dtype=torch.uint8, device="cuda")
status = torch.empty(2, dtype=torch.int64, device="cuda")
dcf.status_reset(status)
def count(run):
    run()
    torch.cuda.synchronize()
    graph, n = ctypes.c_void_p(), ctypes.c_size_t(0)
    check(cu.cuStreamBeginCapture_v2(ctypes.c_void_p(stream.cuda_stream), 2))
    run()
    check(cu.cuStreamEndCapture(ctypes.c_void_p(stream.cuda_stream), ctypes.byref(graph)))
    check(cu.cuGraphGetEdges_v2(graph, None, None, None, ctypes.byref(n)))
    start, end, data = (ctypes.c_void_p * n.value)(), (ctypes.c_void_p * n.value)(), (ctypes.c_uint8 * (8 * n.value))()
    check(cu.cuGraphGetEdges_v2(graph, start, end, data, ctypes.byref(n)))
    check(cu.cuGraphDestroy(graph))
    return n.value, sum(data[8 * i + 2] == 1 for i in range(n.value))
a = count(lambda: dcf.orthogonalize_async(orth, x, out, work, status, stream=stream))
b = count(lambda: dcf.position_bias_grad_async(grad, g, table, work, stream=stream))
assert dcf.status_read(status).folded
print(*a, *b, out.double().sum().item().hex(), table.double().sum().item().hex())
"""


def test_launches_as_programmatic_dependents_can_be_turned_off():
    """DCF_PDL=0 reaches every launch of these operators: no programmatic edge in a captured graph, the same bits."""
    import os
    import subprocess
    import sys
    import conftest
    got = {}
    for value in ("1", "0"):
        env = dict(os.environ, DCF_PDL=value, PYTHONPATH=conftest.ROOT)
        run = subprocess.run([sys.executable, "-c", PROGRAMMATIC_EDGES], env=env, capture_output=True, text=True, timeout=300)
        assert run.returncode == 0, run.stderr[-2000:]
        got[value] = run.stdout.split()
    assert got["1"][4:] == got["0"][4:] and got["1"][0::2][:2] == got["0"][0::2][:2]
    assert int(got["1"][0]) >= 10 and int(got["1"][1]) >= 10 and int(got["1"][3]) == 1
    assert got["0"][1] == got["0"][3] == "0"


# --------------------------------------- gradient sums that are exact


def whole(shape, dtype, seed):
    import torch
    return torch.from_numpy(lo.whole_values(shape, seed)).cuda().to(tdtype(dtype))


def check_exact(got, g, ids, hidden, num_buckets=32, start=0.0):
    want, mag = lo.bias_grad(values(g), ids, num_buckets, hidden)
    assert mag.max() + abs(start) < 2 ** 24
    assert np.array_equal(values(got), want + start)


@pytest.mark.parametrize("batch,queries,keys", [(1, 1, 1), (2, 1, 9), (1, 3, 40), (3, 17, 33), (1, 64, 64),
                                                (9, 50, 131), (2, 257, 513), (1, 1, 5000), (40, 7, 65), (3, 1000, 12)])
@pytest.mark.parametrize("both,causal", [(True, False), (False, True), (False, False), (True, True)])
@pytest.mark.parametrize("dtype", ["bf16", "f32", "f16", "f64"])
def test_grad_exact_sizes(dcf, batch, queries, keys, both, causal, dtype):
    g = whole((batch, 3, queries, keys), dtype, 111)
    first = max(0, keys - queries)
    got = run_grad(dcf, g, dtype, bidirectional=both, causal=causal, first_query=first)
    q = lo.positions(queries, first)
    check_exact(got, g, lo.buckets(q, keys, 32, 128, both), lo.masked(q, keys) if causal else None)


@pytest.mark.parametrize("off", [0, 1, 3, 7])
@pytest.mark.parametrize("batch,queries,keys,first", [(2, 20, 512, 100), (8, 40, 512, -600), (5, 3, 1024, 900),
                                                      (6, 700, 256, 0), (2, 30, 1023, 500), (1, 9, 4097, 8000)])
@pytest.mark.parametrize("dtype,causal", [("bf16", False), ("f16", True), ("f16", False), ("f32", True), ("f64", False)])
def test_grad_exact_from_any_start(dcf, off, batch, queries, keys, first, dtype, causal):
    """Every step of every row counts once, wherever rows begin within 16 bytes."""
    import torch
    n = batch * 2 * queries * keys
    flat = torch.zeros(n + 8, device="cuda", dtype=tdtype(dtype))
    g = flat[off:off + n].view(batch, 2, queries, keys)
    g.copy_(whole((batch, 2, queries, keys), dtype, 119))
    got = run_grad(dcf, g, dtype, first_query=first, bidirectional=not causal, causal=causal)
    at = lo.positions(queries, first)
    check_exact(got, g, lo.buckets(at, keys, 32, 128, not causal), lo.masked(at, keys) if causal else None)


@pytest.mark.parametrize("shape,strides,off", [((2, 3, 20, 45), (8000, 2000, 50, 1), 0), ((2, 3, 20, 45), (3 * 20 * 45 + 1, 45, 135, 1), 0),
                                               ((1, 2, 30, 70), (9999, 2101, 70, 1), 3), ((3, 2, 11, 600), (20007, 9001, 640, 1), 5)])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32", "f64"])
def test_grad_exact_strides(dcf, shape, strides, off, dtype):
    """What lies between rows (here NaN) is not summed."""
    import torch
    n = sum((s - 1) * t for s, t in zip(shape, strides)) + 1
    flat = torch.full((n + off + 8,), float("nan"), device="cuda", dtype=tdtype(dtype))
    g = flat[off:].as_strided(shape, strides, off)
    g.copy_(whole(shape, dtype, 115))
    got = run_grad(dcf, g, dtype, first_query=3)
    check_exact(got, g, lo.buckets(lo.positions(shape[2], 3), shape[3], 32, 128, True), None)


@pytest.mark.parametrize("num_buckets,max_distance,both", [(1, 1, False), (2, 1, True), (3, 2, True), (5, 3, False),
                                                           (64, 300, True), (100, 3000, False), (128, 70, True), (256, 400, False)])
@pytest.mark.parametrize("dtype", ["f16", "f32", "f64"])
def test_grad_exact_buckets_and_positions(dcf, num_buckets, max_distance, both, dtype):
    rng = np.random.default_rng(5)
    given = [int(v) for v in rng.integers(-400, 900, 60)] + [0, 0, 299, -1, 300, 5000, -(1 << 31), (1 << 31) - 1]
    g = whole((2, 2, len(given), 300), dtype, 112)
    for causal in (False, True):
        got = run_grad(dcf, g, dtype, given=given, num_buckets=num_buckets, max_distance=max_distance, bidirectional=both,
                       causal=causal)
        check_exact(got, g, lo.buckets(given, 300, num_buckets, max_distance, both),
                    lo.masked(given, 300) if causal else None, num_buckets)


@pytest.mark.parametrize("shape", [(1, 2, 1, 3), (2, 2, 300, 300)])
@pytest.mark.parametrize("dtype", ["bf16", "f64"])
def test_grad_exact_accumulates(dcf, shape, dtype):
    import torch
    g = whole(shape, dtype, 116)
    out = torch.full((32, 2), 5.0, device="cuda", dtype=torch.float64 if dtype == "f64" else torch.float32)
    for k in range(3):
        run_grad(dcf, g, dtype, out=out)
    ids = lo.buckets(lo.positions(shape[2], 0), shape[3], 32, 128, True)
    assert np.array_equal(values(out), 3 * lo.bias_grad(values(g), ids, 32)[0] + 5.0)


# ------------------------------------------------- clusters, low rank, not finite


@pytest.mark.parametrize("batch", [1, 150])
@pytest.mark.parametrize("longer", [256, 257, 512, 513, 1024, 1025, 1100, 2048])
@pytest.mark.parametrize("shorter", [30, 128])
@pytest.mark.parametrize("tall", [False, True])
def test_orth_clusters_of_one_to_eight(dcf, batch, longer, shorter, tall):
    """A matrix takes a cluster of 1, 2, 4 or 8 CTAs by its longer side alone; the last CTAs may
    hold few columns or none.  One matrix, and more of them than SMs."""
    shape = (batch, longer, shorter) if tall else (batch, shorter, longer)
    x = randn(shape, "f32", 133)
    got = run_orth(dcf, x, "f32", steps=3)
    some = sorted({0, batch // 2, batch - 1})
    check_orth(got[some], x[some], "f32", [COEF] * 3)
    assert bool(got.isfinite().all())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [(60, 200), (100, 120), (200, 260), (700, 150)])
def test_orth_low_rank_of_16_bits(dcf, rows, cols, dtype):
    """Whole numbers of four directions: the rank is exact in 16 bits, the null space is amplified the most."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(125)
    a = torch.randint(-3, 4, (1, rows, 4), device="cuda", generator=gen).float()
    b = torch.randint(-3, 4, (1, 4, cols), device="cuda", generator=gen).float()
    x = (a @ b).to(tdtype(dtype))
    assert torch.linalg.matrix_rank(x[0].double()) == 4
    check_orth(run_orth(dcf, x, dtype), x, dtype, [COEF] * 5)
    check_orth(run_orth(dcf, x, dtype, out_dtype="f32"), x, "f32", [COEF] * 5)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(33, 40), (40, 900), (150, 170), (300, 140)])
def test_orth_not_finite_in_a_batch(dcf, rows, cols, dtype):
    """NaN or an infinity makes its own matrix NaN and no other; zeros stay zeros."""
    x = randn((6, rows, cols), dtype, 128)
    x[0] = 0
    x[2, 3, 3] = float("nan")
    x[3, rows - 1, cols - 1] = float("inf")
    x[4, 0, cols - 1] = float("-inf")
    got = run_orth(dcf, x, dtype)
    assert (got[0] == 0).all()
    assert all(got[k].isnan().all() for k in (2, 3, 4))
    check_orth(got[[1, 5]], x[[1, 5]], dtype, [COEF] * 5)
