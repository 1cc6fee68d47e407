"""The tiles of the 8-bit product and of the gradient from a checkpoint, on the GPU: every kernel over several
stages, tiles and parts of varied data, each size with the kernel that it reaches (as the restated cost rules say)."""

import pytest

import int8_cuts as cuts
import int8_oracle as io
from test_gpu_int8 import exact_inputs, new_status, randn, rounded, run_grad, run_matmul, same, scales_for, whole, wide

pytestmark = pytest.mark.gpu


def plain(a, b, sa=None, sb=None, bias=None):
    """The product's f32 result (i32 sums where there are no scales) of int8 a, b: sums in 64 bits, which hold them
    exactly, then the f32 steps of its definition."""
    import torch
    sums = a.double() @ b.double().T
    if sb is None:
        return sums.to(torch.int32)
    out = sums.float() * sa[:, None] * sb[None, :]
    return out if bias is None else out + bias[None, :]


def check(dcf, tokens, channels, depth, out, *, bias=False, seed=0, a_dtype="i8", **kw):
    import torch
    b = whole((channels, depth), seed + 1)
    sa, sb, add = scales_for(tokens, channels, seed + 2)
    add = add if bias else None
    if a_dtype != "i8":
        x = randn((tokens, depth), a_dtype, seed)
        got = run_matmul(dcf, x, b, a_dtype=a_dtype, out=out, b_scale=sb, bias=add, **kw)
        q, s = io.quantize(wide(x), "rows")
        want = plain(torch.from_numpy(q).cuda(), b, torch.from_numpy(s).cuda(), sb, add)
    else:
        a = whole((tokens, depth), seed)
        if out == "i32":
            assert torch.equal(run_matmul(dcf, a, b, out=out, **kw), plain(a, b))
            return
        got = run_matmul(dcf, a, b, out=out, a_scale=sa, b_scale=sb, bias=add, **kw)
        want = plain(a, b, sa, sb, add)
    assert torch.equal(got, want.to(got.dtype))


# (tokens, channels, depth) and what they are cut into: tokens of a tile, whether more tiles than pairs of CTAs, whether parts.
PRODUCTS = [
    ((300, 3000, 1100), 64, False, False), ((150, 530, 9000), 64, False, True), ((100, 9001, 520), 64, False, False),
    ((150, 20001, 272), 64, True, False),
    ((1001, 2047, 1531), 128, False, False), ((900, 2049, 1100), 128, False, False), ((2300, 4100, 1100), 128, True, False),
    ((700, 700, 5000), 128, False, True), ((257, 257, 9000), 128, False, True),
    ((1100, 2100, 2100), 256, False, False), ((3000, 5001, 700), 256, True, False), ((1000, 1030, 6000), 256, False, True),
]
IDS = ["x".join(map(str, size)) for size, *_ in PRODUCTS]


@pytest.fixture(params=PRODUCTS, ids=IDS)
def product(request):
    (tokens, channels, depth), tile, many, parts = request.param
    tn, tiles, n = cuts.matmul_cut(tokens, channels, depth)
    assert (tn, tiles > cuts.PAIRS, n > 1) == (tile, many, parts)
    return tokens, channels, depth


@pytest.mark.parametrize("out", ["i32", "f32", "bf16", "f16"])
def test_products(dcf, product, out):
    """A weight that a tensor map describes, or one of odd depth: copied, or read by threads in tiles of 64."""
    check(dcf, *product, out, bias=out in ("f32", "f16"), seed=len(out))


@pytest.mark.parametrize("out,offset", [("i32", 1), ("bf16", 8), ("f32", 15)])
def test_products_of_a_weight_whose_start_lies_off_a_boundary(dcf, product, out, offset):
    """Rows a multiple of 16 bytes apart that start off 16-byte boundaries: read by threads in tiles of any width."""
    depth = product[2]
    check(dcf, *product, out, bias=True, seed=offset, pads=(0, -depth % 16 or 16, 0), offsets=(0, offset, 0))


@pytest.mark.parametrize("out,pads,offsets", [("bf16", (5, 16, 1), (0, 0, 0)), ("f16", (16, 0, 8), (3, 0, 1)), ("f32", (0, 3, 3), (0, 5, 1))])
def test_products_in_padded_rows(dcf, product, out, pads, offsets):
    check(dcf, *product, out, bias=True, seed=pads[0], pads=pads, offsets=offsets)


@pytest.mark.parametrize("a_dtype,out,offset", [("bf16", "bf16", 0), ("f16", "f32", 0), ("f32", "f16", 0), ("bf16", "f32", 3)])
def test_products_of_float_tokens(dcf, product, a_dtype, out, offset):
    """Tokens that the call quantises; the first stages of a weight that is not copied are loaded meanwhile."""
    pad = (-product[2] % 16 or 16) if offset else 0
    check(dcf, *product, out, bias=True, seed=7, a_dtype=a_dtype, pads=(0, pad, 0), offsets=(0, offset, 0))


# ---------------------------------------------- a weight that is loaded early


@pytest.mark.parametrize("tokens,channels,depth", [(2, 300, 5000), (3, 70, 4096), (4, 4096, 4096), (4, 100, 15000), (2, 64, 30000), (4, 33, 4099)])
@pytest.mark.parametrize("a_dtype,out", [("bf16", "bf16"), ("f32", "f32"), ("f16", "f16")])
def test_few_float_tokens_that_a_launch_of_their_own_quantises(dcf, tokens, channels, depth, a_dtype, out):
    assert cuts.few_tokens(tokens, depth) and tokens * depth > 8192
    check(dcf, tokens, channels, depth, out, bias=True, seed=3, a_dtype=a_dtype)
    check(dcf, tokens, channels, depth, out, seed=4, a_dtype=a_dtype, pads=(3, 16, 0), offsets=(0, 1, 0))


@pytest.mark.parametrize("tokens,channels,depth", [(4, 1024, 4096), (48, 4096, 4096), (900, 2049, 1104), (1100, 2100, 2112), (4, 512, 4095), (48, 1024, 4095)])
def test_a_weight_that_is_written_right_before(dcf, tokens, channels, depth):
    """Every product reads what the launch before its own wrote, though its weight is loaded ahead of its tokens; the
    same buffers each time."""
    import torch
    x = randn((tokens, depth), "bf16", 1)
    weights = [randn((channels, depth), "bf16", 10 + i, 0.05 * (i + 1)) for i in range(6)]
    wplan, plan = dcf.quantize_plan("bf16", channels, depth), dcf.int8_matmul_plan(tokens, channels, depth, a_dtype="bf16", out_dtype="f32")
    wq, ws = torch.empty(channels, depth, dtype=torch.int8, device="cuda"), torch.empty(channels, device="cuda")
    work, status = torch.empty(plan.workspace, dtype=torch.uint8, device="cuda"), new_status(dcf)
    outs = [torch.empty(tokens, channels, device="cuda") for _ in weights]
    torch.cuda.synchronize()
    for w, out in zip(weights, outs):
        dcf.quantize_async(wplan, w, wq, ws)
        dcf.int8_matmul_async(plan, x, wq, out, work, status, b_scale=ws)
    assert dcf.status_read(status).folded
    q, s = (torch.from_numpy(v).cuda() for v in io.quantize(wide(x), "rows"))
    for w, out in zip(weights, outs):
        wq, ws = (torch.from_numpy(v).cuda() for v in io.quantize(wide(w), "rows"))
        assert torch.equal(out, plain(q, wq, s, ws))


# ------------------------------------------------------------------ gradient

GRADIENTS = [
    ((2000, 500, 1000), 128, False, True), ((2600, 1100, 1030), 128, False, False), ((1500, 3000, 2000), 128, True, False),
    ((600, 513, 2000), 128, False, False),
    ((300, 1024, 4096), 256, False, False), ((700, 2000, 1300), 256, False, False), ((1000, 2048, 4096), 256, True, False),
    ((4001, 1000, 1531), 256, False, True), ((300, 5000, 300), 256, False, False),
]


@pytest.fixture(params=GRADIENTS, ids=["x".join(map(str, size)) for size, *_ in GRADIENTS])
def gradient(request):
    (tokens, channels, depth), tile, many, parts = request.param
    tn, tiles, n = cuts.grad_cut(tokens, channels, depth)
    assert (tn, tiles > cuts.PAIRS, n > 1) == (tile, many, parts)
    return tokens, channels, depth


def exact_grad(g, q, scale):
    """In 64 bits, which hold these sums of whole numbers exactly."""
    x = q.double() * scale.double().repeat_interleave(io.RUN, 0)[:len(q)]
    return g.double().T @ x


@pytest.mark.parametrize("dtype,out", [("bf16", "f32"), ("f16", "bf16"), ("bf16", "f16")])
def test_gradients(dcf, gradient, dtype, out):
    import torch
    g, q, scale = exact_inputs(*gradient, dtype, 1)
    got = run_grad(dcf, g, q, scale, dtype, out=out)
    assert torch.equal(got, exact_grad(g, q, scale).float().to(got.dtype))


def test_gradients_added_to(dcf, gradient):
    import torch
    g, q, scale = exact_inputs(*gradient, "f16", 2)
    onto = whole(gradient[1:], 3).float()
    for pads in ((0, 0, 0), (8, 0, 3)):
        got = run_grad(dcf, g, q, scale, "f16", onto=onto, pads=pads)
        assert torch.equal(got.double(), exact_grad(g, q, scale) + onto.double())


@pytest.mark.parametrize("out,pads,offsets", [("f32", (8, 16, 4), (1, 0, 0)), ("bf16", (8, 3, 2), (7, 5, 0)), ("f16", (3, 0, 1), (0, 0, 1)),
                                              ("f32", (0, 0, 0), (5, 1, 3))])
def test_gradients_in_padded_rows(dcf, gradient, out, pads, offsets):
    import torch
    g, q, scale = exact_inputs(*gradient, "bf16", 4)
    got = run_grad(dcf, g, q, scale, "bf16", out=out, pads=pads, offsets=offsets)
    assert torch.equal(got, exact_grad(g, q, scale).float().to(got.dtype))


@pytest.mark.parametrize("tokens", [300, 6000])
@pytest.mark.parametrize("channels", [121, 125, 127, 128, 249, 250, 255, 256])
@pytest.mark.parametrize("start", [1, 7])
def test_columns_before_a_gradient_that_fill_another_tile(dcf, tokens, channels, start):
    """Rows of whole vectors, the first channel `start` elements into one: the columns before it belong to the tiles."""
    import torch
    depth, pad = 300, 16 - channels % 8
    g, q, scale = exact_inputs(tokens, channels, depth, "bf16", channels)
    assert cuts.grad_cut(tokens, channels, depth, start)[2] > 1 or tokens < 6000
    for out in ("f32", "bf16"):
        got = run_grad(dcf, g, q, scale, "bf16", out=out, pads=(pad, 0, 0), offsets=(start, 0, 0))
        assert torch.equal(got, exact_grad(g, q, scale).float().to(got.dtype))


@pytest.mark.parametrize("channels,depth", [(512, 384), (1100, 1030), (2000, 1300)])
def test_gradients_round_no_more_than_their_runs_do(dcf, channels, depth):
    """8192 tokens are 64 runs.  A rounding of the running sum is 2^-24 / sqrt(3) of it in the mean, and the sums grow as a random
    walk does: 3.44e-8 sqrt(65 / 2) = 2.0e-7 of the result.  Inside a run the tensor core drops what is below a step, half
    of one in the mean (0.72 2^-24 of the sum there), eight times while the sum grows: 4.3e-8 sum sqrt(j / 8) = 2.5e-7 of the
    run, and runs err on their own.  Together 3.2e-7."""
    import torch
    g, q = randn((8192, channels), "bf16", 1), whole((8192, depth), 2)
    scale = randn((64, depth), "f32", 3).abs() * 0.01 + 1e-3
    want = exact_grad(g, q, scale)
    got = run_grad(dcf, g, q, scale, "bf16").double()
    error = float(torch.linalg.norm(got - want) / torch.linalg.norm(want))
    assert error <= 3.2e-7, error
