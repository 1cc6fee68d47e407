"""The operators on 8-bit integers on the GPU against statements of them in numpy."""
import math

import numpy as np
import pytest

import int8_oracle as io

pytestmark = pytest.mark.gpu


def tdtype(name):
    import torch
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "i8": torch.int8,
            "i32": torch.int32}[name]


def wide(t) -> np.ndarray:
    return t.double().cpu().numpy()


def rounded(x: np.ndarray, dtype: str):
    """f32 values rounded once to a type, as a tensor on the GPU."""
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).cuda().to(tdtype(dtype))


def same(got, want) -> bool:
    """Equal bits, NaN equal to NaN."""
    import torch
    return torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0, math.inf, -math.inf),
                                                                 want.nan_to_num(0.0, math.inf, -math.inf))


def randn(shape, dtype, seed, scale=1.0):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=gen, dtype=torch.float64) * scale).to(tdtype(dtype))


def whole(shape, seed, most=127):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-most, most + 1, shape, device="cuda", generator=gen, dtype=torch.int32).to(torch.int8)


class Room:
    """A [rows, cols] view inside memory that is filled with a mark, to see that nothing else is written."""

    def __init__(self, rows, cols, dtype, stride=0, offset=0, mark=77):
        import torch
        self.stride, self.offset, self.mark = stride or cols, offset, mark
        self.flat = torch.full((offset + rows * self.stride + 40,), mark, dtype=tdtype(dtype), device="cuda")
        self.view = self.flat[offset:].as_strided((rows, cols), (self.stride, 1))

    def put(self, t):
        self.view.copy_(t)
        return self

    def untouched(self) -> bool:
        kept = self.view.clone()
        self.view.fill_(self.mark)
        ok = bool((self.flat == self.mark).all())
        self.view.copy_(kept)
        return ok


def new_status(dcf):
    import torch
    st = torch.empty(2, dtype=torch.int64, device="cuda")
    dcf.status_reset(st)
    return st


# ------------------------------------------------------------- quantising


def run_quantize(dcf, x, dtype, along, *, pad=0, q_pad=0, offset=0, q_offset=0):
    import torch
    rows, cols = x.shape
    plan = dcf.quantize_plan(dtype, rows, cols, along=along, row_stride=cols + pad, q_row_stride=cols + q_pad)
    a = Room(rows, cols, dtype, cols + pad, offset).put(x)
    q = Room(rows, cols, "i8", cols + q_pad, q_offset)
    scale = torch.full((plan.scales + 3,), 5.0, device="cuda")
    dcf.quantize_async(plan, a.view, q.view, scale)
    back = Room(rows, cols, dtype, cols + pad, offset)
    dcf.dequantize_async(plan, q.view, scale, back.view)
    assert q.untouched() and back.untouched() and (scale[plan.scales:] == 5.0).all()
    return q.view.cpu().numpy(), scale[:plan.scales].reshape(plan.scale_shape).cpu().numpy(), back.view


def check_quantize(dcf, x, dtype, along, **kw):
    q, scale, back = run_quantize(dcf, x, dtype, along, **kw)
    want_q, want_s = io.quantize(wide(x), along)
    assert np.array_equal(scale, want_s, equal_nan=True)
    assert np.array_equal(q, want_q)
    assert same(back, rounded(io.values(want_q, want_s, along), dtype))


SIZES = [(1, 1), (1, 7), (1, 4096), (2, 33), (3, 1000), (127, 64), (128, 128), (129, 130), (300, 257), (5, 8193),
         (257, 1023), (9, 1024), (2, 20000), (1, 70001)]


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("along", ["rows", "columns"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_quantize_sizes(dcf, rows, cols, along, dtype):
    check_quantize(dcf, randn((rows, cols), dtype, rows + cols), dtype, along)


@pytest.mark.parametrize("along", ["rows", "columns"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("pad,q_pad,offset,q_offset", [(8, 8, 0, 0), (3, 3, 0, 0), (8, 1, 0, 0), (1, 8, 0, 0),
                                                       (8, 8, 1, 0), (8, 8, 0, 3), (8, 8, 8, 8), (24, 40, 4, 4)])
def test_quantize_strides_and_what_lies_between(dcf, along, dtype, pad, q_pad, offset, q_offset):
    check_quantize(dcf, randn((140, 136), dtype, 3), dtype, along, pad=pad, q_pad=q_pad, offset=offset, q_offset=q_offset)


@pytest.mark.parametrize("along", ["rows", "columns"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_quantize_ties_and_borders(dcf, along, dtype):
    """Values around every half, beside a largest one of 127 (where ties are exact) and of one."""
    import torch
    steps = torch.arange(-254, 255, device="cuda", dtype=torch.float64) / 2
    near = torch.cat([steps, steps * (1 + 2.0 ** -22), steps * (1 - 2.0 ** -22)])
    rows = [torch.cat([near * unit, torch.tensor([127 * unit], device="cuda", dtype=torch.float64)])
            for unit in (1.0, 1 / 127, 0.3, 2.0 ** -10, 3.7)]
    x = torch.stack(rows).to(tdtype(dtype))
    check_quantize(dcf, x if along == "rows" else x.T.contiguous()[-128:], dtype, along)
    check_quantize(dcf, x if along == "rows" else x.T.contiguous(), dtype, along)


@pytest.mark.parametrize("along", ["rows", "columns"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_quantize_zeros_infinities_and_the_ends_of_the_range(dcf, along, dtype):
    import torch
    big = float(torch.finfo(tdtype(dtype)).max)
    tiny = float(torch.finfo(tdtype(dtype)).smallest_normal)
    x = randn((12, 40), "f32", 5).double()
    x[0] = 0
    x[1] = -0.0
    x[2, 3] = math.nan
    x[3, 39] = math.inf
    x[4, 0] = -math.inf
    x[5] *= tiny
    x[6] = 0
    x[6, 7] = big
    x[7] = -big
    x[8] *= 2.0 ** -119
    x[9] = 2.0 ** -119 if dtype != "f16" else 2.0 ** -24
    x[10] *= tiny / 8
    x[11] = math.nan
    x = x.to(tdtype(dtype))
    check_quantize(dcf, x if along == "rows" else x.T.contiguous(), dtype, along)


def test_quantize_a_nan_spoils_its_own_run_only(dcf):
    x = randn((300, 24), "bf16", 6)
    x[130, 5] = math.nan
    q, scale, back = run_quantize(dcf, x, "bf16", "columns")
    assert np.isnan(scale[1, 5]) and np.isnan(scale).sum() == 1
    assert back[128:256, 5].isnan().all() and back.isnan().sum() == 128


def test_quantize_empty(dcf):
    import torch
    plan = dcf.quantize_plan("bf16", 0, 8)
    empty = torch.empty(0, 8, dtype=torch.bfloat16, device="cuda")
    dcf.quantize_async(plan, empty, empty.to(torch.int8), torch.empty(0, device="cuda"))
    # rows without columns: nothing is there, and their scale says so
    plan = dcf.quantize_plan("bf16", 5, 0)
    scale = torch.full((5,), 3.0, device="cuda")
    empty = torch.empty(5, 0, dtype=torch.bfloat16, device="cuda")
    dcf.quantize_async(plan, empty, empty.to(torch.int8), scale)
    dcf.dequantize_async(plan, empty.to(torch.int8), scale, empty)
    assert (scale == 0).all()


def test_dequantize_any_whole_number_and_scale(dcf):
    """All 256 bytes, -128 among them, and scales from a checkpoint of someone else's."""
    import torch
    q = torch.arange(-128, 128, device="cuda").to(torch.int8).repeat(5, 1)
    scale = torch.tensor([1.0, -2.5, 3e38, 1e-45, math.inf], device="cuda")
    for dtype in ("f16", "bf16", "f32"):
        plan = dcf.quantize_plan(dtype, 5, 256)
        out = torch.empty(5, 256, dtype=tdtype(dtype), device="cuda")
        dcf.dequantize_async(plan, q, scale, out)
        assert same(out, rounded(io.values(q.cpu().numpy(), scale.cpu().numpy(), "rows"), dtype))


# ---------------------------------------------------------------- product


def run_matmul(dcf, a, b, *, a_dtype="i8", out="bf16", a_scale=None, b_scale=None, bias=None, pads=(0, 0, 0),
               offsets=(0, 0, 0)):
    import torch
    (tokens, depth), channels = a.shape, b.shape[0]
    plan = dcf.int8_matmul_plan(tokens, channels, depth, a_dtype=a_dtype, out_dtype=out, a_row_stride=depth + pads[0],
                                b_row_stride=depth + pads[1], out_row_stride=channels + pads[2])
    x = Room(tokens, depth, a_dtype, depth + pads[0], offsets[0]).put(a)
    w = Room(channels, depth, "i8", depth + pads[1], offsets[1]).put(b)
    to = Room(tokens, channels, out, channels + pads[2], offsets[2])
    work = torch.full((plan.workspace + 64,), 0x5A, dtype=torch.uint8, device="cuda")
    status = new_status(dcf)
    dcf.int8_matmul_async(plan, x.view, w.view, to.view, work, status, a_scale=a_scale, b_scale=b_scale, bias=bias)
    assert dcf.status_read(status).folded
    assert to.untouched() and (work[plan.workspace:] == 0x5A).all()
    return to.view


def scales_for(tokens, channels, seed):
    import torch
    a, b = randn((tokens,), "f32", seed).abs() * 0.03 + 1e-3, randn((channels,), "f32", seed + 1).abs() * 0.01 + 1e-4
    return a, b, randn((channels,), "f32", seed + 2).to(torch.float32)


def check_matmul(dcf, tokens, channels, depth, out, *, bias=False, seed=0, **kw):
    a, b = whole((tokens, depth), seed), whole((channels, depth), seed + 1)
    sa, sb, add = scales_for(tokens, channels, seed + 2)
    if out == "i32":
        got = run_matmul(dcf, a, b, out=out, **kw)
        assert np.array_equal(got.cpu().numpy(), io.matmul(a.cpu().numpy(), None, b.cpu().numpy(), None, None))
        return
    got = run_matmul(dcf, a, b, out=out, a_scale=sa, b_scale=sb, bias=add if bias else None, **kw)
    want = io.matmul(a.cpu().numpy(), sa.cpu().numpy(), b.cpu().numpy(), sb.cpu().numpy(), add.cpu().numpy() if bias else None)
    assert same(got, rounded(want, out))


MM = [(1, 1, 1), (1, 1, 0), (1, 5, 16), (1, 300, 1000), (2, 64, 64), (3, 129, 257), (5, 17, 4096), (8, 256, 128), (9, 33, 100),
      (17, 500, 31), (31, 64, 2048), (33, 40, 63), (64, 64, 64), (65, 257, 129), (100, 384, 512), (127, 128, 1000),
      (130, 250, 272), (255, 513, 96), (257, 256, 160), (300, 1000, 333), (520, 264, 1040)]


@pytest.mark.parametrize("tokens,channels,depth", MM)
@pytest.mark.parametrize("out", ["i32", "f32", "bf16"])
def test_matmul_sizes(dcf, tokens, channels, depth, out):
    check_matmul(dcf, tokens, channels, depth, out, bias=depth % 2 == 0, seed=tokens + depth)


@pytest.mark.parametrize("tokens", [3, 40, 200])
@pytest.mark.parametrize("out", ["f16", "f32", "i32"])
@pytest.mark.parametrize("pads,offsets", [((16, 0, 0), (0, 0, 0)), ((0, 16, 3), (0, 0, 0)), ((3, 0, 8), (0, 0, 0)),
                                          ((0, 5, 0), (0, 0, 1)), ((16, 16, 16), (1, 0, 0)), ((16, 16, 16), (0, 7, 0)),
                                          ((16, 16, 16), (16, 32, 8)), ((1, 1, 1), (1, 1, 1))])
def test_matmul_strides_and_what_lies_between(dcf, tokens, out, pads, offsets):
    check_matmul(dcf, tokens, 136, 160, out, bias=out == "f32", pads=pads, offsets=offsets)


@pytest.mark.parametrize("tokens", [1, 4, 24, 130])
def test_matmul_largest_sums(dcf, tokens):
    """-128 times -128 over the longest depth is 2^31 - 2^14, and f32 takes all of it in one rounding."""
    import torch
    depth = dcf.INT8_MAX_DEPTH
    a = torch.full((tokens, depth), -128, dtype=torch.int8, device="cuda")
    b = torch.full((3, depth), -128, dtype=torch.int8, device="cuda")
    b[1] = 127
    b[2, 1:] = 0
    want = np.tile(np.array([[1 << 14], [-128 * 127], [0]]).T * depth, (tokens, 1))
    want[:, 2] = 1 << 14
    assert np.array_equal(run_matmul(dcf, a, b, out="i32").cpu().numpy(), want)
    one = torch.ones(max(tokens, 3), device="cuda")
    got = run_matmul(dcf, a, b, out="f32", a_scale=one[:tokens].contiguous(), b_scale=one[:3].contiguous())
    assert np.array_equal(got.cpu().numpy(), want.astype(np.float32))


@pytest.mark.parametrize("tokens", [2, 50])
def test_matmul_scales_of_no_use(dcf, tokens):
    """Scales of 0, NaN, infinity and either sign go into their own rows and columns."""
    a, b = whole((tokens, 64), 1), whole((70, 64), 2)
    sa, sb, add = scales_for(tokens, 70, 3)
    sa[0], sb[1], sb[2], sb[3] = math.nan, 0.0, math.inf, -sb[3]
    add[5] = math.nan
    for out in ("f16", "bf16", "f32"):
        got = run_matmul(dcf, a, b, out=out, a_scale=sa, b_scale=sb, bias=add)
        want = io.matmul(a.cpu().numpy(), sa.cpu().numpy(), b.cpu().numpy(), sb.cpu().numpy(), add.cpu().numpy())
        assert same(got, rounded(want, out))


@pytest.mark.parametrize("tokens,channels,depth", [(1, 40, 64), (1, 300, 4096), (3, 70, 1001), (8, 128, 512), (20, 256, 300),
                                                   (129, 130, 131), (256, 64, 2048)])
@pytest.mark.parametrize("a_dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_matmul_quantises_its_tokens_as_the_operator_does(dcf, tokens, channels, depth, a_dtype, out):
    x, b = randn((tokens, depth), a_dtype, 7), whole((channels, depth), 8)
    if tokens > 2:
        x[1] = 0
        x[2, depth // 2] = math.inf
    _, sb, add = scales_for(tokens, channels, 9)
    got = run_matmul(dcf, x, b, a_dtype=a_dtype, out=out, b_scale=sb, bias=add, pads=(depth % 3, 0, 0))
    q, s = io.quantize(wide(x), "rows")
    want = io.matmul(q, s, b.cpu().numpy(), sb.cpu().numpy(), add.cpu().numpy())
    assert same(got, rounded(want, out))


# ------------------------------------------------- gradient from a checkpoint


def run_grad(dcf, g, q, scale, dtype, *, out="f32", pads=(0, 0, 0), offsets=(0, 0, 0), onto=None):
    import torch
    (tokens, channels), depth = g.shape, q.shape[1]
    plan = dcf.checkpoint_grad_plan(dtype, tokens, channels, depth, out_dtype=out, grad_row_stride=channels + pads[0],
                                    q_row_stride=depth + pads[1], out_row_stride=depth + pads[2], accumulate=onto is not None)
    x = Room(tokens, channels, dtype, channels + pads[0], offsets[0]).put(g)
    a = Room(tokens, depth, "i8", depth + pads[1], offsets[1]).put(q)
    to = Room(channels, depth, out, depth + pads[2], offsets[2])
    if onto is not None:
        to.put(onto)
    work = torch.full((plan.workspace + 64,), 0x5A, dtype=torch.uint8, device="cuda")
    status = new_status(dcf)
    dcf.checkpoint_grad_async(plan, x.view, a.view, scale, to.view, work, status)
    assert dcf.status_read(status).folded
    assert to.untouched() and (work[plan.workspace:] == 0x5A).all()
    return to.view


def exact_inputs(tokens, channels, depth, dtype, seed):
    """Whole numbers and powers of two whose sums are exact in f32: |g| <= 4, |q| <= 15, scales 1 to 8, so that
    sums stay below 2^24 up to 2^24 / (4 * 15 * 8) = 34952 tokens."""
    import torch
    g, q = whole((tokens, channels), seed, 4).to(tdtype(dtype)), whole((tokens, depth), seed + 1, 15)
    runs = -(-tokens // io.RUN)
    scale = 2.0 ** whole((runs, depth), seed + 2, 3).abs().float()
    return g, q, scale.to(torch.float32)


GRADS = [(1, 1, 1), (0, 5, 7), (1, 300, 17), (7, 8, 64), (64, 64, 64), (127, 130, 65), (128, 128, 128), (129, 256, 256),
         (200, 257, 100), (256, 40, 300), (300, 513, 129), (1000, 64, 520), (2049, 96, 264), (4000, 31, 33), (513, 260, 1000)]


@pytest.mark.parametrize("tokens,channels,depth", GRADS)
@pytest.mark.parametrize("dtype,out", [("bf16", "f32"), ("f16", "f32"), ("bf16", "bf16"), ("f16", "f16")])
def test_grad_of_whole_numbers_is_exact(dcf, tokens, channels, depth, dtype, out):
    g, q, scale = exact_inputs(tokens, channels, depth, dtype, tokens + channels)
    want, _ = io.grad(wide(g), q.cpu().numpy(), scale.cpu().numpy())
    assert same(run_grad(dcf, g, q, scale, dtype, out=out), rounded(want.astype(np.float32), out))


@pytest.mark.parametrize("pads,offsets", [((8, 16, 4), (0, 0, 0)), ((3, 0, 0), (0, 0, 0)), ((0, 3, 0), (0, 0, 0)),
                                          ((0, 0, 1), (0, 0, 0)), ((8, 16, 4), (1, 0, 0)), ((8, 16, 4), (0, 5, 0)),
                                          ((8, 16, 4), (0, 0, 1)), ((8, 16, 4), (8, 16, 4)), ((1, 1, 1), (1, 1, 1)),
                                          ((0, 0, 0), (3, 0, 0)), ((0, 0, 0), (7, 9, 3))])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_grad_strides_and_what_lies_between(dcf, pads, offsets, out):
    g, q, scale = exact_inputs(300, 136, 160, "bf16", 4)
    want, _ = io.grad(wide(g), q.cpu().numpy(), scale.cpu().numpy())
    assert same(run_grad(dcf, g, q, scale, "bf16", out=out, pads=pads, offsets=offsets), rounded(want.astype(np.float32), out))


@pytest.mark.parametrize("tokens,channels,depth", [(1, 40, 50), (128, 128, 64), (1000, 200, 300), (6000, 130, 70), (8192, 256, 256)])
@pytest.mark.parametrize("dtype,out", [("bf16", "f32"), ("f16", "f32"), ("bf16", "bf16"), ("f16", "f16")])
def test_grad_against_64_bits(dcf, tokens, channels, depth, dtype, out):
    """Each of a run's 128 additions, each run's product and addition, and their parts' joining (32 parts at most)
    may be off by a step of 2^-23 of the magnitudes summed; a 16-bit result by half a step more, 2^-25 at least in f16."""
    g, q = randn((tokens, channels), dtype, 1), whole((tokens, depth), 2)
    runs = -(-tokens // io.RUN)
    scale = randn((runs, depth), "f32", 3).abs() * 0.01 + 1e-4
    got = wide(run_grad(dcf, g, q, scale, dtype, out=out))
    want, size = io.grad(wide(g), q.cpu().numpy(), scale.cpu().numpy())
    bound = (min(tokens, io.RUN) + 2 * runs + 32) * 2.0 ** -23 * size
    if out != "f32":
        bound = bound + np.abs(want) * {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}[out] + (2.0 ** -25 if out == "f16" else 0)
    assert (np.abs(got - want) <= bound).all()


def test_grad_is_as_near_to_64_bits_as_fp32_products(dcf):
    """The product of f32 values, which rounds every addition, against the gradient: over 8192 tokens both err by
    their additions alone.  A run's sum here rounds once in 16 products at the most, a f32 product's every time."""
    import torch
    g, q = randn((8192, 512), "bf16", 1), whole((8192, 384), 2)
    scale = randn((64, 384), "f32", 3).abs() * 0.01 + 1e-3
    want, _ = io.grad(wide(g), q.cpu().numpy(), scale.cpu().numpy())
    got = wide(run_grad(dcf, g, q, scale, "bf16"))
    plain = wide(g.float().T @ (q.float() * scale.repeat_interleave(io.RUN, 0)))
    norm = np.linalg.norm(want)
    here, there = np.linalg.norm(got - want) / norm, np.linalg.norm(plain - want) / norm
    assert here <= max(1.5 * there, 1e-6), (here, there)


def test_grad_is_the_differences_of_the_layer(dcf):
    """loss = sum(g * (x w^T)) is linear in w: moving one weight by one changes it by exactly that gradient."""
    import torch
    g, q, scale = exact_inputs(150, 6, 9, "bf16", 5)
    x = q.double() * scale.double().repeat_interleave(io.RUN, 0)[:150]
    w = torch.zeros(6, 9, dtype=torch.float64, device="cuda")
    grad = run_grad(dcf, g, q, scale, "bf16").double()

    def loss(w):
        return (g.double() * (x @ w.T)).sum()

    for c, k in ((0, 0), (5, 8), (3, 4), (2, 7)):
        step = torch.zeros_like(w)
        step[c, k] = 1
        assert loss(w + step) - loss(w) == grad[c, k]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_grad_of_every_whole_number(dcf, dtype):
    """All 256 bytes, -128 among them, each picked out by a token of its own."""
    import torch
    g = torch.eye(256, device="cuda").to(tdtype(dtype))
    q = torch.arange(-128, 128, device="cuda").to(torch.int8)[:, None].repeat(1, 20)
    scale = torch.tensor([[1.0], [0.5]], device="cuda").repeat(1, 20)
    got = run_grad(dcf, g, q, scale, dtype)
    want = q.float() * scale.repeat_interleave(128, 0)
    assert torch.equal(got, want)


def test_matmul_of_no_depth(dcf):
    """Float tokens without a single value: nothing but the bias is left."""
    import torch
    for tokens in (2, 40):
        x, b = torch.empty(tokens, 0, dtype=torch.bfloat16, device="cuda"), torch.empty(6, 0, dtype=torch.int8, device="cuda")
        _, sb, add = scales_for(tokens, 6, 1)
        assert torch.equal(run_matmul(dcf, x, b, a_dtype="bf16", out="f32", b_scale=sb, bias=add), add.repeat(tokens, 1))
    fold, scale = dcf.quantize(dcf.quantize_plan("f32", 5, 0), np.empty((5, 0), np.float32))
    assert fold.folded and (scale == 0).all()


@pytest.mark.parametrize("tokens,channels,depth", [(300, 70, 90), (300, 256, 256), (130, 600, 520), (6000, 128, 40), (2, 400, 33)])
def test_grad_adds_to_what_is_there(dcf, tokens, channels, depth):
    g, q, scale = exact_inputs(tokens, channels, depth, "f16", 6)
    onto = whole((channels, depth), 9).float()
    want, _ = io.grad(wide(g), q.cpu().numpy(), scale.cpu().numpy())
    assert same(run_grad(dcf, g, q, scale, "f16", onto=onto), rounded((want + wide(onto)).astype(np.float32), "f32"))
    none = run_grad(dcf, g[:0], q[:0], scale[:0], "f16", onto=onto)
    assert same(none, onto)


@pytest.mark.parametrize("tokens", [100, 700])
def test_grad_of_infinities_and_spoilt_runs(dcf, tokens):
    """NaN and infinities reach exactly the results that they are part of."""
    g, q, scale = exact_inputs(tokens, 40, 50, "bf16", 7)
    g[3, 5], g[60, 6] = math.nan, math.inf
    q[60, 7], q[60, 8], q[60, 9] = 2, -2, 0
    scale[0, 11] = math.nan
    scale[-1, 12] = math.inf
    got = run_grad(dcf, g, q, scale, "bf16")
    want, _ = io.grad(wide(g), q.cpu().numpy(), scale.cpu().numpy())
    assert got[5].isnan().all() and got[:, 11].isnan().all()
    assert got[6, 7] == math.inf and got[6, 8] == -math.inf and got[6, 9].isnan()
    fine = np.isfinite(want)
    assert np.array_equal(wide(got)[fine], want[fine])
    assert not np.isfinite(wide(got))[~fine].any()


# ----------------------------------------------------------- all of them


def test_layer_forward_checkpoint_backward_and_step(dcf):
    """A layer as a training step runs it: its product with an 8-bit weight, the checkpoint of its input, the weight's
    gradient from that, and the orthogonalised gradient; each against what its own inputs say."""
    import torch
    tokens, channels, depth = 300, 200, 264
    x, w = randn((tokens, depth), "bf16", 1), randn((channels, depth), "bf16", 2, 0.05)
    wplan = dcf.quantize_plan("bf16", channels, depth)
    wq, ws = torch.empty(channels, depth, dtype=torch.int8, device="cuda"), torch.empty(channels, device="cuda")
    dcf.quantize_async(wplan, w, wq, ws)
    mm = dcf.int8_matmul_plan(tokens, channels, depth, a_dtype="bf16")
    y, status = torch.empty(tokens, channels, dtype=torch.bfloat16, device="cuda"), new_status(dcf)
    work = torch.empty(dcf.int8_matmul_workspace(mm), dtype=torch.uint8, device="cuda")
    dcf.int8_matmul_async(mm, x, wq, y, work, status, b_scale=ws)
    cplan = dcf.quantize_plan("bf16", tokens, depth, along="columns")
    q, s = torch.empty(tokens, depth, dtype=torch.int8, device="cuda"), torch.empty(*cplan.scale_shape, device="cuda")
    dcf.quantize_async(cplan, x, q, s)
    g = dcf.checkpoint_grad_plan("bf16", tokens, channels, depth)
    dw = torch.empty(channels, depth, device="cuda")
    gwork = torch.empty(dcf.checkpoint_grad_workspace(g), dtype=torch.uint8, device="cuda")
    dcf.checkpoint_grad_async(g, y, q, s, dw, gwork, status)
    orth = dcf.orthogonalize_plan("f32", channels, depth)
    step = torch.empty_like(dw)
    owork = torch.empty(dcf.orthogonalize_workspace(orth), dtype=torch.uint8, device="cuda")
    dcf.orthogonalize_async(orth, dw, step, owork, status)
    assert dcf.status_read(status).folded
    want_wq, want_ws = io.quantize(wide(w), "rows")
    assert np.array_equal(wq.cpu().numpy(), want_wq) and np.array_equal(ws.cpu().numpy(), want_ws)
    xq, xs = io.quantize(wide(x), "rows")
    assert same(y, rounded(io.matmul(xq, xs, want_wq, want_ws, None), "bf16"))
    want_q, want_s = io.quantize(wide(x), "columns")
    assert np.array_equal(q.cpu().numpy(), want_q) and np.array_equal(s.cpu().numpy(), want_s)
    want, size = io.grad(wide(y), want_q, want_s)
    assert (np.abs(wide(dw) - want) <= (io.RUN + 2 * 3 + 32) * 2.0 ** -23 * size).all()
    sv = torch.linalg.svdvals(step)
    assert sv.max() < 1.3                                 # what the quintic leaves of the largest
    # the checkpoint stands for the input to half a step of its column's scale, and bf16's own rounding
    values = torch.empty_like(x)
    dcf.dequantize_async(cplan, q, s, values)
    half = wide(s).repeat(io.RUN, 0)[:tokens] / 2
    assert (np.abs(wide(values) - wide(x)) <= half * (1 + 2.0 ** -20) + np.abs(wide(values)) * 2.0 ** -8).all()


# ------------------------------------- streams, graphs, large offsets, many rows


def calls_of(dcf, seed, tokens=300, channels=200, depth=264):
    """Every operator once, on buffers of its own: (inputs, outputs, a function that queues all of them)."""
    import torch
    x, w = randn((tokens, depth), "bf16", seed), randn((channels, depth), "bf16", seed + 1, 0.05)
    cplan, wplan = dcf.quantize_plan("bf16", tokens, depth, along="columns"), dcf.quantize_plan("bf16", channels, depth)
    mm, gp = dcf.int8_matmul_plan(tokens, channels, depth, a_dtype="bf16"), dcf.checkpoint_grad_plan("bf16", tokens, channels, depth)
    status = new_status(dcf)
    room = {n: torch.empty(s, dtype=t, device="cuda") for n, s, t in (
        ("wq", (channels, depth), torch.int8), ("ws", (channels,), torch.float32), ("q", (tokens, depth), torch.int8),
        ("s", cplan.scale_shape, torch.float32), ("y", (tokens, channels), torch.bfloat16), ("dw", (channels, depth), torch.float32),
        ("back", (tokens, depth), torch.bfloat16), ("work", (max(mm.workspace, gp.workspace),), torch.uint8))}

    def queue(stream=None):
        dcf.quantize_async(wplan, w, room["wq"], room["ws"], stream=stream)
        dcf.int8_matmul_async(mm, x, room["wq"], room["y"], room["work"], status, b_scale=room["ws"], stream=stream)
        dcf.quantize_async(cplan, x, room["q"], room["s"], stream=stream)
        dcf.dequantize_async(cplan, room["q"], room["s"], room["back"], stream=stream)
        dcf.checkpoint_grad_async(gp, room["y"], room["q"], room["s"], room["dw"], room["work"], status, stream=stream)

    return (x, w), room, queue


def results(room):
    return [room[n].clone() for n in ("wq", "ws", "q", "s", "back", "y", "dw")]


def equal(a, b) -> bool:
    import torch
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_equal_calls_give_equal_bits_on_two_streams_at_once(dcf):
    import torch
    sets = [calls_of(dcf, 10 * k, depth=264 if k else 4096, tokens=300 + 77 * k) for k in range(2)]
    want = []
    for _, room, queue in sets:
        queue()
        torch.cuda.synchronize()
        want.append(results(room))
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(20):
        for (_, _, queue), stream in zip(sets, streams):
            queue(stream)
    torch.cuda.synchronize()
    for (_, room, _), w in zip(sets, want):
        assert equal(results(room), w)


def test_captured_and_replayed_on_new_inputs(dcf):
    import torch
    (x, w), room, queue = calls_of(dcf, 3)
    (x2, w2), room2, queue2 = calls_of(dcf, 50)
    queue2()
    torch.cuda.synchronize()
    want = results(room2)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        queue()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            queue()
    x.copy_(x2)
    w.copy_(w2)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert equal(results(room), want)


def test_graphs_that_share_a_workspace_one_after_the_other(dcf):
    import torch
    one, two = calls_of(dcf, 4), calls_of(dcf, 60, tokens=1000)
    two[1]["work"] = one[1]["work"] = torch.empty(max(one[1]["work"].numel(), two[1]["work"].numel()), dtype=torch.uint8, device="cuda")
    graphs, want = [], []
    stream = torch.cuda.Stream()
    for _, room, queue in (one, two):
        with torch.cuda.stream(stream):
            queue()
            torch.cuda.synchronize()
            want.append(results(room))
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                queue()
            graphs.append(g)
    for _ in range(5):
        graphs[0].replay()
        graphs[1].replay()
    torch.cuda.synchronize()
    assert equal(results(one[1]), want[0]) and equal(results(two[1]), want[1])


def test_rows_past_32_bits_of_elements(dcf):
    """Two rows 2^31 and some elements apart, in every operand that has rows."""
    import torch
    far = (1 << 31) + 16
    big = torch.empty(far + 4096, dtype=torch.bfloat16, device="cuda")
    bytes_ = torch.empty(far + 4096, dtype=torch.int8, device="cuda")
    x, b = randn((2, 256), "bf16", 1), whole((2, 256), 2)
    values, levels = big.as_strided((2, 256), (far, 1)), bytes_.as_strided((2, 256), (far, 1))
    values.copy_(x)
    for along in ("rows", "columns"):
        plan = dcf.quantize_plan("bf16", 2, 256, along=along, row_stride=far, q_row_stride=far)
        scale = torch.empty(*plan.scale_shape, device="cuda")
        dcf.quantize_async(plan, values, levels, scale)
        want_q, want_s = io.quantize(wide(x), along)
        assert np.array_equal(levels.cpu().numpy(), want_q) and np.array_equal(scale.cpu().numpy(), want_s)
        back = big[512:].as_strided((2, 256), (far, 1))
        dcf.dequantize_async(plan, levels, scale, back)
        assert same(back, rounded(io.values(want_q, want_s, along), "bf16"))
    levels.copy_(b)
    tokens = whole((40, 256), 3)
    # the weight's rows, and a result's
    for a in (tokens, tokens[:2]):
        n = len(a)
        p = dcf.int8_matmul_plan(n, 2, 256, out_dtype="i32", b_row_stride=far)
        out, work, st = torch.empty(n, 2, dtype=torch.int32, device="cuda"), torch.empty(p.workspace, dtype=torch.uint8, device="cuda"), new_status(dcf)
        dcf.int8_matmul_async(p, a, levels, out, work, st)
        assert np.array_equal(out.cpu().numpy(), io.matmul(a.cpu().numpy(), None, b.cpu().numpy(), None, None))
    p = dcf.int8_matmul_plan(2, 40, 256, out_dtype="bf16", a_row_stride=far, out_row_stride=far)
    sa, sb, _ = scales_for(2, 40, 4)
    work = torch.empty(p.workspace, dtype=torch.uint8, device="cuda")
    to = big[1024:].as_strided((2, 40), (far, 1))
    dcf.int8_matmul_async(p, levels, tokens, to, work, st, a_scale=sa, b_scale=sb)
    assert same(to, rounded(io.matmul(b.cpu().numpy(), sa.cpu().numpy(), tokens.cpu().numpy(), sb.cpu().numpy(), None), "bf16"))
    # a gradient's rows, a checkpoint's, and a result's
    g, q, scale = exact_inputs(2, 2, 256, "bf16", 5)
    values[:, :2].copy_(g)
    levels.copy_(q)
    p = dcf.checkpoint_grad_plan("bf16", 2, 2, 256, out_dtype="bf16", grad_row_stride=far, q_row_stride=far, out_row_stride=far)
    work, to = torch.empty(p.workspace, dtype=torch.uint8, device="cuda"), big[2048:].as_strided((2, 256), (far, 1))
    dcf.checkpoint_grad_async(p, values[:, :2], levels, scale, to, work, st)
    want, _ = io.grad(wide(g), q.cpu().numpy(), scale.cpu().numpy())
    assert same(to, rounded(want.astype(np.float32), "bf16"))
    assert dcf.status_read(st).folded


def test_many_rows(dcf):
    """More rows, tokens and runs than a grid's second dimension has blocks."""
    rows = 9_000_000
    x = randn((rows, 2), "bf16", 1)
    check_quantize(dcf, x, "bf16", "rows")
    check_quantize(dcf, x, "bf16", "columns")
    check_matmul(dcf, 300_000, 3, 5, "f32", seed=1)
    check_matmul(dcf, 3, 300_000, 5, "bf16", seed=2)
    check_matmul(dcf, 70, 70_001, 16, "i32", seed=3)
    for tokens, channels, depth in ((30_000, 3, 5), (5, 70_001, 3), (130, 2, 70_001)):
        g, q, scale = exact_inputs(tokens, channels, depth, "bf16", tokens)
        want, _ = io.grad(wide(g), q.cpu().numpy(), scale.cpu().numpy())
        assert same(run_grad(dcf, g, q, scale, "bf16"), rounded(want.astype(np.float32), "f32"))


def test_host_forms(dcf):
    x = randn((140, 40), "f32", 1).cpu().numpy()
    for along in ("rows", "columns"):
        plan = dcf.quantize_plan("f32", 140, 40, along=along)
        fold, scale = dcf.quantize(plan, x)
        q, s = io.quantize(x.astype(np.float64), along)
        assert fold.folded and not fold.is_splat and np.array_equal(fold.out, q) and np.array_equal(scale, s)
        back = dcf.dequantize(plan, q, s)
        assert np.array_equal(back.out.view(np.float32), io.values(q, s, along))
    rng = np.random.default_rng(2)
    a, b = rng.integers(-127, 128, (50, 40)).astype(np.int8), rng.integers(-127, 128, (9, 40)).astype(np.int8)
    sa, sb, add = (rng.random(n).astype(np.float32) for n in (50, 9, 9))
    got = dcf.int8_matmul(dcf.int8_matmul_plan(50, 9, 40, out_dtype="f32"), a, b, a_scale=sa, b_scale=sb, bias=add)
    assert np.array_equal(got.out.view(np.float32), io.matmul(a, sa, b, sb, add))
    got = dcf.int8_matmul(dcf.int8_matmul_plan(50, 9, 40, out_dtype="i32"), a, b)
    assert np.array_equal(got.out.view(np.int32), io.matmul(a, None, b, None, None))
    got = dcf.int8_matmul(dcf.int8_matmul_plan(140, 9, 40, a_dtype="f32", out_dtype="f32"), x, b, b_scale=sb)
    assert np.array_equal(got.out.view(np.float32), io.matmul(*io.quantize(x.astype(np.float64), "rows"), b, sb, None))
    g, q, scale = (t.cpu().numpy() for t in exact_inputs(300, 7, 40, "f16", 3))
    onto = np.ones((7, 40), np.float32)
    want, _ = io.grad(g.astype(np.float64), q, scale)
    assert np.array_equal(dcf.checkpoint_grad(dcf.checkpoint_grad_plan("f16", 300, 7, 40), g, q, scale).out.view(np.float32), want)
    got = dcf.checkpoint_grad(dcf.checkpoint_grad_plan("f16", 300, 7, 40, accumulate=True), g, q, scale, out=onto)
    assert np.array_equal(got.out, want + 1)
