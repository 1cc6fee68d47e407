"""The 8-bit product of weights and tokens that end where their memory ends, on the GPU."""
import numpy as np
import pytest

import int8_oracle as io
from test_gpu_int8 import new_status, rounded, same, scales_for, whole

pytestmark = pytest.mark.gpu


def at_the_end(t, stride: int, before: int):
    """A copy of an int8 matrix whose last byte is the last one of its storage, `before` bytes ahead of it."""
    import torch
    rows, cols = t.shape
    flat = torch.full((before + (rows - 1) * stride + cols,), 77, dtype=torch.int8, device="cuda")
    view = flat[before:].as_strided((rows, cols), (stride, 1))
    view.copy_(t)
    assert before + (rows - 1) * stride + cols == flat.untyped_storage().nbytes()
    return view


def check(dcf, a, b, out="i32"):
    import torch
    (tokens, depth), channels = a.shape, b.shape[0]
    plan = dcf.int8_matmul_plan(tokens, channels, depth, out_dtype=out, a_row_stride=a.stride(0), b_row_stride=b.stride(0))
    to, status = torch.empty(tokens, channels, dtype=getattr(torch, {"i32": "int32", "bf16": "bfloat16"}[out]), device="cuda"), new_status(dcf)
    work = torch.empty(plan.workspace, dtype=torch.uint8, device="cuda")
    sa, sb, add = scales_for(tokens, channels, 5) if out != "i32" else (None, None, None)
    dcf.int8_matmul_async(plan, a, b, to, work, status, a_scale=sa, b_scale=sb, bias=add)
    assert dcf.status_read(status).folded
    host = [None if v is None else v.cpu().numpy() for v in (a, sa, b, sb, add)]
    want = io.matmul(*host)
    if out == "i32":
        assert np.array_equal(to.cpu().numpy(), want)
    else:
        assert same(to, rounded(want, out))


@pytest.mark.parametrize("tokens", [1, 2, 4, 40])
@pytest.mark.parametrize("depth", [1, 5, 15, 16, 17, 31, 100, 497, 513, 1030])
def test_weights_that_end_with_their_memory(dcf, tokens, depth):
    """Whatever the last vector holds of the last rows, and wherever rows start."""
    a = whole((tokens, depth), depth)
    for channels in (1, 2, 9, 37):
        b = whole((channels, depth), depth + channels)
        for before in (0, 1, 7, 15):
            check(dcf, a, at_the_end(b, depth, before))
        check(dcf, a, at_the_end(b, -(-depth // 16) * 16, 0), "bf16")
        check(dcf, a, at_the_end(b, depth + 3, 16))


@pytest.mark.parametrize("tokens", [1, 3, 40, 300])
@pytest.mark.parametrize("stride", [1, 2, 7, 15, 16, 17])
def test_weights_whose_rows_overlap(dcf, tokens, stride):
    """A window that moves along one row of bytes: the last vectors of many rows reach behind the last row."""
    import torch
    channels, depth = 45, 90
    flat = whole(((channels - 1) * stride + depth,), stride)
    for before in (0, 5):
        memory = torch.cat([torch.full((before,), 77, dtype=torch.int8, device="cuda"), flat])
        b = memory[before:].as_strided((channels, depth), (stride, 1))
        check(dcf, whole((tokens, depth), 3), b)


@pytest.mark.parametrize("tokens", [1, 2, 3, 4])
@pytest.mark.parametrize("depth", [1, 15, 17, 40, 1003])
def test_tokens_that_end_with_their_memory(dcf, tokens, depth):
    b = whole((20, depth), 1)
    for stride, before in ((depth, 0), (-(-depth // 16) * 16, 0), (depth, 9), (depth + 1, 16)):
        check(dcf, at_the_end(whole((tokens, depth), 2), stride, before), b)
