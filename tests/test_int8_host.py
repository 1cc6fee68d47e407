"""Operators on 8-bit integers, on the CPU: descriptors and calls that are
refused, workspace sizes, and that a call without a GPU says so."""
import ctypes

import numpy as np
import pytest

import int8_oracle as io
import mlirpass_b200 as m
from conftest import have_gpu


def refused(make, *args, **kw):
    with pytest.raises(m.DcfError) as e:
        make(*args, **kw)
    assert e.value.code == -1, e.value
    return str(e.value)


def last() -> str:
    return m.lib().dcf_last_error().decode()


# Addresses that no call may look behind: every one of these calls is refused before.
A, B, C, D, E, F = (0x100000 * (i + 1) for i in range(6))


def quant_desc(**kw):
    d = dict(dtype=m.DTYPES["bf16"], along=0, rows=8, cols=16, row_stride=0, q_row_stride=0)
    d.update(kw)
    return m.QuantDesc(*d.values())


@pytest.mark.parametrize("kw,word,calls", [
    (dict(dtype=m.DTYPES["f64"]), "dtype", "both"), (dict(dtype=m.DTYPES["i8"]), "dtype", "both"), (dict(dtype=0), "dtype", "both"),
    (dict(along=2), "along", "both"), (dict(rows=1 << 31), "rows", "both"), (dict(cols=(1 << 31) - 65535), "cols", "both"),
    (dict(row_stride=-1), "stride", "both"), (dict(q_row_stride=-16), "stride", "both"),
    (dict(rows=1 << 30, cols=1 << 17), "large", "both"), (dict(row_stride=1 << 44), "large", "both"),
    (dict(q_row_stride=15), "overlap", "quantize"), (dict(row_stride=15), "overlap", "dequantize"),
])
def test_quantize_refusals(kw, word, calls):
    d = ctypes.byref(quant_desc(**kw))
    if calls in ("both", "quantize"):
        assert m.lib().dcf_quantize_async(d, A, B, C, None) == -1 and word in last()
    if calls in ("both", "dequantize"):
        assert m.lib().dcf_dequantize_async(d, B, C, A, None) == -1 and word in last()


def test_quantize_pointers_that_are_refused():
    L = m.lib()
    for along in (0, 1):
        d = ctypes.byref(quant_desc(along=along))
        for args in ((None, B, C), (A, None, C), (A, B, None)):
            assert L.dcf_quantize_async(d, *args, None) == -1 and "null" in last()
            assert L.dcf_dequantize_async(d, args[1], args[2], args[0], None) == -1 and "null" in last()
        # 8 x 16 bf16 are 256 bytes, whole numbers 128, scales 32 or 64
        for args in ((A, A + 255, C), (A, B, A + 252), (A, B, B + 127), (A, A, C)):
            assert L.dcf_quantize_async(d, *args, None) == -1 and "overlap" in last()
        for args in ((A + 255, C, A), (B, A + 252, A)):
            assert L.dcf_dequantize_async(d, *args, None) == -1 and "overlap" in last()
    assert L.dcf_quantize_async(None, A, B, C, None) == -1
    # nothing to do: no pointer is looked at
    for kw in (dict(rows=0), dict(rows=0, along=1), dict(cols=0, along=1)):
        d = ctypes.byref(quant_desc(**kw))
        assert L.dcf_quantize_async(d, None, None, None, None) == 0
        assert L.dcf_dequantize_async(d, None, None, None, None) == 0
    assert L.dcf_dequantize_async(ctypes.byref(quant_desc(cols=0)), None, None, None, None) == 0


def test_parts_of_one_wide_tensor_do_not_overlap():
    """Rows of a result between the rows of an operand, the same stride apart: only what they share is refused."""
    L = m.lib()
    d = quant_desc(dtype=m.DTYPES["f32"], row_stride=64, q_row_stride=256)          # rows of 64 and 16 bytes, 256 apart
    r = ctypes.byref(d)
    for q, meets in ((A + 64, False), (A + 240, False), (A + 63, True), (A + 241, True), (A, True), (A + 256 + 64, False),
                     (A - 256 + 64, False), (A - 16, False), (A - 15, True), (A + 256 * 7 + 63, True), (A + 256 * 7 + 64, False)):
        assert L.dcf_quantize_async(r, A, q, C, None) == -1            # no such memory, at the latest
        assert ("overlap" in last()) == meets, hex(q - A)
        assert L.dcf_dequantize_async(r, q, C, A, None) == -1
        assert ("overlap" in last()) == meets, hex(q - A)
    d.q_row_stride = 255                                                # another stride: any reach into it is refused
    assert L.dcf_quantize_async(r, A, A + 64, C, None) == -1 and "overlap" in last()


def test_quantize_plans():
    for kw in (dict(rows=-1), dict(cols=1 << 31), dict(row_stride=-1)):
        with pytest.raises(ValueError):
            m.quantize_plan("bf16", **{**dict(rows=4, cols=4), **kw})
    with pytest.raises(ValueError):
        m.quantize_plan("f64", 4, 4)
    with pytest.raises(KeyError):
        m.quantize_plan("bf16", 4, 4, along="tensor")
    p = m.quantize_plan("f32", 300, 20, along="columns", row_stride=24)
    assert p.scale_shape == (3, 20) and p.scales == 60
    assert p.values == (299 * 24 + 20, (300, 20), (24, 1)) and p.levels[0] == 6000


@pytest.mark.parametrize("kw,word", [
    (dict(a_dtype="f64"), "a must"), (dict(a_dtype="i16"), "a must"), (dict(out_dtype="f64"), "result"),
    (dict(out_dtype="i8"), "result"), (dict(a_dtype="bf16", out_dtype="i32"), "result"),
    (dict(depth=131072), "131071"), (dict(tokens=(1 << 31) - 65535), "tokens"), (dict(channels=(1 << 31) - 1), "channels"),
    (dict(out_row_stride=15), "overlap"), (dict(a_row_stride=1 << 45), "large"), (dict(b_row_stride=1 << 45), "large"),
    (dict(tokens=1 << 30, channels=1 << 17), "large"),
])
def test_int8_plans_that_are_refused(kw, word):
    assert word in refused(m.int8_matmul_plan, **{**dict(tokens=8, channels=16, depth=32), **kw})


def test_int8_calls_that_are_refused():
    call = m.lib().dcf_int8_matmul_async
    p = m.int8_matmul_plan(8, 16, 32)
    ok = dict(a=A, a_scale=B, b=C, b_scale=D, bias=None, out=E, ws=F, n=p.workspace, st=F + (1 << 19))

    def rc(plan=p, **kw):
        v = {**ok, **kw}
        return call(plan.ref, v["a"], v["a_scale"], v["b"], v["b_scale"], v["bias"], v["out"], v["ws"], v["n"], v["st"], None)

    for name in ("a", "a_scale", "b", "b_scale", "out", "st"):
        assert rc(**{name: None}) == -1 and "null" in last(), name
    for kw in (dict(out=A), dict(out=A + 255), dict(out=C + 511), dict(out=B + 28), dict(out=D), dict(bias=E + 255),
               dict(st=A + 8), dict(st=E)):
        assert rc(**kw) == -1 and "overlap" in last(), kw
    sums = m.int8_matmul_plan(8, 16, 32, out_dtype="i32")
    for kw in (dict(), dict(a_scale=None), dict(b_scale=None), dict(a_scale=None, b_scale=None, bias=D)):
        assert rc(sums, **kw) == -1 and "sums" in last(), kw
    tokens = m.int8_matmul_plan(8, 16, 32, a_dtype="bf16")
    assert tokens.workspace % 256 == 0
    assert rc(tokens, n=tokens.workspace) == -1 and "no scales yet" in last()
    if tokens.workspace:
        assert rc(tokens, a_scale=None, n=tokens.workspace - 1) == -1 and "workspace" in last()
        assert rc(tokens, a_scale=None, ws=None, n=tokens.workspace) == -1 and "null" in last()
    for kw in (dict(tokens=0), dict(channels=0)):
        assert rc(m.int8_matmul_plan(**{**dict(tokens=8, channels=16, depth=32), **kw}), a=None, out=None, st=None) == 0
    assert call(None, A, B, C, D, None, E, F, 0, F, None) == -1
    assert m.lib().dcf_int8_matmul_workspace(p.ref, None) == -1


@pytest.mark.parametrize("kw,word", [
    (dict(dtype="f32"), "gradient"), (dict(dtype="i8"), "gradient"), (dict(out_dtype="f64"), "result"), (dict(out_dtype="i32"), "result"),
    (dict(out_dtype="bf16", accumulate=True), "accumulates"), (dict(tokens=(1 << 31) - 65535), "at most"),
    (dict(channels=(1 << 31) - 65535), "at most"), (dict(depth=(1 << 31) - 65535), "at most"),
    (dict(out_row_stride=31), "overlap"), (dict(grad_row_stride=1 << 45), "large"), (dict(q_row_stride=1 << 45), "large"),
    (dict(channels=1 << 30, depth=1 << 17), "large"),
])
def test_checkpoint_plans_that_are_refused(kw, word):
    base = dict(dtype="bf16", tokens=8, channels=16, depth=32)
    assert word in refused(m.checkpoint_grad_plan, **{**base, **kw})


def test_checkpoint_calls_that_are_refused():
    call = m.lib().dcf_checkpoint_grad_async
    p = m.checkpoint_grad_plan("bf16", 300, 16, 32)
    ok = dict(g=A, q=B, s=C, out=D, ws=E, n=p.workspace, st=F)

    def rc(plan=p, **kw):
        v = {**ok, **kw}
        return call(plan.ref, v["g"], v["q"], v["s"], v["out"], v["ws"], v["n"], v["st"], None)

    for name in ("g", "q", "s", "out", "st"):
        assert rc(**{name: None}) == -1 and "null" in last(), name
    for kw in (dict(out=A + 9599), dict(out=B), dict(out=C + 380), dict(st=D + 2040), dict(st=A)):
        assert rc(**kw) == -1 and "overlap" in last(), kw
    large = m.checkpoint_grad_plan("bf16", 8192, 128, 128)
    if large.workspace:
        assert large.workspace % 256 == 0
        assert rc(large, n=large.workspace - 1) == -1 and "workspace" in last()
        assert rc(large, ws=None, n=large.workspace) == -1 and "null" in last()
    d = m.CheckpointDesc(m.DTYPES["bf16"], m.DTYPES["f32"], 2, 0, 8, 16, 32, 0, 0, 0)
    assert call(ctypes.byref(d), A, B, C, D, E, 0, F, None) == -1 and "flag" in last()
    d.flags, d.reserved = 0, 1
    assert call(ctypes.byref(d), A, B, C, D, E, 0, F, None) == -1 and "reserved" in last()
    for kw in (dict(channels=0), dict(depth=0)):
        empty = m.checkpoint_grad_plan(**{**dict(dtype="bf16", tokens=8, channels=16, depth=32), **kw})
        assert rc(empty, g=None, out=None, st=None) == 0


class Fake:
    """What the binding looks at in a tensor."""

    def __init__(self, shape, dtype, strides=None, room=None):
        self.shape, self.dtype = tuple(shape), dtype
        self.strides = strides or tuple(int(np.prod(shape[i + 1:])) for i in range(len(shape)))
        self.room = room if room is not None else int(np.prod(shape))

    def stride(self):
        return self.strides

    def is_contiguous(self):
        return self.strides == tuple(int(np.prod(self.shape[i + 1:])) for i in range(len(self.shape)))

    def numel(self):
        return int(np.prod(self.shape))

    def element_size(self):
        return self.dtype.itemsize

    def storage_offset(self):
        return 0

    def untyped_storage(self):
        fake = self

        class Storage:
            def nbytes(self):
                return fake.room * fake.dtype.itemsize
        return Storage()

    def data_ptr(self):
        return A

    def get_device(self):
        return 0


def test_binding_refuses_tensors_that_do_not_lie_as_the_call_reads_them():
    import torch
    plan = m.quantize_plan("bf16", 300, 20, along="columns")
    x, q, s = Fake((300, 20), torch.bfloat16), Fake((300, 20), torch.int8), Fake((3, 20), torch.float32)
    for args in ((Fake((300, 20), torch.float16), q, s), (x, Fake((300, 20), torch.uint8), s),
                 (x, q, Fake((3, 20), torch.float64)), (Fake((300, 20), torch.bfloat16, (1, 300)), q, s),
                 (Fake((299, 20), torch.bfloat16), q, s), (x, Fake((300, 20), torch.int8, (24, 1)), s), (x, q, Fake((2, 20), torch.float32)),
                 (x, q, Fake((3, 20), torch.float32, (40, 2), 120))):
        with pytest.raises(ValueError):
            m.quantize_async(plan, *args, stream=0)
        with pytest.raises(ValueError):
            m.dequantize_async(plan, args[1], args[2], args[0], stream=0)
    mm = m.int8_matmul_plan(8, 16, 32)
    st, work = Fake((2,), torch.int64), Fake((0,), torch.uint8)
    good = dict(a=Fake((8, 32), torch.int8), b=Fake((16, 32), torch.int8), out=Fake((8, 16), torch.bfloat16))
    for kw in (dict(a=Fake((8, 32), torch.bfloat16)), dict(b=Fake((16, 32), torch.int8, (1, 16))), dict(out=Fake((8, 16), torch.float16)),
               dict(a_scale=Fake((7,), torch.float32)), dict(b_scale=Fake((16,), torch.float16)), dict(bias=Fake((16,), torch.float32, (2,), 32))):
        v = {**good, **kw}
        with pytest.raises(ValueError):
            m.int8_matmul_async(mm, v.pop("a"), v.pop("b"), v.pop("out"), work, st, stream=0, **v)
    p = m.checkpoint_grad_plan("f16", 300, 16, 20)
    g, out = Fake((300, 16), torch.float16), Fake((16, 20), torch.float32)
    for args in ((Fake((300, 16), torch.bfloat16), q, s, out), (g, Fake((300, 20), torch.int8, (1, 300)), s, out),
                 (g, q, Fake((300, 20), torch.float16), out), (g, q, s, Fake((16, 20), torch.bfloat16)), (g, q, s, Fake((16, 20), torch.float32, (1, 16)))):
        with pytest.raises(ValueError):
            m.checkpoint_grad_async(p, *args, work, st, stream=0)


def test_host_arrays_that_are_refused():
    p = m.quantize_plan("f32", 4, 8)
    with pytest.raises(ValueError):
        m.quantize(p, np.zeros((4, 7), np.float32))
    with pytest.raises(ValueError):
        m.dequantize(p, np.zeros((4, 8), np.uint8), np.zeros(4, np.float32))
    with pytest.raises(ValueError):
        m.dequantize(p, np.zeros((4, 8), np.int8), np.zeros(3, np.float32))
    mm = m.int8_matmul_plan(2, 3, 4)
    with pytest.raises(ValueError):
        m.int8_matmul(mm, np.zeros((2, 4), np.int8), np.zeros((3, 4), np.int16))
    with pytest.raises(ValueError):
        m.int8_matmul(mm, np.zeros((2, 4), np.int8), np.zeros((3, 4), np.int8), b_scale=np.zeros(2, np.float32))
    g = m.checkpoint_grad_plan("bf16", 2, 3, 4, accumulate=True)
    with pytest.raises(ValueError):
        m.checkpoint_grad(g, np.zeros((2, 3), np.uint16), np.zeros((2, 4), np.int8), np.zeros((1, 4), np.float32))
    # strides describe device tensors
    strided = m.quantize_plan("f32", 4, 8, row_stride=9)
    assert "dense" in refused(m.quantize, strided, np.zeros((4, 8), np.float32))


@pytest.mark.skipif(have_gpu(), reason="checks the no-GPU failure path")
def test_no_cpu_fallback():
    p = m.quantize_plan("f32", 4, 8)
    for call in (lambda: m.quantize(p, np.ones((4, 8), np.float32)),
                 lambda: m.dequantize(p, np.ones((4, 8), np.int8), np.ones(4, np.float32)),
                 lambda: m.int8_matmul(m.int8_matmul_plan(4, 4, 8, out_dtype="i32"), np.ones((4, 8), np.int8), np.ones((4, 8), np.int8)),
                 lambda: m.checkpoint_grad(m.checkpoint_grad_plan("f16", 4, 4, 8), np.ones((4, 4), np.float16),
                                           np.ones((4, 8), np.int8), np.ones((1, 8), np.float32))):
        with pytest.raises(m.DcfError) as e:
            call()
        assert e.value.code == -2


# ------------------------------------------------------------- the oracle


def test_oracle_rounds_half_to_even_and_marks_what_is_not_finite():
    x = np.array([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 63.5], [0, 0, 0, 0, 0, 0, -0.0], [1, np.nan, 2, 3, 4, 5, 6],
                  [np.inf, 1, 2, 3, 4, 5, 6], [2.0 ** -120] * 7])
    q, s = io.quantize(x, "rows")
    assert q.tolist() == [[127, 0, 2, 2, 0, -2, 64], [0] * 7, [0] * 7, [0] * 7, [0] * 7]
    assert s[0] == 1 and s[1] == 0 and np.isnan(s[2:4]).all() and s[4] == 0
    q, s = io.quantize(np.ones((300, 3)), "columns")
    assert q.shape == (300, 3) and (q == 127).all() and s.shape == (3, 3) and (s == np.float32(1) / np.float32(127)).all()


def test_oracle_gradient_is_that_of_the_layer():
    """loss = sum(g * (x w^T)) has the oracle's gradient in w, by central differences of a bilinear form (exact up to rounding)."""
    rng = np.random.default_rng(0)
    g, q, s = rng.standard_normal((150, 4)), rng.integers(-127, 128, (150, 5)).astype(np.int8), rng.random((2, 5)).astype(np.float32)
    x = q * io.spread(s, 150, "columns").astype(np.float64)
    w = rng.standard_normal((4, 5))
    want, _ = io.grad(g, q, s)
    for c in range(4):
        for k in range(5):
            step = np.zeros_like(w)
            step[c, k] = 0.5
            rise = np.sum(g * (x @ (w + step).T)) - np.sum(g * (x @ (w - step).T))
            assert abs(rise - want[c, k]) <= 1e-9 * np.abs(g).sum() * np.abs(x).max()
