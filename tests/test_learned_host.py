"""Operators on learned tensors, on the CPU: descriptors that are refused,
workspace sizes, and that a call without a GPU says so."""
import ctypes
import math

import numpy as np
import pytest

import learned_oracle as lo
import mlirpass_b200 as m
from conftest import have_gpu


def refused(make, *args, **kw):
    with pytest.raises(m.DcfError) as e:
        make(*args, **kw)
    assert e.value.code == -1, e.value
    return str(e.value)


def bias(**kw):
    base = dict(dtype="bf16", heads=4, queries=8, keys=16)
    base.update(kw)
    return m.position_bias_plan(base.pop("dtype"), base.pop("heads"), base.pop("queries"), base.pop("keys"), **base)


@pytest.mark.parametrize("kw,word", [
    (dict(dtype="i32"), "dtype"), (dict(dtype="f8E4M3"), "dtype"),
    (dict(num_buckets=0), "num_buckets"), (dict(num_buckets=1), "num_buckets"), (dict(num_buckets=257), "num_buckets"),
    (dict(max_distance=8), "max_distance"),                       # 32 buckets, 16 a side: 8 are exact
    (dict(max_distance=16, bidirectional=False), "max_distance"),
    (dict(heads=65536), "heads"),
    (dict(first_query=(1 << 40) + 1), "first_query"), (dict(first_query=-(1 << 40) - 1), "first_query"),
    (dict(row_stride=-1), "stride"), (dict(head_stride=-128), "stride"), (dict(batch_stride=-1), "stride"),
    (dict(row_stride=1 << 45), "large"), (dict(head_stride=1 << 45), "large"),
])
def test_bias_plans_that_are_refused(kw, word):
    assert word in refused(bias, **kw)


def test_bias_calls_that_are_refused():
    call = m.lib().dcf_position_bias_async

    def rc(plan, table=256, out=256):
        return call(plan.ref, table, None, out, None)

    for kw in (dict(dtype="f32", table_dtype="bf16"), dict(dtype="f64", table_dtype="f32"),
               dict(accumulate=True),                       # the gradient's flag
               dict(row_stride=15), dict(head_stride=127),  # rows that overlap
               dict(row_stride=16, head_stride=64)):
        plan = bias(**kw)
        assert rc(plan) == -1, kw
    # heads inside rows is a layout, not an overlap: refused only for its pointers
    assert rc(bias(row_stride=64, head_stride=16), table=None) == -1
    assert b"null" in m.lib().dcf_last_error()
    # nothing to write: no pointer is looked at
    for kw in (dict(heads=0), dict(queries=0), dict(keys=0)):
        assert rc(bias(**kw), None, None) == 0
    assert call(None, 256, None, 256, None) == -1


def test_bias_grad_workspace_and_its_checks():
    plan = bias(heads=16, queries=1000, keys=1000)
    assert plan.workspace > 0 and plan.workspace % 256 == 0
    assert bias(queries=1, keys=4).workspace == 0
    call = m.lib().dcf_position_bias_grad_async
    assert call(plan.ref, 256, None, 256, 256, plan.workspace - 1, None) == -1
    assert b"workspace" in m.lib().dcf_last_error()
    assert call(plan.ref, 256, None, 256, None, plan.workspace, None) == -1
    assert call(plan.ref, None, None, 256, 256, plan.workspace, None) == -1
    assert call(plan.ref, 256, None, None, 256, plan.workspace, None) == -1
    assert m.lib().dcf_position_bias_grad_workspace(plan.ref, None) == -1
    assert m.lib().dcf_position_bias_grad_workspace(None, ctypes.byref(ctypes.c_size_t())) == -1


@pytest.mark.parametrize("kw,word", [
    (dict(dtype="f64"), "dtype"), (dict(dtype="i8"), "dtype"), (dict(out_dtype="f64"), "dtype"),
    (dict(rows=65537), "65536"), (dict(cols=65537), "65536"), (dict(batch=65536), "65535"),
    (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"), (dict(eps=math.inf), "eps"),
    (dict(row_stride=-1), "stride"), (dict(out_row_stride=-1), "stride"), (dict(batch_stride=-1), "stride"),
    (dict(out_row_stride=15), "overlap"), (dict(batch=2, out_batch_stride=127), "overlap"),
    (dict(row_stride=1 << 45), "large"),
    (dict(coef=(math.nan, 0, 0)), "coefficient"), (dict(coef=(1e5, 0, 0)), "coefficient"),
    (dict(coef=(3.0, 0, 0)), "past 64"),                    # 3^5 = 243
    (dict(coef=(3.4445, 4.7750, 2.0315)), "past 64"),
    (dict(coef=(0, 0, 0)), "nothing"), (dict(coef=(1e-31, 0, 0)), "nothing"), (dict(coef=(1e-8, 0, 0), steps=5), "nothing"),
    (dict(rows=65536, cols=65536, batch=65535), "tiles"),
])
def test_orth_plans_that_are_refused(kw, word):
    base = dict(dtype="bf16", rows=8, cols=16)
    base.update(kw)
    assert word in refused(m.orthogonalize_plan, base.pop("dtype"), base.pop("rows"), base.pop("cols"), **base)


def test_orth_bound_follows_the_interior_of_the_interval():
    # 4 s - 4 s^3 is 0 at 0 and at 1; its largest value lies between (1.54), and grows from there
    m.orthogonalize_plan("f32", 8, 8, steps=2, coef=(4, -4, 0))
    assert "past 64" in refused(m.orthogonalize_plan, "f32", 8, 8, steps=4, coef=(4, -4, 0))
    # the quintic used by default settles for any number of steps
    m.orthogonalize_plan("f32", 8, 8, steps=16)
    # a step of its own for each
    m.orthogonalize_plan("f32", 8, 8, steps=3, coef=[(4, -4, 0), (1, 0, 0), (0.25, 0, 0)])


def test_orth_calls_that_are_refused():
    plan = m.orthogonalize_plan("f32", 400, 500)
    assert plan.workspace > 0
    call = m.lib().dcf_orthogonalize_async
    assert call(plan.ref, 256, 256, 256, plan.workspace - 1, 256, None) == -1
    for ptrs in ((None, 256, 256, 256), (256, None, 256, 256), (256, 256, None, 256), (256, 256, 256, None)):
        i, o, w, s = ptrs
        assert call(plan.ref, i, o, w, plan.workspace, s, None) == -1
    # a matrix of few rows stays on the chip: no workspace, unless it is too long
    assert m.orthogonalize_plan("f32", 128, 2048).workspace == m.orthogonalize_plan("f32", 2048, 1).workspace == 0
    assert m.orthogonalize_plan("f32", 129, 129).workspace > 0 and m.orthogonalize_plan("f32", 8, 2049).workspace > 0
    bad = m.OrthDesc.from_buffer_copy(plan.desc)
    bad.reserved = 1
    assert call(ctypes.byref(bad), 256, 256, 256, plan.workspace, 256, None) == -1
    # in place only where a matrix is written where it was read
    for kw in (dict(out_dtype="bf16"), dict(out_row_stride=501), dict(batch=2, out_batch_stride=400 * 500 + 1)):
        other = m.orthogonalize_plan("f32", 400, 500, **kw)
        assert call(other.ref, 256, 256, 512, other.workspace, 1024, None) == -1
        assert b"in place" in m.lib().dcf_last_error()
    bad = m.OrthDesc.from_buffer_copy(plan.desc)
    bad.steps = 17
    assert call(ctypes.byref(bad), 256, 256, 256, plan.workspace, 256, None) == -1
    for kw in (dict(rows=0, cols=5), dict(rows=5, cols=0), dict(rows=5, cols=5, batch=0)):
        empty = m.orthogonalize_plan("f32", **kw)
        assert empty.workspace == 0
        assert call(empty.ref, None, None, None, 0, None, None) == 0


@pytest.mark.parametrize("args", [dict(steps=17), dict(steps=-1), dict(coef=(1, 2)), dict(coef=[(1, 2, 3)] * 4),
                                  dict(rows=-1)])
def test_orth_python_arguments(args):
    base = dict(rows=8, cols=8)
    base.update(args)
    with pytest.raises(ValueError):
        m.orthogonalize_plan("f32", **base)


def test_host_forms_take_dense_tensors_of_the_right_size():
    plan = bias(dtype="f32")
    with pytest.raises(ValueError):
        m.position_bias(plan, np.zeros((32, 3), np.float32))
    with pytest.raises(ValueError):
        m.position_bias(plan, np.zeros((32, 4), np.float32), positions=[1, 2])
    with pytest.raises(ValueError):
        m.position_bias_grad(plan, np.zeros(7, np.float32))
    with pytest.raises(ValueError):
        m.position_bias_grad(bias(dtype="f32", accumulate=True), np.zeros((1, 4, 8, 16), np.float32))
    with pytest.raises(ValueError):
        m.orthogonalize(m.orthogonalize_plan("f32", 4, 4), np.zeros(15, np.float32))
    assert "dense" in refused(m.position_bias, bias(dtype="f32", row_stride=32), np.zeros((32, 4), np.float32))
    assert "dense" in refused(m.orthogonalize, m.orthogonalize_plan("f32", 4, 4, row_stride=8),
                              np.zeros((4, 4), np.float32))


@pytest.mark.skipif(have_gpu(), reason="checks the no-GPU failure path")
def test_no_cpu_fallback():
    for call in (lambda: m.position_bias(bias(dtype="f32"), np.zeros((32, 4), np.float32)),
                 lambda: m.position_bias_grad(bias(dtype="f32"), np.zeros((1, 4, 8, 16), np.float32)),
                 lambda: m.orthogonalize(m.orthogonalize_plan("f32", 4, 4), np.zeros((4, 4), np.float32))):
        with pytest.raises(m.DcfError) as e:
            call()
        assert e.value.code == -2


def test_oracle_buckets_at_the_borders():
    # 32 buckets both ways, distance 128: exact to 7, then 8 * 2^(k/2) rounded up
    b = [lo.bucket(-n, 32, 128, True) for n in range(200)]
    starts = [b.index(v) for v in range(16)]
    assert starts == lo.starts(32, 128, True) == [0, 1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 23, 32, 46, 64, 91]
    assert b[127] == b[128] == b[199] == 15
    assert lo.bucket(1, 32, 128, True) == 17 and lo.bucket(5, 32, 128, False) == 0
    # plain floating point agrees away from the borders
    for n in (9, 13, 25, 50, 100):
        assert b[n] == 8 + int(math.log(n / 8) / math.log(16) * 8)


@pytest.mark.parametrize("num_buckets,max_distance,both", [(1, 1, False), (2, 1, True), (3, 2, False), (7, 5, True),
                                                           (33, 200, True), (64, 33, True), (32, 512, False)])
def test_oracle_starts_and_buckets_agree(num_buckets, max_distance, both):
    reach = max_distance + 30
    ids = lo.buckets([reach], 2 * reach + 1, num_buckets, max_distance, both)[0]
    assert list(ids) == [lo.bucket(d, num_buckets, max_distance, both) for d in range(-reach, reach + 1)]


@pytest.mark.parametrize("c", [1e-17, -1e-17, 5.5e-17, 1e-300, -1e-300, 5e-324])
def test_orth_bound_with_a_leftover_in_the_last_coefficient(c):
    """What cancellation leaves of a zero changes no bound: the largest value inside the interval is found."""
    assert "past 64" in refused(m.orthogonalize_plan, "f32", 8, 8, steps=4, coef=(4, -4, c))
    m.orthogonalize_plan("f32", 8, 8, steps=2, coef=(4, -4, c))
    m.orthogonalize_plan("f32", 8, 8, steps=2, coef=(3, -3, c))
    m.orthogonalize_plan("f32", 8, 8, steps=5, coef=(1.5, -0.5, c))
    m.orthogonalize_plan("f32", 8, 8, steps=2, coef=(c, 1, 1))
    m.orthogonalize_plan("f32", 8, 8, steps=2, coef=(1, c, 1))


def test_orth_bounds_against_a_fine_grid():
    """Accepted or refused as the polynomial's values on a grid say, for coefficients of any sign."""
    rng = np.random.default_rng(7)
    for _ in range(400):
        coef = [rng.choice([0.0, 1e-17, 1.0]) * rng.uniform(-8, 8) for _ in range(3)]
        s, least = 1.0, math.inf
        for _ in range(3):
            t = np.linspace(0, s, 4001) ** 2
            f = np.abs(coef[0] + t * (coef[1] + t * coef[2]))
            least, s = min(least, f.max(), (np.sqrt(t) * f).max()), (np.sqrt(t) * f).max()
            if s > 64:
                break
        if abs(s - 64) < 1 or 1e-40 < least < 1e-20:      # too near a border for a grid
            continue
        if s > 64 or least < 1e-30:
            refused(m.orthogonalize_plan, "f32", 8, 8, steps=3, coef=coef)
        else:
            m.orthogonalize_plan("f32", 8, 8, steps=3, coef=coef)


def device_call(call, *args, **kw):
    """A device form on CPU tensors: what the binding lets pass is refused by the library (host memory, or no GPU)."""
    with pytest.raises((ValueError, m.DcfError)) as e:
        call(*args, stream=0, **kw)
    return "binding" if isinstance(e.value, ValueError) else "library"


def test_tensors_without_strides_in_the_plan_are_contiguous():
    import torch
    plan = m.position_bias_plan("f32", 4, 10, 16)
    table, out = torch.zeros(32, 4), torch.zeros(4, 10, 16)
    grad, work = torch.zeros(1, 4, 10, 16), torch.zeros(m.position_bias_grad_workspace(plan) + 8, dtype=torch.uint8)
    ids = torch.zeros(10, 2, dtype=torch.int32)
    assert device_call(m.position_bias_async, plan, table, out) == "library"
    assert device_call(m.position_bias_async, plan, torch.zeros(128), out) == "library"
    assert device_call(m.position_bias_async, plan, torch.zeros(40, 4)[2:], out) == "library"
    for t in (torch.zeros(4, 32).T, torch.zeros(32, 8)[:, :4], torch.zeros(64, 4)[::2], torch.zeros(1, 4).expand(32, 4),
              torch.zeros(31, 4), torch.zeros(40, 4)[:31]):
        assert device_call(m.position_bias_async, plan, t, out) == "binding"
        assert device_call(m.position_bias_grad_async, plan, grad, t, work) == "binding"
    assert device_call(m.position_bias_async, plan, table, out, positions=ids[:, 0].contiguous()) == "library"
    for p in (ids[:, 0], ids[::2, :1], ids[:9, 0].contiguous(), torch.zeros(1, dtype=torch.int32).expand(10)):
        assert device_call(m.position_bias_async, plan, table, out, positions=p) == "binding"
        assert device_call(m.position_bias_grad_async, plan, grad, table, work, positions=p) == "binding"
    orth, x = m.orthogonalize_plan("f32", 4, 4), torch.zeros(4, 4)
    none = torch.zeros(0, dtype=torch.uint8)
    status = torch.zeros(2, 2, dtype=torch.int64)
    assert device_call(m.orthogonalize_async, orth, x, x, none, status[1]) == "library"
    assert device_call(m.orthogonalize_async, orth, x, x, none, status[:, 0]) == "binding"


def test_tensors_lie_as_the_plan_says():
    import torch
    work, status = torch.zeros(1 << 20, dtype=torch.uint8), torch.zeros(2, dtype=torch.int64)

    def orth(t, batch=2, rows=6, cols=8, **kw):
        plan = m.orthogonalize_plan("f32", rows, cols, batch=batch, **kw)
        keep = torch.zeros(4096)
        got = {device_call(m.orthogonalize_async, plan, t, keep, work, status)}
        plan = m.orthogonalize_plan("f32", rows, cols, batch=batch, **{"out_" + k: v for k, v in kw.items()})
        return (got | {device_call(m.orthogonalize_async, plan, keep, t, work, status)}).pop()

    square = torch.zeros(8, 8)
    assert orth(torch.zeros(2, 6, 8)) == orth(torch.zeros(96)) == orth(torch.zeros(200)[7:]) == "library"
    assert orth(torch.zeros(12, 8)) == orth(torch.zeros(1, 2, 6, 8)) == orth(torch.zeros(6, 8), batch=1) == "library"
    wide = torch.zeros(2, 6, 11)
    assert orth(wide[..., :8], row_stride=11) == orth(wide[..., 3:], row_stride=11) == "library"
    assert orth(wide.view(12, 11)[:, 2:10], row_stride=11) == orth(wide[0, :, :8], batch=1, row_stride=11) == "library"
    assert orth(wide[:, :, 1:], row_stride=11) == "library"               # wider than the plan's rows
    assert orth(torch.zeros(6, 2, 8).transpose(0, 1), batch_stride=200) == "binding"
    for t in (torch.zeros(2, 8, 6).transpose(1, 2), torch.zeros(2, 6, 11)[..., :8], torch.zeros(2, 6, 16)[..., ::2],
              torch.zeros(4, 6, 8)[::2], torch.zeros(2, 12, 8)[:, ::2], torch.zeros(1, 6, 8).expand(2, 6, 8)):
        assert orth(t) == "binding", t.stride()
    assert orth(square.T, batch=1, rows=8) == "binding"
    assert orth(torch.zeros(200)[:96].view(2, 6, 8), row_stride=11) == "binding"    # dense, with room behind

    def bias(t, **kw):
        plan = m.position_bias_plan("f32", 3, 5, 7, **kw)
        got = {device_call(m.position_bias_async, plan, torch.zeros(32, 3), t)}
        grad = device_call(m.position_bias_grad_async, plan, t, torch.zeros(32, 3), work)
        assert got == {grad}
        return grad

    assert bias(torch.zeros(3, 5, 7)) == bias(torch.zeros(3, 5, 9)[..., :7], row_stride=9) == "library"
    inside = dict(row_stride=27, head_stride=9)                                     # heads inside rows
    buffer = torch.zeros(5, 3, 9)
    assert bias(buffer[..., :7].transpose(0, 1), **inside) == bias(buffer[..., :7], **inside) == "library"
    assert bias(buffer, **inside) == bias(buffer.view(-1), **inside) == "library"
    for t in (torch.zeros(5, 3, 7).transpose(0, 1), torch.zeros(3, 7, 5).transpose(1, 2), torch.zeros(3, 5, 9)[..., :7],
              torch.zeros(3, 5, 7)[:, :, :1].expand(3, 5, 7)):
        assert bias(t) == "binding"
    assert bias(torch.zeros(3, 5, 9)[..., :7], **inside) == "binding"


def test_tensors_have_the_plans_types():
    import torch
    work, status = torch.zeros(1 << 20, dtype=torch.uint8), torch.zeros(2, dtype=torch.int64)
    types = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "f64": torch.float64}
    others = [torch.float16, torch.bfloat16, torch.float32, torch.float64, torch.int16, torch.int32, torch.int64,
              torch.complex64]
    for name, own in types.items():
        wide = torch.float64 if name == "f64" else torch.float32
        plan = m.position_bias_plan(name, 4, 10, 16)
        orth = m.orthogonalize_plan(name, 10, 16) if name != "f64" else None
        back = m.orthogonalize_plan("f32", 10, 16, out_dtype=name) if name != "f64" else None
        for t in others:
            table, bias = torch.zeros(32, 4, dtype=t), torch.zeros(4, 10, 16, dtype=t)
            x, f = torch.zeros(10, 16, dtype=t), torch.zeros(10, 16)
            want = "library" if t == own else "binding"
            assert device_call(m.position_bias_async, plan, table, torch.zeros(4, 10, 16, dtype=own)) == want
            assert device_call(m.position_bias_async, plan, torch.zeros(32, 4, dtype=own), bias) == want
            assert device_call(m.position_bias_grad_async, plan, bias, torch.zeros(32, 4, dtype=wide), work) == want
            assert device_call(m.position_bias_grad_async, plan, torch.zeros(4, 10, 16, dtype=own), table, work) == \
                ("library" if t == wide else "binding")
            if orth:
                assert device_call(m.orthogonalize_async, orth, x, torch.zeros(10, 16, dtype=own), work, status) == want
                assert device_call(m.orthogonalize_async, back, f, x, work, status) == want
    plan = m.position_bias_plan("bf16", 4, 10, 16, table_dtype="f32")
    for t in others:
        assert device_call(m.position_bias_async, plan, torch.zeros(32, 4, dtype=t), torch.zeros(4, 10, 16).bfloat16()) == \
            ("library" if t == torch.float32 else "binding")
    for t in (torch.int32, torch.uint32, torch.int64, torch.float32):
        assert device_call(m.position_bias_async, plan, torch.zeros(32, 4), torch.zeros(4, 10, 16).bfloat16(),
                           positions=torch.zeros(10, dtype=t)) == ("library" if t == torch.int32 else "binding")


def test_host_positions_keep_their_value():
    plan = m.position_bias_plan("f32", 1, 3, 4)
    for p in ([0, 1, 1 << 31], np.array([0, 1, (1 << 32) + 2]), np.array([0, 1, 1 << 63], np.uint64), [0, 1, 2.5],
              [0, 1, math.nan], np.array([0.0, 1.0, 3e9]), [0, 1, -(1 << 31) - 1], ["0", "1", "2"], [0, 1]):
        with pytest.raises(ValueError):
            m.position_bias(plan, np.zeros((32, 1), np.float32), positions=p)
        with pytest.raises(ValueError):
            m.position_bias_grad(plan, np.zeros((1, 1, 3, 4), np.float32), positions=p)
    for p in ([0, -5, (1 << 31) - 1], np.array([0, -(1 << 31), 7]), np.array([0.0, 1.0, 2.0]), np.arange(6, dtype=np.int16)[::2],
              np.array([1, 2, 3], np.uint64), [True, False, True]):
        assert m._host_positions(p, 3).tolist() == [int(v) for v in p]
    assert len(m._host_positions([], 0)) == 0


def test_orth_workspace_without_steps():
    """No workspace is for matrices that stay on the chip; without steps nothing does."""
    call = m.lib().dcf_orthogonalize_async
    for rows, cols in ((96, 96), (128, 2048), (1, 1)):
        assert m.orthogonalize_plan("f32", rows, cols, steps=1).workspace == 0
        plan = m.orthogonalize_plan("f32", rows, cols, steps=0)
        assert plan.workspace > 0
        assert call(plan.ref, 256, 256, None, 0, 256, None) == -1 and b"null" in m.lib().dcf_last_error()
        assert call(plan.ref, 256, 256, 256, plan.workspace - 1, 256, None) == -1
        assert b"workspace" in m.lib().dcf_last_error()


@pytest.mark.parametrize("batch,queries,keys,first", [(6, 700, 256, 0), (8, 40, 512, -600), (2, 20, 512, 100), (1, 3, 9, 0)])
def test_whole_values_show_what_is_missing(batch, queries, keys, first):
    """One element, one step of 32 vectors, one row or one far range left out changes a sum."""
    g = lo.whole_values((batch, 1, queries, keys), 1)
    ids = lo.buckets(lo.positions(queries, first), keys, 32, 128, True)
    want, mag = lo.bias_grad(g, ids, 32)
    assert mag.max() < 2 ** 24 and np.array_equal(want, mag)
    rng = np.random.default_rng(2)
    for _ in range(5):
        b, q, k = rng.integers(batch), rng.integers(queries), rng.integers(keys)
        for cut in (np.s_[b, :, q, k], np.s_[b, :, q, k:k + 256], np.s_[b, :, q], np.s_[:, :, ids == ids[q, k]]):
            less = g.copy()
            less[cut] = 0
            assert not np.array_equal(lo.bias_grad(less, ids, 32)[0], want)
        more = g.copy()
        more[b, 0, q, k] *= 2
        assert not np.array_equal(lo.bias_grad(more, ids, 32)[0], want)
