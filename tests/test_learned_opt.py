"""learned-constant-fold in the pass driver: the dcf.* operators on learned
tensors fold where their operand is a constant, and stay as they are where
their types or properties are not the operator's."""
import numpy as np
import pytest

import learned_oracle as lo
from mlir_text import parse_funcs
from mlirpass_b200 import opt

PIPELINE = "builtin.module(func.func(learned-constant-fold,canonicalize))"


def hexed(a: np.ndarray) -> str:
    return f'dense<"0x{a.tobytes().hex().upper()}">'


def module(in_ty: str, literal: str, op: str, props: str, out_ty: str, name: str = "f") -> str:
    return ('"builtin.module"() ({\n'
            f'  "func.func"() <{{function_type = () -> {out_ty}, sym_name = "{name}"}}> ({{\n'
            f'    %0 = "arith.constant"() <{{value = {literal} : {in_ty}}}> : () -> {in_ty}\n'
            f'    %1 = "{op}"(%0){props} : ({in_ty}) -> {out_ty}\n'
            f'    "func.return"(%1) : ({out_ty}) -> ()\n'
            '  }) : () -> ()\n}) : () -> ()\n')


def result(text: str, n_gpus: int = 1, name: str = "f"):
    out, stats = opt.run(text, PIPELINE, n_gpus=n_gpus)
    f = parse_funcs(out)[name]
    return f.defs[f.ret.operands[0]], stats


TABLE = np.arange(32 * 3, dtype=np.float32).reshape(32, 3) / 8


@pytest.mark.parametrize("op,in_ty,props,out_ty", [
    ("dcf.position_bias", "tensor<32x3xf32>", "", "tensor<4x5x6xf32>"),                       # heads differ
    ("dcf.position_bias", "tensor<32x3xf32>", "", "tensor<3x5x6xi32>"),
    ("dcf.position_bias", "tensor<32x3xf32>", " <{max_distance = 8 : i64}>", "tensor<3x5x6xf32>"),
    ("dcf.position_bias", "tensor<32x3xf32>", " <{max_distance = -1 : i64}>", "tensor<3x5x6xf32>"),
    ("dcf.position_bias", "tensor<32x3xf32>", " <{causal = 3 : i64}>", "tensor<3x5x6xf32>"),
    ("dcf.position_bias", "tensor<96xf32>", "", "tensor<3x5x6xf32>"),
    ("dcf.position_bias", "tensor<32x3xf32>", "", "tensor<3x200000x200000xf32>"),             # 480 GB
    ("dcf.position_bias", "tensor<32x3xf32>", "", "tensor<3x0x6xf32>"),
    ("dcf.position_bias", "tensor<32x3xf32>", "", "tensor<3x5x?xf32>"),
    ("dcf.position_bias_grad", "tensor<3x4x8xf32>", "", "tensor<32x3xbf16>"),
    ("dcf.position_bias_grad", "tensor<32x3xf32>", "", "tensor<32x3xf32>"),
    ("dcf.orthogonalize", "tensor<32x3xf32>", "", "tensor<3x32xf32>"),
    ("dcf.orthogonalize", "tensor<32x3xf32>", "", "tensor<32x3xf64>"),
    ("dcf.orthogonalize", "tensor<32x3xf32>", " <{steps = 17 : i64}>", "tensor<32x3xf32>"),
    ("dcf.orthogonalize", "tensor<32x3xf32>", " <{coef = array<f64: 1.0, 2.0>}>", "tensor<32x3xf32>"),
    ("dcf.orthogonalize", "tensor<32x3xf32>", " <{coef = array<f64: 9.0, 9.0, 9.0>}>", "tensor<32x3xf32>"),
    ("dcf.orthogonalize", "tensor<32x3xf32>", " <{eps = -1.0 : f64}>", "tensor<32x3xf32>"),
    ("dcf.unknown", "tensor<32x3xf32>", "", "tensor<32x3xf32>"),
])
def test_ops_that_stay(op, in_ty, props, out_ty):
    d, stats = result(module(in_ty, hexed(TABLE), op, props, out_ty), n_gpus=0)
    assert d.name == op and stats["folds"] == 0


def test_other_passes_leave_them_alone():
    text = module("tensor<32x3xf32>", hexed(TABLE), "dcf.position_bias", "", "tensor<3x5x6xf32>")
    for pipeline in ("canonicalize", "builtin.module(func.func(tosa-layerwise-constant-fold,canonicalize))"):
        out, stats = opt.run(text, pipeline, n_gpus=0)
        assert '"dcf.position_bias"' in out and stats["folds"] == 0


def test_element_work_needs_a_gpu():
    text = module("tensor<32x3xf32>", hexed(TABLE), "dcf.position_bias", "", "tensor<3x5x6xf32>")
    with pytest.raises(Exception):
        opt.run(text, PIPELINE, n_gpus=0)


@pytest.mark.gpu
def test_bias_folds():
    props = " <{bidirectional = false, causal = true, first_query = 3 : i64, max_distance = 64 : i64}>"
    d, stats = result(module("tensor<32x3xf32>", hexed(TABLE), "dcf.position_bias", props, "tensor<3x9x12xf32>"))
    q = lo.positions(9, 3)
    want = np.where(lo.masked(q, 12), -np.inf, TABLE.T[:, lo.buckets(q, 12, 32, 64, False)]).astype(np.float32)
    assert d.name == "arith.constant" and stats["folds"] == 1
    assert np.array_equal(np.array(d.const.bits, np.uint32).reshape(3, 9, 12), want.view(np.uint32))


@pytest.mark.gpu
def test_bias_of_a_splat_table_is_a_splat_and_folds_on():
    """The bias folds, then canonicalize folds what reads it."""
    text = ('"builtin.module"() ({\n'
            '  "func.func"() <{function_type = () -> tensor<3x40x50xf32>, sym_name = "f"}> ({\n'
            '    %0 = "arith.constant"() <{value = dense<2.5> : tensor<32x3xf32>}> : () -> tensor<32x3xf32>\n'
            '    %1 = "dcf.position_bias"(%0) : (tensor<32x3xf32>) -> tensor<3x40x50xf32>\n'
            '    %2 = "arith.addf"(%1, %1) <{fastmath = #arith.fastmath<none>}> : (tensor<3x40x50xf32>, tensor<3x40x50xf32>) -> tensor<3x40x50xf32>\n'
            '    "func.return"(%2) : (tensor<3x40x50xf32>) -> ()\n'
            '  }) : () -> ()\n}) : () -> ()\n')
    d, stats = result(text)
    assert d.name == "arith.constant" and d.const.splat and stats["folds"] == 2
    assert d.const.bits[0] == np.float32(5.0).view(np.uint32)


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [0, 2])
def test_gradient_folds(batch):
    rng = np.random.default_rng(1)
    g = rng.standard_normal((max(batch, 1), 3, 20, 30)).astype(np.float32)
    in_ty = "tensor<" + (f"{batch}x" if batch else "") + "3x20x30xf32>"
    d, _ = result(module(in_ty, hexed(g), "dcf.position_bias_grad", "", "tensor<32x3xf32>"))
    want, mag = lo.bias_grad(g, lo.buckets(lo.positions(20, 0), 30, 32, 128, True), 32)
    got = np.array(d.const.bits, np.uint32).view(np.float32).reshape(32, 3)
    assert d.name == "arith.constant"
    assert (np.abs(got - want) <= lo.bias_grad_bound(mag, g.shape[0], 20, 30, 4, lo.U32)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape,props,coef,steps", [
    ((24, 40), "", (3.4445, -4.7750, 2.0315), 5),
    ((2, 150, 140), " <{steps = 2 : i64, coef = array<f64: 1.5, -0.5, 0.0>, eps = 1.0e-3 : f64}>", (1.5, -0.5, 0.0), 2)])
def test_orthogonalize_folds(shape, props, coef, steps):
    x = np.random.default_rng(2).standard_normal(shape).astype(np.float32)
    ty = "tensor<" + "x".join(map(str, shape)) + "xf32>"
    d, _ = result(module(ty, hexed(x), "dcf.orthogonalize", props, ty))
    got = np.array(d.const.bits, np.uint32).view(np.float32).reshape((-1,) + shape[-2:])
    eps = 1e-3 if "eps" in props else 1e-7
    for k, m in enumerate(x.reshape((-1,) + shape[-2:])):
        want = lo.newton_schulz(m, [coef] * steps, eps)
        tol = lo.orth_tolerance(m, [coef] * steps, eps) + lo.U32
        assert np.linalg.norm(got[k] - want) <= tol * np.linalg.norm(want)


def taken(props: str, op: str = "dcf.orthogonalize", out_ty: str = "tensor<32x3xf32>") -> bool:
    """Whether the pass takes the op for folding (which fails here for want of a GPU) or leaves it."""
    try:
        d, _ = result(module("tensor<32x3xf32>", hexed(TABLE), op, props, out_ty), n_gpus=0)
    except Exception as e:
        assert "needs a GPU" in str(e)
        return True
    assert d.name == op
    return False


def f64_bits(v: float) -> str:
    return f"0x{np.float64(v).view(np.uint64):016X}"


@pytest.mark.parametrize("eps,is_eps", [
    ("1.0e-7 : f64", True), ("1.0e-7", True), ("1.000000e-03 : f32", True), ("0.0 : f64", True), ("12.5E+1 : f64", True),
    (f64_bits(1e-7) + " : f64", True), ("0x33D6BF95 : f32", True), (f64_bits(0.0) + " : f64", True), ("1 : i64", True),
    (f64_bits(-1.0) + " : f64", False), (f64_bits(np.nan) + " : f64", False), (f64_bits(np.inf) + " : f64", False),
    ("0xBF800000 : f32", False), (f64_bits(1e-7) + " : f32", False), ("0x7FC00000 : f32", False),
    (f64_bits(1e-7), False), ("0x10 : i64", False), ("-0x1 : f64", False), ("0x : f64", False),
    ("1e-3junk : f64", False), ("1.0e-3 junk", False), ("nan", False), ("inf : f64", False), ("1.0e-7 : f16", False),
    ("1.0e-7 : tensor<f64>", False), ("0x1p-3 : f64", False), ("1.0e999 : f64", False), ("", False), ("-1.0 : f64", False),
    ('"1.0"', False), (".5 : f64", False), ("1.0e : f64", False), ("--1.0 : f64", False)])
def test_spellings_of_eps(eps, is_eps):
    assert taken(f" <{{eps = {eps}}}>") == is_eps


@pytest.mark.parametrize("coef,is_coef", [
    ("array<f64: 1.5, -0.5, 0.0>", True), ("array<f64: 1.5,-5.0e-1,0.0>", True), ("array<f64: 1, 0, 0>", True),
    (f"array<f64: {f64_bits(1.5)}, {f64_bits(-0.5)}, {f64_bits(0.0)}>", True),
    ("array<f32: 1.5, -0.5, 0.0>", False), ("array<i64: 1, 0, 0>", False), ("array<f64: 1.5 junk, -0.5, 0.0>", False),
    ("array<f64: 1.5, -0.5, 0.0> junk", False), ("array<f64: 1.5, -0.5, 0.0,>", False),
    ("array<f64: , -0.5, 0.0>", False), ("array<f64>", False), ("dense<[1.5, -0.5, 0.0]> : tensor<3xf64>", False),
    (f"array<f64: {f64_bits(np.nan)}, -0.5, 0.0>", False), ("array<f64: 0x3FF80000000000000, -0.5, 0.0>", False)])
def test_spellings_of_coefficients(coef, is_coef):
    assert taken(f" <{{coef = {coef}}}>") == is_coef


def test_an_open_list_is_a_parse_error():
    with pytest.raises(opt.OptError, match="parse error"):
        result(module("tensor<32x3xf32>", hexed(TABLE), "dcf.orthogonalize", " <{coef = array<f64: 1.5, -0.5, 0.0}>",
                      "tensor<32x3xf32>"), n_gpus=0)


@pytest.mark.gpu
@pytest.mark.parametrize("eps,same", [(f64_bits(1e-3) + " : f64", 1e-3), ("0x3A83126F : f32", float(np.float32(1e-3))),
                                      ("1.0e-3 : f32", float(np.float32(1e-3)))])
def test_eps_in_bits_means_its_value(eps, same):
    ty = "tensor<8x8xf32>"
    x = (np.random.default_rng(3).standard_normal((8, 8)) * 1e-3).astype(np.float32)
    a, _ = result(module(ty, hexed(x), "dcf.orthogonalize", f" <{{steps = 0 : i64, eps = {eps}}}>", ty))
    got = np.array(a.const.bits, np.uint32).view(np.float32).reshape(8, 8)
    want = x.astype(np.float64) / (np.sqrt((x.astype(np.float64) ** 2).sum()) + same)
    assert (np.abs(got - want) <= 2 * lo.U32 * np.abs(want)).all()


@pytest.mark.parametrize("value,is_steps", [
    ("3 : i64", True), ("3", True), ("0x3 : i64", True), ("3 : i32", True), ("3 : index", True), ("+3 : i64", False),
    ("3.7 : i64", False), ("3.0 : f64", False), ("3junk : i64", False), ("3 junk", False), ("-1 : i64", False),
    ("0x11 : i64", False), ("0xFFFFFFFFFFFFFFFD : i64", False), ("99999999999999999999 : i64", False), ("300 : i8", False),
    ("0x : i64", False), ("", False), ("true", False), ("3 : tensor<i64>", False), ("3 : i0", False), ("3 : i65", False),
    ("array<i64: 3>", False)])
def test_spellings_of_whole_numbers(value, is_steps):
    assert taken(f" <{{steps = {value}}}>") == is_steps


@pytest.mark.parametrize("value,is_flag", [("true", True), ("false", True), ("true junk", False), ("truejunk", False),
                                           ("1 : i1", False), ("unit", False), ("", False), ("false : i64", False)])
def test_spellings_of_flags(value, is_flag):
    assert taken(f" <{{causal = {value}}}>", "dcf.position_bias", "tensor<3x5x6xf32>") == is_flag


@pytest.mark.gpu
@pytest.mark.parametrize("first,value", [("0x10 : i64", 16), ("0xFFFFFFFFFFFFFFFE : i64", -2), ("0xFE : i8", -2),
                                         ("-3 : i32", -3), ("250 : ui8", 250), ("0xFE : ui8", 254)])
def test_whole_numbers_mean_their_value(first, value):
    d, _ = result(module("tensor<32x3xf32>", hexed(TABLE), "dcf.position_bias", f" <{{first_query = {first}}}>",
                         "tensor<3x5x20xf32>"))
    want = TABLE.T[:, lo.buckets(lo.positions(5, value), 20, 32, 128, True)]
    assert np.array_equal(np.array(d.const.bits, np.uint32).reshape(want.shape), want.view(np.uint32))


@pytest.mark.parametrize("op,out_ty,props", [
    ("dcf.position_bias", "tensor<3x5x6xf32>", " <{casual = true}>"),
    ("dcf.position_bias", "tensor<3x5x6xf32>", " <{num_buckets = 64 : i64}>"),
    ("dcf.position_bias", "tensor<3x5x6xf32>", " <{causal}>"),
    ("dcf.position_bias", "tensor<3x5x6xf32>", " <{steps = 3 : i64}>"),
    ("dcf.position_bias", "tensor<3x5x6xf32>", " <{causal = true, causal = false}>"),
    ("dcf.position_bias", "tensor<3x5x6xf32>", " {causal = true}"),                  # not as a property
    ("dcf.position_bias", "tensor<3x5x6xf32>", " {some.mark = 1 : i64, causal = true}"),
    ("dcf.position_bias", "tensor<3x5x6xf32>", ' {some.mark = "a, b", "causal" = true}'),
    ("dcf.position_bias", "tensor<3x5x6xf32>", " {max_distance = 64 : i64}"),
    ("dcf.position_bias", "tensor<3x5x6xf32>", " {unit}"),
    ("dcf.orthogonalize", "tensor<32x3xf32>", " <{step = 3 : i64}>"),
    ("dcf.orthogonalize", "tensor<32x3xf32>", " <{steps = 3 : i64, causal = false}>"),
    ("dcf.orthogonalize", "tensor<32x3xf32>", " {eps = 1.0e-3 : f64}"),
])
def test_properties_that_the_op_does_not_know(op, out_ty, props):
    assert not taken(props, op, out_ty)


@pytest.mark.parametrize("props", ["", " <{}>", " {}", " {some.mark = 1 : i64}", ' {some.mark = "causal = x, y", other.mark}',
                                   " <{causal = true, first_query = 1 : i64, max_distance = 64 : i64, bidirectional = false}>",
                                   ' <{causal = true}> {some.mark = {a = 1 : i64, b = [1, 2]}, "other.mark" = 2 : i64}'])
def test_properties_and_marks_of_other_dialects_that_fold(props):
    assert taken(props, "dcf.position_bias", "tensor<3x5x6xf32>")


def test_an_op_with_a_region_stays():
    out, stats = opt.run(module("tensor<32x3xf32>", hexed(TABLE), "dcf.position_bias", " ({\n    })", "tensor<3x5x6xf32>"),
                         PIPELINE, n_gpus=0)
    assert '"dcf.position_bias"' in out and stats["folds"] == 0


MEMORY_OF_MANY = """
import sys
import torch
from mlirpass_b200 import opt
def module(n):
    ty = "tensor<1024x1024xbf16>"
    return '"builtin.module"() ({\\n' + "".join(
        f'  "func.func"() <{{function_type = () -> {ty}, sym_name = "f{k}"}}> ({{\\n'
        f'    %0 = "arith.constant"() <{{value = dense<{k + 1}.0> : {ty}}}> : () -> {ty}\\n'
        f'    %1 = "dcf.orthogonalize"(%0) <{{steps = 2 : i64}}> : ({ty}) -> {ty}\\n'
        f'    "func.return"(%1) : ({ty}) -> ()\\n'
        '  }) : () -> ()\\n' for k in range(n)) + '}) : () -> ()\\n'
def used():
    free, total = torch.cuda.mem_get_info()
    return total - free
pipeline = "builtin.module(func.func(learned-constant-fold,canonicalize))"
out, stats = opt.run(module(1), pipeline, n_gpus=1)
one = used()
out, stats = opt.run(module(64), pipeline, n_gpus=1)
assert stats["folds"] == 64 and "dcf.orthogonalize" not in out
print(used() - one)
"""


@pytest.mark.gpu
def test_folds_of_one_batch_share_a_workspace():
    """64 functions, each with a matrix of 2 MB: operands and results (4 MB a function, at most
    twice that in their size classes) stay on the device, a workspace of 16 MB or more each does not."""
    import os
    import subprocess
    import sys
    import conftest
    run = subprocess.run([sys.executable, "-c", MEMORY_OF_MANY], env=dict(os.environ, PYTHONPATH=conftest.ROOT),
                         capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
    assert int(run.stdout) <= 64 * 2 * (4 << 20) + (64 << 20)


@pytest.mark.gpu
def test_operators_of_different_sizes_in_one_batch():
    """Functions whose workspaces differ, folded in one batch, each as it folds alone."""
    rng = np.random.default_rng(9)
    parts, alone = [], {}
    for k, (op, shape, props, out) in enumerate([
            ("dcf.orthogonalize", (150, 170), "", None), ("dcf.position_bias_grad", (2, 3, 300, 200), "", (32, 3)),
            ("dcf.orthogonalize", (2, 30, 40), "", None), ("dcf.orthogonalize", (400, 131), " <{steps = 3 : i64}>", None),
            ("dcf.position_bias", (32, 3), "", (3, 20, 30)), ("dcf.position_bias_grad", (1, 700, 700), " <{causal = true}>", (64, 1)),
            ("dcf.orthogonalize", (64, 64), " <{steps = 0 : i64}>", None)]):
        x = rng.standard_normal(shape).astype(np.float32)
        ty, out_ty = ("tensor<" + "x".join(map(str, s)) + "xf32>" for s in (shape, out or shape))
        text = module(ty, hexed(x), op, props, out_ty, f"f{k}")
        alone[f"f{k}"] = result(text, name=f"f{k}")[0].const.bits
        parts.append(text.split("\n", 1)[1].rsplit("}) : () -> ()", 1)[0])
    out, stats = opt.run('"builtin.module"() ({\n' + "".join(parts) + "}) : () -> ()\n", PIPELINE, n_gpus=1)
    assert stats["folds"] == len(alone)
    funcs = parse_funcs(out)
    for name, bits in alone.items():
        f = funcs[name]
        assert f.defs[f.ret.operands[0]].const.bits == bits
