"""learned-constant-fold and the operators on 8-bit integers: they fold where
all of their operands are constants, and stay as they are where their types,
shapes or properties are not the operator's."""
import numpy as np
import pytest

import int8_oracle as io
from mlir_text import parse_funcs
from mlirpass_b200 import opt

PIPELINE = "builtin.module(func.func(learned-constant-fold,canonicalize))"
NAMES = {"int8": "i8", "int32": "i32", "float32": "f32", "float16": "f16", "float64": "f64"}


def ty(a) -> str:
    if isinstance(a, str):
        return a
    return "tensor<" + "".join(f"{d}x" for d in a.shape) + NAMES[str(a.dtype)] + ">"


def literal(a: np.ndarray) -> str:
    flat = a.reshape(-1)
    if len(flat) == 1:
        return f"dense<{flat[0]}>"
    return f'dense<"0x{a.tobytes().hex().upper()}">'


def body(op: str, operands, props: str, results, name: str = "f") -> str:
    outs = ", ".join(results)
    lines = [f'  "func.func"() <{{function_type = () -> ({outs}), sym_name = "{name}"}}> ({{\n']
    for i, a in enumerate(operands):
        lines.append(f'    %{i} = "arith.constant"() <{{value = {literal(a)} : {ty(a)}}}> : () -> {ty(a)}\n')
    n = len(operands)
    ins, ins_ty = ", ".join(f"%{i}" for i in range(n)), ", ".join(ty(a) for a in operands)
    res = f"%{n}" + (f":{len(results)}" if len(results) > 1 else "")
    back = ", ".join(f"%{n}#{i}" for i in range(len(results))) if len(results) > 1 else f"%{n}"
    to = f"({outs})" if len(results) > 1 else outs
    lines.append(f'    {res} = "{op}"({ins}){props} : ({ins_ty}) -> {to}\n    "func.return"({back}) : ({outs}) -> ()\n  }}) : () -> ()\n')
    return "".join(lines)


def module(*args, **kw) -> str:
    return '"builtin.module"() ({\n' + body(*args, **kw) + "}) : () -> ()\n"


def constants(out: str, name: str = "f"):
    f = parse_funcs(out)[name]
    defs = [f.defs[v] for v in f.ret.operands]
    assert all(d.name == "arith.constant" for d in defs), [d.name for d in defs]
    return [d.const for d in defs]


def bits(const, dtype, shape) -> np.ndarray:
    raw = np.array(const.bits, {1: np.uint8, 2: np.uint16, 4: np.uint32}[np.dtype(dtype).itemsize]).view(dtype)
    return np.broadcast_to(raw, shape).copy() if const.splat else raw.reshape(shape)


RNG = np.random.default_rng(0)
X = RNG.standard_normal((140, 40)).astype(np.float32)
A, B = RNG.integers(-127, 128, (9, 40)).astype(np.int8), RNG.integers(-127, 128, (11, 40)).astype(np.int8)
SA, SB, ADD = (RNG.random(n).astype(np.float32) for n in (9, 11, 11))
G = RNG.integers(-4, 5, (140, 6)).astype(np.float16)
Q, S = RNG.integers(-15, 16, (140, 40)).astype(np.int8), (2.0 ** RNG.integers(0, 4, (2, 40))).astype(np.float32)


@pytest.mark.parametrize("op,operands,props,results", [
    ("dcf.quantize", [X], "", ["tensor<140x40xi8>"]),                                        # one result
    ("dcf.quantize", [X], "", ["tensor<140x40xi8>", "tensor<40xf32>"]),
    ("dcf.quantize", [X], "", ["tensor<140x40xi16>", "tensor<140xf32>"]),
    ("dcf.quantize", [X], "", ["tensor<140x40xi8>", "tensor<140xf16>"]),
    ("dcf.quantize", [X], "", ["tensor<40x140xi8>", "tensor<140xf32>"]),
    ("dcf.quantize", [X], " <{columns = true}>", ["tensor<140x40xi8>", "tensor<140xf32>"]),
    ("dcf.quantize", [X], " <{columns = true}>", ["tensor<140x40xi8>", "tensor<3x40xf32>"]),
    ("dcf.quantize", [X], " <{rows = true}>", ["tensor<140x40xi8>", "tensor<140xf32>"]),
    ("dcf.quantize", [X], " <{columns = 1 : i1}>", ["tensor<140x40xi8>", "tensor<2x40xf32>"]),
    ("dcf.quantize", [X], " {columns = true}", ["tensor<140x40xi8>", "tensor<2x40xf32>"]),
    ("dcf.quantize", [X.astype(np.float64)], "", ["tensor<140x40xi8>", "tensor<140xf32>"]),
    ("dcf.quantize", [A], "", ["tensor<9x40xi8>", "tensor<9xf32>"]),
    ("dcf.quantize", [X.reshape(-1)], "", ["tensor<5600xi8>", "tensor<1xf32>"]),
    ("dcf.quantize", [X, X], "", ["tensor<140x40xi8>", "tensor<140xf32>"]),
    ("dcf.dequantize", [Q], "", ["tensor<140x40xf32>"]),
    ("dcf.dequantize", [Q, S], "", ["tensor<140x40xf32>"]),
    ("dcf.dequantize", [Q, S], " <{columns = true}>", ["tensor<140x40xf64>"]),
    ("dcf.dequantize", [X, S], " <{columns = true}>", ["tensor<140x40xf32>"]),
    ("dcf.int8_matmul", [A, B], "", ["tensor<9x11xi64>"]),
    ("dcf.int8_matmul", [A, B], "", ["tensor<11x9xi32>"]),
    ("dcf.int8_matmul", [A, B], "", ["tensor<9x11xf32>"]),
    ("dcf.int8_matmul", [A, SA, B, SB], "", ["tensor<9x11xi32>"]),
    ("dcf.int8_matmul", [A, B, SB], "", ["tensor<9x11xf32>"]),
    ("dcf.int8_matmul", [A, SB, B, SA], "", ["tensor<9x11xf32>"]),
    ("dcf.int8_matmul", [A, SA, B, SB, ADD, ADD], "", ["tensor<9x11xf32>"]),
    ("dcf.int8_matmul", [A, SA, B, SB, SA], "", ["tensor<9x11xf32>"]),
    ("dcf.int8_matmul", [A, SA, B, SB], "", ["tensor<9x11xf64>"]),
    ("dcf.int8_matmul", [A, SA, B, SB], " <{columns = true}>", ["tensor<9x11xf32>"]),
    ("dcf.int8_matmul", [A, SA, B[:, :39].copy(), SB], "", ["tensor<9x11xf32>"]),
    ("dcf.int8_matmul", [X, SA, B, SB], "", ["tensor<140x11xf32>"]),
    ("dcf.int8_matmul", [X, B], "", ["tensor<140x11xi32>"]),
    ("dcf.checkpoint_grad", [G, Q, S], "", ["tensor<40x6xf32>"]),
    ("dcf.checkpoint_grad", [G, Q], "", ["tensor<6x40xf32>"]),
    ("dcf.checkpoint_grad", [G.astype(np.float32), Q, S], "", ["tensor<6x40xf32>"]),
    ("dcf.checkpoint_grad", [G, Q, S[:1].copy()], "", ["tensor<6x40xf32>"]),
    ("dcf.checkpoint_grad", [G[:139].copy(), Q, S], "", ["tensor<6x40xf32>"]),
    ("dcf.checkpoint_grad", [G, Q, S], " <{accumulate = true}>", ["tensor<6x40xf32>"]),
])
def test_ops_that_stay(op, operands, props, results):
    out, stats = opt.run(module(op, operands, props, results), PIPELINE, n_gpus=0)
    assert f'"{op}"' in out and stats["folds"] == 0


TAKEN = [
    ("dcf.quantize", [X], "", ["tensor<140x40xi8>", "tensor<140xf32>"]),
    ("dcf.quantize", [X], " <{columns = false}> {some.mark}", ["tensor<140x40xi8>", "tensor<140xf32>"]),
    ("dcf.quantize", [X], " <{columns = true}>", ["tensor<140x40xi8>", "tensor<2x40xf32>"]),
    ("dcf.dequantize", [Q, S], " <{columns = true}>", ["tensor<140x40xbf16>"]),
    ("dcf.int8_matmul", [A, B], "", ["tensor<9x11xi32>"]),
    ("dcf.int8_matmul", [A, SA, B, SB], "", ["tensor<9x11xf32>"]),
    ("dcf.int8_matmul", [A, SA, B, SB, ADD], "", ["tensor<9x11xf16>"]),
    ("dcf.int8_matmul", [X, B, SB], "", ["tensor<140x11xbf16>"]),
    ("dcf.int8_matmul", [X, B, SB, ADD], "", ["tensor<140x11xf32>"]),
    ("dcf.checkpoint_grad", [G, Q, S], "", ["tensor<6x40xf32>"]),
]


@pytest.mark.parametrize("op,operands,props,results", TAKEN)
def test_ops_that_are_taken(op, operands, props, results):
    with pytest.raises(Exception, match="needs a GPU"):
        opt.run(module(op, operands, props, results), PIPELINE, n_gpus=0)
    for pipeline in ("canonicalize", "builtin.module(func.func(tosa-layerwise-constant-fold,canonicalize))"):
        out, stats = opt.run(module(op, operands, props, results), pipeline, n_gpus=0)
        assert f'"{op}"' in out and stats["folds"] == 0


def test_an_operand_that_is_no_constant_keeps_the_op():
    text = module("dcf.int8_matmul", [A, B], "", ["tensor<9x11xi32>"]).replace(
        f'"arith.constant"() <{{value = {literal(B)} : {ty(B)}}}>', '"some.source"()')
    out, stats = opt.run(text, PIPELINE, n_gpus=0)
    assert '"dcf.int8_matmul"' in out and stats["folds"] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("along", ["rows", "columns"])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_quantize_folds_and_folds_back(along, dtype):
    x = X.astype(dtype)
    props = " <{columns = true}>" if along == "columns" else ""
    q, s = io.quantize(x.astype(np.float64), along)
    out, stats = opt.run(module("dcf.quantize", [x], props, ["tensor<140x40xi8>", ty(s)]), PIPELINE, n_gpus=1)
    got_q, got_s = constants(out)
    assert stats["folds"] == 1
    assert np.array_equal(bits(got_q, np.int8, q.shape), q) and np.array_equal(bits(got_s, np.float32, s.shape), s)
    out, _ = opt.run(module("dcf.dequantize", [q, s], props, [ty(x)]), PIPELINE, n_gpus=1)
    (got,) = constants(out)
    assert np.array_equal(bits(got, dtype, x.shape), io.values(q, s, along).astype(dtype))


@pytest.mark.gpu
def test_quantize_of_a_splat_gives_splats():
    text = module("dcf.quantize", [X], " <{columns = true}>", ["tensor<140x40xi8>", "tensor<2x40xf32>"]).replace(
        literal(X), "dense<2.54>")
    q, s = constants(opt.run(text, PIPELINE, n_gpus=1)[0])
    assert q.splat and s.splat and q.bits[0] == 127
    assert np.uint32(s.bits[0]) == (np.float32(2.54) / np.float32(127)).view(np.uint32)


@pytest.mark.gpu
def test_products_fold():
    (got,) = constants(opt.run(module("dcf.int8_matmul", [A, B], "", ["tensor<9x11xi32>"]), PIPELINE, n_gpus=1)[0])
    assert np.array_equal(bits(got, np.int32, (9, 11)), io.matmul(A, None, B, None, None))
    for add in (None, ADD):
        more = [] if add is None else [add]
        (got,) = constants(opt.run(module("dcf.int8_matmul", [A, SA, B, SB] + more, "", ["tensor<9x11xf32>"]), PIPELINE, n_gpus=1)[0])
        assert np.array_equal(bits(got, np.float32, (9, 11)), io.matmul(A, SA, B, SB, add))
        (got,) = constants(opt.run(module("dcf.int8_matmul", [X, B, SB] + more, "", ["tensor<140x11xf32>"]), PIPELINE, n_gpus=1)[0])
        assert np.array_equal(bits(got, np.float32, (140, 11)), io.matmul(*io.quantize(X.astype(np.float64), "rows"), B, SB, add))


@pytest.mark.gpu
@pytest.mark.parametrize("n_gpus_flags", [{}, {"verbatim": True}])
def test_gradient_folds(n_gpus_flags):
    (got,) = constants(opt.run(module("dcf.checkpoint_grad", [G, Q, S], "", ["tensor<6x40xf32>"]), PIPELINE, n_gpus=1, **n_gpus_flags)[0])
    want, _ = io.grad(G.astype(np.float64), Q, S)
    assert np.array_equal(bits(got, np.float32, (6, 40)), want.astype(np.float32))


@pytest.mark.gpu
def test_a_chain_of_them_folds_through():
    """A learned weight is quantised, multiplied and read back in one module; scales go from one op to the next."""
    w = RNG.standard_normal((24, 40)).astype(np.float32)
    text = ('"builtin.module"() ({\n  "func.func"() <{function_type = () -> (tensor<140x24xf32>, tensor<24x40xf32>), sym_name = "f"}> ({\n'
            f'    %0 = "arith.constant"() <{{value = {literal(X)} : {ty(X)}}}> : () -> {ty(X)}\n'
            f'    %1 = "arith.constant"() <{{value = {literal(w)} : {ty(w)}}}> : () -> {ty(w)}\n'
            '    %2:2 = "dcf.quantize"(%1) : (tensor<24x40xf32>) -> (tensor<24x40xi8>, tensor<24xf32>)\n'
            '    %3 = "dcf.int8_matmul"(%0, %2#0, %2#1) : (tensor<140x40xf32>, tensor<24x40xi8>, tensor<24xf32>) -> tensor<140x24xf32>\n'
            '    %4 = "dcf.dequantize"(%2#0, %2#1) : (tensor<24x40xi8>, tensor<24xf32>) -> tensor<24x40xf32>\n'
            '    "func.return"(%3, %4) : (tensor<140x24xf32>, tensor<24x40xf32>) -> ()\n  }) : () -> ()\n}) : () -> ()\n')
    out, stats = opt.run(text, PIPELINE, n_gpus=1)
    y, back = constants(out)
    wq, ws = io.quantize(w.astype(np.float64), "rows")
    xq, xs = io.quantize(X.astype(np.float64), "rows")
    assert stats["folds"] == 3
    assert np.array_equal(bits(y, np.float32, (140, 24)), io.matmul(xq, xs, wq, ws, None))
    assert np.array_equal(bits(back, np.float32, (24, 40)), io.values(wq, ws, "rows"))


@pytest.mark.gpu
def test_many_functions_in_one_batch():
    """Folds of different kinds and workspaces in one batch, each as it folds alone."""
    parts, alone = [], {}
    for k, (op, operands, props, results) in enumerate(TAKEN):
        name = f"f{k}"
        alone[name] = [c.bits for c in constants(opt.run(module(op, operands, props, results, name), PIPELINE, n_gpus=1)[0], name)]
        parts.append(body(op, operands, props, results, name))
    out, stats = opt.run('"builtin.module"() ({\n' + "".join(parts) + "}) : () -> ()\n", PIPELINE, n_gpus=1)
    assert stats["folds"] == len(TAKEN)
    for name, want in alone.items():
        assert [c.bits for c in constants(out, name)] == want
