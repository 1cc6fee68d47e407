"""mlirpass_b200 — B200-native dense-constant folding for mlirpass.

Python binding of libdcfold.so (include/dcfold.h).  The library replaces the
per-element loops of mlirpass's fold hooks (Folder::binary / Folder::unary in
src/patterns/arith/canonicalize.rs, Tf::transpose / Tf::reciprocal in
src/patterns/tosa/canonicalize.rs) with sm_100a kernels.

Values cross the boundary as raw little-endian element storage: numpy arrays
whose itemsize equals the element size (bit patterns; a float32 array is fine
for f32).  Importing this package does not need a GPU; every compute call
does, and raises DcfError when the library reports no device — there is no
CPU fallback.
"""
from __future__ import annotations

import ctypes
import math
import os
from dataclasses import dataclass

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libdcfold.so")

DTYPES = {
    "i1": 1, "i8": 2, "i16": 3, "i32": 4, "i64": 5,
    "f16": 16, "bf16": 17, "f32": 18, "f64": 19,
    "f8E5M2": 20, "f8E4M3": 21, "f8E3M4": 22,
}
DTYPE_SIZE = {"i1": 1, "i8": 1, "i16": 2, "i32": 4, "i64": 8, "f16": 2, "bf16": 2, "f32": 4, "f64": 8,
              "f8E5M2": 1, "f8E4M3": 1, "f8E3M4": 1}
FLOAT_DTYPES = ("f16", "bf16", "f32", "f64", "f8E5M2", "f8E4M3", "f8E3M4")
INT_DTYPES = ("i1", "i8", "i16", "i32", "i64")
STORAGE = {1: np.uint8, 2: np.uint16, 4: np.uint32, 8: np.uint64}

OPS = {
    "addf": 1, "subf": 2, "mulf": 3, "divf": 4, "maximumf": 5, "minimumf": 6, "maxnumf": 7, "minnumf": 8,
    "remf": 9,
    "addi": 16, "subi": 17, "muli": 18, "andi": 19, "ori": 20, "xori": 21, "shli": 22, "shrui": 23,
    "shrsi": 24, "divsi": 25, "divui": 26, "remsi": 27, "remui": 28, "maxsi": 29, "maxui": 30,
    "minsi": 31, "minui": 32, "ceildivui": 33, "ceildivsi": 34, "floordivsi": 35, "mulsi_hi": 36,
    "mului_hi": 37, "cmpi": 48, "cmpf": 49, "addui_carry": 50,
    "extf": 64, "truncf": 65, "sitofp": 66, "uitofp": 67, "fptosi": 68, "fptoui": 69,
    "negf": 70, "flush_denormals": 71, "extsi": 72, "extui": 73, "trunci": 74,
    "reciprocal": 80,
    # math dialect (exact folds only)
    "absf": 96, "ceil": 97, "floor": 98, "roundeven": 99, "round": 100, "trunc": 101, "sqrt": 102,
    "rsqrt": 103, "absi": 104, "ctlz": 105, "cttz": 106, "ctpop": 107, "copysign": 112, "ipowi": 113,
}
BINARY_OPS = tuple(k for k, v in OPS.items() if v < 64 or k in ("copysign", "ipowi"))
FLOAT_BINARY_OPS = tuple(k for k, v in OPS.items() if v < 16 or k in ("cmpf", "copysign"))
MATH_FLOAT_UNARY_OPS = ("absf", "ceil", "floor", "roundeven", "round", "trunc", "sqrt", "rsqrt")
MATH_INT_UNARY_OPS = ("absi", "ctlz", "cttz", "ctpop")
INT_BINARY_OPS = tuple(k for k in BINARY_OPS if k not in FLOAT_BINARY_OPS)
BOOL_RESULT_OPS = ("cmpi", "cmpf", "addui_carry")
CONVERT_OPS = ("extf", "truncf", "sitofp", "uitofp", "fptosi", "fptoui", "negf", "flush_denormals", "extsi",
               "extui", "trunci") + MATH_FLOAT_UNARY_OPS + MATH_INT_UNARY_OPS

FLAG_PRED_SHIFT = 8
FLAG_NEG_DEFAULT_NAN = 1 << 16

ERRORS = {-1: "EINVAL", -2: "ENODEV", -3: "ENOMEM", -4: "ECUDA", -5: "EUNSUPPORTED", -6: "ETIMEOUT",
          -7: "EPARSE"}


def flags(roundingmode: int = 0, predicate: int = 0, neg_default_nan: bool = False) -> int:
    """Pack the flags word (DCF_FLAG_* in include/dcfold.h)."""
    return (roundingmode & 7) | ((predicate & 15) << FLAG_PRED_SHIFT) | (FLAG_NEG_DEFAULT_NAN if neg_default_nan else 0)


class DcfError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"dcfold {ERRORS.get(code, code)}: {msg}")
        self.code = code


class Result(ctypes.Structure):
    _fields_ = [("folded", ctypes.c_uint8), ("is_splat", ctypes.c_uint8), ("reserved", ctypes.c_uint8 * 6),
                ("first_fail_index", ctypes.c_uint64)]


class Status(ctypes.Structure):
    _fields_ = [("first_fail", ctypes.c_uint64), ("splat_word", ctypes.c_uint32), ("error", ctypes.c_uint32)]


class Job(ctypes.Structure):
    _fields_ = [("op", ctypes.c_uint32), ("dtype", ctypes.c_uint32), ("out_dtype", ctypes.c_uint32),
                ("flags", ctypes.c_uint32), ("lhs", ctypes.c_void_p), ("rhs", ctypes.c_void_p),
                ("out", ctypes.c_void_p), ("n", ctypes.c_uint64), ("lhs_splat", ctypes.c_uint8),
                ("rhs_splat", ctypes.c_uint8), ("reserved", ctypes.c_uint8 * 6), ("result", Result)]


class BiasDesc(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_uint32), ("table_dtype", ctypes.c_uint32), ("num_buckets", ctypes.c_uint32),
                ("max_distance", ctypes.c_uint32), ("flags", ctypes.c_uint32), ("heads", ctypes.c_uint32),
                ("batch", ctypes.c_uint64), ("queries", ctypes.c_uint64), ("keys", ctypes.c_uint64),
                ("first_query", ctypes.c_int64), ("row_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64),
                ("batch_stride", ctypes.c_int64)]


ORTH_MAX_STEPS = 16


class OrthDesc(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_uint32), ("out_dtype", ctypes.c_uint32), ("steps", ctypes.c_uint32),
                ("reserved", ctypes.c_uint32), ("batch", ctypes.c_uint64), ("rows", ctypes.c_uint64),
                ("cols", ctypes.c_uint64), ("row_stride", ctypes.c_int64), ("batch_stride", ctypes.c_int64),
                ("out_row_stride", ctypes.c_int64), ("out_batch_stride", ctypes.c_int64), ("eps", ctypes.c_double),
                ("coef", (ctypes.c_double * 3) * ORTH_MAX_STEPS)]


class QuantDesc(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_uint32), ("along", ctypes.c_uint32), ("rows", ctypes.c_uint64),
                ("cols", ctypes.c_uint64), ("row_stride", ctypes.c_int64), ("q_row_stride", ctypes.c_int64)]


class Int8Desc(ctypes.Structure):
    _fields_ = [("a_dtype", ctypes.c_uint32), ("out_dtype", ctypes.c_uint32), ("tokens", ctypes.c_uint64),
                ("channels", ctypes.c_uint64), ("depth", ctypes.c_uint64), ("a_row_stride", ctypes.c_int64),
                ("b_row_stride", ctypes.c_int64), ("out_row_stride", ctypes.c_int64)]


class CheckpointDesc(ctypes.Structure):
    _fields_ = [("grad_dtype", ctypes.c_uint32), ("out_dtype", ctypes.c_uint32), ("flags", ctypes.c_uint32),
                ("reserved", ctypes.c_uint32), ("tokens", ctypes.c_uint64), ("channels", ctypes.c_uint64),
                ("depth", ctypes.c_uint64), ("grad_row_stride", ctypes.c_int64), ("q_row_stride", ctypes.c_int64),
                ("out_row_stride", ctypes.c_int64)]


# Every symbol include/dcfold.h declares, with its ctypes signature.
_VP, _U64, _I, _U32, _SZ = ctypes.c_void_p, ctypes.c_uint64, ctypes.c_int, ctypes.c_uint32, ctypes.c_size_t
_RP, _SP = ctypes.POINTER(Result), ctypes.POINTER(Status)
_BP, _OP, _SZP = ctypes.POINTER(BiasDesc), ctypes.POINTER(OrthDesc), ctypes.POINTER(ctypes.c_size_t)
_QP, _IP, _CP = ctypes.POINTER(QuantDesc), ctypes.POINTER(Int8Desc), ctypes.POINTER(CheckpointDesc)
SIGNATURES = {
    "dcf_init": (_I, [_I]),
    "dcf_shutdown": (_I, []),
    "dcf_device_count": (_I, []),
    "dcf_last_error": (ctypes.c_char_p, []),
    "dcf_version": (ctypes.c_char_p, []),
    "dcf_dtype_size": (_SZ, [_I]),
    "dcf_kernel_launches": (_U64, []),
    "dcf_binary": (_I, [_I, _I, _VP, _I, _VP, _I, _U64, _U32, _VP, _RP]),
    "dcf_convert": (_I, [_I, _I, _I, _VP, _I, _U64, _U32, _VP, _RP]),
    "dcf_reciprocal": (_I, [_I, _VP, _I, _U64, _U32, _VP, _RP]),
    "dcf_select": (_I, [_SZ, _VP, _I, _VP, _I, _VP, _I, _U64, _VP, _RP]),
    "dcf_transpose": (_I, [_SZ, _I, ctypes.POINTER(ctypes.c_int64), ctypes.POINTER(ctypes.c_int64), _VP, _VP, _RP]),
    "dcf_hex_encode": (_I, [_VP, _U64, _VP]),
    "dcf_hex_decode": (_I, [_VP, _U64, _VP]),
    "dcf_splat_check": (_I, [_VP, _SZ, _U64, ctypes.POINTER(ctypes.c_int)]),
    "dcf_batch": (_I, [ctypes.POINTER(Job), _SZ]),
    "dcf_batch_noalloc": (_I, [ctypes.POINTER(Job), _SZ, _VP]),
    "dcf_status_reset_async": (_I, [_VP, _VP]),
    "dcf_binary_async": (_I, [_I, _I, _VP, _I, _VP, _I, _U64, _U32, _VP, _VP, _VP]),
    "dcf_convert_async": (_I, [_I, _I, _I, _VP, _I, _U64, _U32, _VP, _VP, _VP]),
    "dcf_reciprocal_async": (_I, [_I, _VP, _I, _U64, _U32, _VP, _VP, _VP]),
    "dcf_select_async": (_I, [_SZ, _VP, _I, _VP, _I, _VP, _I, _U64, _VP, _VP, _VP]),
    "dcf_transpose2d_async": (_I, [_SZ, _U64, _U64, _VP, _VP, _VP]),
    "dcf_permute_async": (_I, [_SZ, _I, ctypes.POINTER(ctypes.c_int64), ctypes.POINTER(ctypes.c_int64), _VP, _VP,
                               _VP]),
    "dcf_permute_status_async": (_I, [_SZ, _I, ctypes.POINTER(ctypes.c_int64), ctypes.POINTER(ctypes.c_int64), _VP,
                                      _VP, _VP, _VP]),
    "dcf_splat_check_async": (_I, [_VP, _SZ, _U64, _VP, _VP]),
    "dcf_hex_encode_async": (_I, [_VP, _U64, _VP, _VP]),
    "dcf_hex_decode_async": (_I, [_VP, _U64, _VP, _VP, _VP]),
    "dcf_hex_decode_many_async": (_I, [_VP, _SZ, _U64, _VP, _VP]),
    "dcf_hash_many_async": (_I, [_VP, _SZ, _U64, _VP, _VP]),
    "dcf_status_read": (_I, [_VP, _VP, _RP]),
    "dcf_position_bias": (_I, [_BP, _VP, _VP, _VP, _RP]),
    "dcf_position_bias_grad": (_I, [_BP, _VP, _VP, _VP, _RP]),
    "dcf_orthogonalize": (_I, [_OP, _VP, _VP, _RP]),
    "dcf_position_bias_async": (_I, [_BP, _VP, _VP, _VP, _VP]),
    "dcf_position_bias_grad_workspace": (_I, [_BP, _SZP]),
    "dcf_position_bias_grad_async": (_I, [_BP, _VP, _VP, _VP, _VP, _SZ, _VP]),
    "dcf_orthogonalize_workspace": (_I, [_OP, _SZP]),
    "dcf_orthogonalize_async": (_I, [_OP, _VP, _VP, _VP, _SZ, _VP, _VP]),
    "dcf_quantize": (_I, [_QP, _VP, _VP, _VP, _RP]),
    "dcf_dequantize": (_I, [_QP, _VP, _VP, _VP, _RP]),
    "dcf_int8_matmul": (_I, [_IP, _VP, _VP, _VP, _VP, _VP, _VP, _RP]),
    "dcf_checkpoint_grad": (_I, [_CP, _VP, _VP, _VP, _VP, _RP]),
    "dcf_quantize_async": (_I, [_QP, _VP, _VP, _VP, _VP]),
    "dcf_dequantize_async": (_I, [_QP, _VP, _VP, _VP, _VP]),
    "dcf_int8_matmul_workspace": (_I, [_IP, _SZP]),
    "dcf_int8_matmul_async": (_I, [_IP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _SZ, _VP, _VP]),
    "dcf_checkpoint_grad_workspace": (_I, [_CP, _SZP]),
    "dcf_checkpoint_grad_async": (_I, [_CP, _VP, _VP, _VP, _VP, _VP, _SZ, _VP, _VP]),
}

_lib = None


def lib() -> ctypes.CDLL:
    """Load libdcfold.so (built by `python -m mlirpass_b200.build`)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"{LIB_PATH} is missing: run `python -m mlirpass_b200.build` first")
        L = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def _check(rc: int) -> int:
    if rc < 0:
        raise DcfError(rc, lib().dcf_last_error().decode())
    return rc


def init(n_gpus: int = 1) -> int:
    """Choose the GPUs host calls shard over (devices 0..n-1)."""
    return _check(lib().dcf_init(n_gpus))


def shutdown() -> None:
    _check(lib().dcf_shutdown())


def device_count() -> int:
    return lib().dcf_device_count()


def kernel_launches() -> int:
    """Kernels launched by libdcfold.so in this process so far."""
    return int(lib().dcf_kernel_launches())


def storage(dtype: str):
    return STORAGE[DTYPE_SIZE[dtype]]


def as_storage(x, dtype: str) -> np.ndarray:
    """A C-contiguous numpy view of x with the element storage of dtype."""
    a = np.ascontiguousarray(x)
    st = storage(dtype)
    if a.dtype.itemsize != np.dtype(st).itemsize:
        raise ValueError(f"array itemsize {a.dtype.itemsize} does not match {dtype}")
    return a.view(st).reshape(-1)


@dataclass
class Fold:
    """Outcome of one fold: `out` is meaningful only when `folded`."""
    folded: bool
    is_splat: bool
    first_fail_index: int
    out: np.ndarray | None


def _ptr(a: np.ndarray):
    return a.ctypes.data_as(ctypes.c_void_p)


def binary(op: str, dtype: str, lhs, rhs, *, n: int | None = None, lhs_splat: bool = False,
           rhs_splat: bool = False, flags: int = 0, out: np.ndarray | None = None) -> Fold:
    """Elementwise binary fold (Folder::binary's loop) on host buffers."""
    l, r = as_storage(lhs, dtype), as_storage(rhs, dtype)
    if n is None:
        n = 1 if (lhs_splat and rhs_splat) else max(len(l), len(r))
    odt = "i1" if op in BOOL_RESULT_OPS else dtype
    if out is None:
        out = np.empty(n, dtype=storage(odt))
    res = Result()
    _check(lib().dcf_binary(OPS[op], DTYPES[dtype], _ptr(l), int(lhs_splat), _ptr(r), int(rhs_splat), n, flags,
                            _ptr(out), ctypes.byref(res)))
    return Fold(bool(res.folded), bool(res.is_splat), int(res.first_fail_index), out)


def convert(op: str, from_dtype: str, to_dtype: str, x, *, n: int | None = None, splat: bool = False,
            flags: int = 0, out: np.ndarray | None = None) -> Fold:
    """Elementwise conversion fold (the Const::map closures of Folder::unary)."""
    a = as_storage(x, from_dtype)
    if n is None:
        n = len(a)
    if out is None:
        out = np.empty(n, dtype=storage(to_dtype))
    res = Result()
    _check(lib().dcf_convert(OPS[op], DTYPES[from_dtype], DTYPES[to_dtype], _ptr(a), int(splat), n, flags,
                             _ptr(out), ctypes.byref(res)))
    return Fold(bool(res.folded), bool(res.is_splat), int(res.first_fail_index), out)


def reciprocal(dtype: str, x, *, n: int | None = None, splat: bool = False, flags: int = 0,
               out: np.ndarray | None = None) -> Fold:
    a = as_storage(x, dtype)
    if n is None:
        n = len(a)
    if out is None:
        out = np.empty(n, dtype=storage(dtype))
    res = Result()
    _check(lib().dcf_reciprocal(DTYPES[dtype], _ptr(a), int(splat), n, flags, _ptr(out), ctypes.byref(res)))
    return Fold(bool(res.folded), bool(res.is_splat), int(res.first_fail_index), out)


def select(cond, t, f, *, n: int | None = None, cond_splat: bool = False, t_splat: bool = False,
           f_splat: bool = False, out: np.ndarray | None = None) -> Fold:
    """Elementwise select over dense constants (Folder::select's value loop):
    out[i] = t[i] if cond[i] else f[i].  t and f share one storage dtype."""
    c = np.ascontiguousarray(cond, dtype=np.uint8).reshape(-1)
    a = np.ascontiguousarray(t).reshape(-1)
    b = np.ascontiguousarray(f).reshape(-1)
    if a.dtype.itemsize != b.dtype.itemsize:
        raise ValueError("t and f must have the same element size")
    if n is None:
        n = max(len(c), len(a), len(b))
    if out is None:
        out = np.empty(n, dtype=a.dtype)
    res = Result()
    _check(lib().dcf_select(a.dtype.itemsize, _ptr(c), int(cond_splat), _ptr(a), int(t_splat), _ptr(b),
                            int(f_splat), n, _ptr(out), ctypes.byref(res)))
    return Fold(bool(res.folded), bool(res.is_splat), int(res.first_fail_index), out)


def transpose(x: np.ndarray, shape, perms, out: np.ndarray | None = None) -> Fold:
    """Permute a dense row-major tensor (elements of x's itemsize)."""
    a = np.ascontiguousarray(x).reshape(-1)
    rank = len(shape)
    if out is None:
        out = np.empty_like(a)
    sh = (ctypes.c_int64 * rank)(*shape)
    pm = (ctypes.c_int64 * rank)(*perms)
    res = Result()
    _check(lib().dcf_transpose(a.dtype.itemsize, rank, sh, pm, _ptr(a), _ptr(out), ctypes.byref(res)))
    out_shape = [shape[p] for p in perms]
    return Fold(bool(res.folded), bool(res.is_splat), int(res.first_fail_index), out.reshape(out_shape))


def hex_encode(data) -> bytes:
    a = np.frombuffer(bytes(data), dtype=np.uint8) if not isinstance(data, np.ndarray) else \
        np.ascontiguousarray(data).view(np.uint8).reshape(-1)
    out = np.empty(2 * len(a), dtype=np.uint8)
    _check(lib().dcf_hex_encode(_ptr(a), len(a), _ptr(out)))
    return out.tobytes()


def hex_decode(text) -> bytes:
    t = text.encode() if isinstance(text, str) else bytes(text)
    a = np.frombuffer(t, dtype=np.uint8)
    out = np.empty(len(a) // 2, dtype=np.uint8)
    _check(lib().dcf_hex_decode(_ptr(a), len(a), _ptr(out)))
    return out.tobytes()


def splat_check(x) -> bool:
    a = np.ascontiguousarray(x).reshape(-1)
    v = ctypes.c_int(0)
    _check(lib().dcf_splat_check(_ptr(a), a.dtype.itemsize, len(a), ctypes.byref(v)))
    return bool(v.value)


def batch(jobs: list[dict]) -> list[Fold]:
    """Run independent folds in one launch per (op, dtype) group per GPU.

    Each job dict: op, dtype, [out_dtype], lhs, [rhs], [lhs_splat], [rhs_splat], [n], [flags].
    """
    arr = (Job * len(jobs))()
    keep = []
    outs = []
    for i, j in enumerate(jobs):
        op, dt = j["op"], j["dtype"]
        odt = j.get("out_dtype") or ("i1" if op in BOOL_RESULT_OPS else dt)
        l = as_storage(j["lhs"], dt)
        r = as_storage(j["rhs"], dt) if "rhs" in j else None
        n = j.get("n") or max(len(l), len(r) if r is not None else 0)
        o = np.empty(n, dtype=storage(odt))
        keep += [l, r]
        outs.append(o)
        arr[i].op, arr[i].dtype, arr[i].out_dtype = OPS[op], DTYPES[dt], DTYPES[odt]
        arr[i].flags = j.get("flags", 0)
        arr[i].lhs = l.ctypes.data
        arr[i].rhs = r.ctypes.data if r is not None else None
        arr[i].out = o.ctypes.data
        arr[i].n = n
        arr[i].lhs_splat = int(j.get("lhs_splat", False))
        arr[i].rhs_splat = int(j.get("rhs_splat", False))
    _check(lib().dcf_batch(arr, len(jobs)))
    return [Fold(bool(arr[i].result.folded), bool(arr[i].result.is_splat), int(arr[i].result.first_fail_index),
                 outs[i]) for i in range(len(jobs))]


# ------------------------------------------------------------------ device

NOALLOC_MAX_JOBS = 1024


def batch_noalloc(jobs: list[dict], stream=None) -> list[Fold]:
    """dcf_batch_noalloc: folds on device tensors with no allocation at all.

    For callers that cannot allocate device memory while they fold (their
    allocator owns all of HBM, or they cannot afford the synchronisation of
    cudaMalloc).  Each job dict: op, dtype, [out_dtype], lhs, [rhs], out
    (torch CUDA tensors on one device), [lhs_splat], [rhs_splat], [n],
    [flags].  At most NOALLOC_MAX_JOBS jobs per call; overlapping calls on
    the GPU race on the library's one scratch array.
    """
    arr = device_jobs(jobs)
    run_device_jobs(arr, stream)
    return [Fold(bool(arr[i].result.folded), bool(arr[i].result.is_splat), int(arr[i].result.first_fail_index),
                 None) for i in range(len(jobs))]


def device_jobs(jobs: list[dict]):
    """The ctypes job table of batch_noalloc, built once so that a caller can
    run the same batch repeatedly (run_device_jobs)."""
    arr = (Job * len(jobs))()
    for i, j in enumerate(jobs):
        op, dt = j["op"], j["dtype"]
        odt = j.get("out_dtype") or ("i1" if op in BOOL_RESULT_OPS else dt)
        arr[i].op, arr[i].dtype, arr[i].out_dtype = OPS[op], DTYPES[dt], DTYPES[odt]
        arr[i].flags = j.get("flags", 0)
        arr[i].lhs = _tptr(j["lhs"])
        arr[i].rhs = _tptr(j["rhs"]) if "rhs" in j else None
        arr[i].out = _tptr(j["out"])
        arr[i].n = j.get("n") or j["out"].numel()
        arr[i].lhs_splat = int(j.get("lhs_splat", False))
        arr[i].rhs_splat = int(j.get("rhs_splat", False))
    return arr


def run_device_jobs(arr, stream=None) -> None:
    """dcf_batch_noalloc on a table from device_jobs; results land in it."""
    _check(lib().dcf_batch_noalloc(arr, len(arr), _stream(stream)))

def _tptr(t) -> int:
    return t.data_ptr()


def _stream(stream) -> int:
    if stream is None:
        import torch
        return torch.cuda.current_stream().cuda_stream
    return stream if isinstance(stream, int) else stream.cuda_stream


def status_reset(status, stream=None) -> None:
    _check(lib().dcf_status_reset_async(_tptr(status), _stream(stream)))


def binary_async(op: str, dtype: str, lhs, rhs, out, status, *, n: int | None = None, lhs_splat: bool = False,
                 rhs_splat: bool = False, flags: int = 0, stream=None) -> None:
    """Launch a binary fold on device tensors (no synchronisation)."""
    if n is None:
        n = out.numel()
    _check(lib().dcf_binary_async(OPS[op], DTYPES[dtype], _tptr(lhs), int(lhs_splat), _tptr(rhs), int(rhs_splat), n,
                                  flags, _tptr(out), _tptr(status), _stream(stream)))


def convert_async(op: str, from_dtype: str, to_dtype: str, x, out, status, *, n: int | None = None,
                  splat: bool = False, flags: int = 0, stream=None) -> None:
    if n is None:
        n = out.numel()
    _check(lib().dcf_convert_async(OPS[op], DTYPES[from_dtype], DTYPES[to_dtype], _tptr(x), int(splat), n, flags,
                                   _tptr(out), _tptr(status), _stream(stream)))


def reciprocal_async(dtype: str, x, out, status, *, n: int | None = None, splat: bool = False, flags: int = 0,
                     stream=None) -> None:
    if n is None:
        n = out.numel()
    _check(lib().dcf_reciprocal_async(DTYPES[dtype], _tptr(x), int(splat), n, flags, _tptr(out), _tptr(status),
                                      _stream(stream)))


def select_async(cond, t, f, out, status, *, n: int | None = None, cond_splat: bool = False, t_splat: bool = False,
                 f_splat: bool = False, stream=None) -> None:
    if n is None:
        n = out.numel()
    _check(lib().dcf_select_async(out.element_size(), _tptr(cond), int(cond_splat), _tptr(t), int(t_splat), _tptr(f),
                                  int(f_splat), n, _tptr(out), _tptr(status), _stream(stream)))


def permute_async(elem_size: int, shape, perms, x, out, status, stream=None) -> None:
    """dcf_permute_status_async on device tensors (2-byte transposes take the
    bulk-tensor kernel)."""
    rank = len(shape)
    sh = (ctypes.c_int64 * rank)(*shape)
    pm = (ctypes.c_int64 * rank)(*perms)
    _check(lib().dcf_permute_status_async(elem_size, rank, sh, pm, _tptr(x), _tptr(out), _tptr(status),
                                          _stream(stream)))


def transpose2d_async(elem_size: int, rows: int, cols: int, x, out, stream=None) -> None:
    _check(lib().dcf_transpose2d_async(elem_size, rows, cols, _tptr(x), _tptr(out), _stream(stream)))


def hex_encode_async(x, nbytes: int, out, stream=None) -> None:
    _check(lib().dcf_hex_encode_async(_tptr(x), nbytes, _tptr(out), _stream(stream)))


def hex_decode_async(x, nchars: int, out, status, stream=None) -> None:
    _check(lib().dcf_hex_decode_async(_tptr(x), nchars, _tptr(out), _tptr(status), _stream(stream)))


def status_read(status, stream=None) -> Fold:
    res = Result()
    _check(lib().dcf_status_read(_tptr(status), _stream(stream), ctypes.byref(res)))
    return Fold(bool(res.folded), bool(res.is_splat), int(res.first_fail_index), None)


# ------------------------------------------- operators on learned tensors

BIAS_BIDIRECTIONAL, BIAS_CAUSAL, BIAS_ACCUMULATE = 1, 2, 4
# The quintic whose singular values settle between about 0.7 and 1.2 in five steps.
ORTH_COEF = (3.4445, -4.7750, 2.0315)


class BiasPlan:
    """The sizes, types and strides of one position bias: a dcf_bias_desc
    that calls reuse.  What no call takes is refused when it is made; what the bias
    alone does not take (rows that overlap, a table of another type, accumulation) by its call."""

    def __init__(self, desc: BiasDesc, dtype: str, table_dtype: str):
        self.desc, self.dtype, self.table_dtype = desc, dtype, table_dtype
        self.ref = ctypes.byref(desc)
        d = desc
        row = d.row_stride or d.keys
        head = d.head_stride or d.queries * row
        batch = d.batch_stride or d.heads * head
        some = d.queries and d.keys and d.heads
        span = (d.queries - 1) * row + (d.heads - 1) * head + d.keys if some else 0
        self.out_elements = span                     # elements from a bias's first to its last
        self.grad_elements = span + (d.batch - 1) * batch if some and d.batch else 0
        self.entries = d.num_buckets * d.heads
        self.out_layout = (d.heads, d.queries, d.keys), (head, row, 1)
        self.grad_layout = (d.batch, d.heads, d.queries, d.keys), (batch, head, row, 1)
        ws = ctypes.c_size_t(0)
        _check(lib().dcf_position_bias_grad_workspace(self.ref, ctypes.byref(ws)))
        self.workspace = ws.value


def position_bias_plan(dtype: str, heads: int, queries: int, keys: int, *, num_buckets: int = 32,
                       max_distance: int = 128, bidirectional: bool = True, causal: bool = False,
                       first_query: int = 0, batch: int = 1, table_dtype: str | None = None, row_stride: int = 0,
                       head_stride: int = 0, batch_stride: int = 0, accumulate: bool = False) -> BiasPlan:
    """Describe a relative position bias (dcf_bias_desc, include/dcfold.h).

    The bias is [heads, queries, keys] of `dtype`, its gradient [batch,
    heads, queries, keys]; the table is [num_buckets, heads] of table_dtype
    (dtype, or f32 beside f16 / bf16).  Strides are in elements, 0 is dense.
    `accumulate` makes the gradient add to what its output holds.
    """
    for name, v in (("heads", heads), ("queries", queries), ("keys", keys), ("batch", batch),
                    ("num_buckets", num_buckets), ("max_distance", max_distance)):
        if not 0 <= v < 1 << 31:
            raise ValueError(f"{name} {v} out of range")
    for name, v in (("first_query", first_query), ("row_stride", row_stride), ("head_stride", head_stride),
                    ("batch_stride", batch_stride)):
        if not -(1 << 62) < v < 1 << 62:
            raise ValueError(f"{name} {v} out of range")
    table_dtype = table_dtype or dtype
    flags = (BIAS_BIDIRECTIONAL if bidirectional else 0) | (BIAS_CAUSAL if causal else 0) | \
        (BIAS_ACCUMULATE if accumulate else 0)
    desc = BiasDesc(DTYPES[dtype], DTYPES[table_dtype], num_buckets, max_distance, flags, heads, batch, queries, keys,
                    first_query, row_stride, head_stride, batch_stride)
    return BiasPlan(desc, dtype, table_dtype)


def position_bias(plan: BiasPlan, table, *, positions=None, out: np.ndarray | None = None) -> Fold:
    """The bias [heads, queries, keys] of a table on host buffers."""
    d = plan.desc
    t = as_storage(table, plan.table_dtype)
    if len(t) != plan.entries:
        raise ValueError(f"table has {len(t)} elements, {plan.entries} expected")
    n = d.heads * d.queries * d.keys
    out = _host_out(out, n, plan.dtype)
    p = _host_positions(positions, d.queries)
    res = Result()
    _check(lib().dcf_position_bias(plan.ref, _ptr(t), _ptr(p) if p is not None else None, _ptr(out),
                                   ctypes.byref(res)))
    return Fold(bool(res.folded), bool(res.is_splat), int(res.first_fail_index),
                out.reshape(d.heads, d.queries, d.keys))


def position_bias_grad(plan: BiasPlan, grad, *, positions=None, out: np.ndarray | None = None) -> Fold:
    """The table's gradient [num_buckets, heads] on host buffers: f32, f64
    for a f64 bias.  With an accumulating plan `out` is added to."""
    d = plan.desc
    g = as_storage(grad, plan.dtype)
    n = d.batch * d.heads * d.queries * d.keys
    if len(g) != n:
        raise ValueError(f"gradient has {len(g)} elements, {n} expected")
    wide = np.float64 if plan.dtype == "f64" else np.float32
    if out is None:
        if d.flags & BIAS_ACCUMULATE:
            raise ValueError("an accumulating plan needs `out`")
        out = np.empty((d.num_buckets, d.heads), wide)
    elif out.dtype != wide or out.size != plan.entries or not out.flags.c_contiguous:
        raise ValueError("out must be a contiguous f32 (f64 for f64) array of the table's size")
    p = _host_positions(positions, d.queries)
    res = Result()
    _check(lib().dcf_position_bias_grad(plan.ref, _ptr(g), _ptr(p) if p is not None else None, _ptr(out),
                                        ctypes.byref(res)))
    return Fold(bool(res.folded), bool(res.is_splat), int(res.first_fail_index), out)


def _host_positions(positions, queries: int):
    if positions is None:
        return None
    given = np.asarray(positions).reshape(-1)
    if len(given) != queries:
        raise ValueError(f"{len(given)} positions for {queries} queries")
    if given.dtype.kind not in "biuf":
        raise ValueError(f"positions: {given.dtype}, whole numbers expected")
    with np.errstate(invalid="ignore"):
        p = np.ascontiguousarray(given, dtype=np.int32)
    if not np.array_equal(p, given):                    # a cast wraps and cuts without a word
        raise ValueError("positions: whole numbers of 32 bits expected")
    return p


def _host_out(out, n: int, dtype: str) -> np.ndarray:
    if out is None:
        return np.empty(n, dtype=storage(dtype))
    if out.size != n or out.dtype.itemsize != DTYPE_SIZE[dtype] or not out.flags.c_contiguous:
        raise ValueError(f"out must be a contiguous array of {n} {dtype} elements")
    return out.reshape(-1)


_CURRENT_STREAM: list = []


def _own_stream(stream, t) -> int:
    """The given stream, or the current one of the tensor's device."""
    if stream is None:
        if not _CURRENT_STREAM:
            import torch
            raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # without a Stream object: 2 us less
            _CURRENT_STREAM.append(raw or (lambda device: torch.cuda.current_stream(device).cuda_stream))
        return _CURRENT_STREAM[0](t.get_device())
    return stream if isinstance(stream, int) else stream.cuda_stream


def _room(t) -> int:
    """Elements from a tensor's first one to the end of its storage."""
    return t.untyped_storage().nbytes() // t.element_size() - t.storage_offset()


_TORCH_TYPES: dict = {}


def _load_torch_types() -> None:
    import torch
    _TORCH_TYPES.update(f16=torch.float16, bf16=torch.bfloat16, f32=torch.float32, f64=torch.float64, i32=torch.int32,
                        i8=torch.int8)


def _typed(t, what: str, dtype: str) -> None:
    """Refuse a tensor whose elements are not of the given type (another of the same size would be read as it)."""
    if not _TORCH_TYPES:
        _load_torch_types()
    if t.dtype is not _TORCH_TYPES[dtype]:
        raise ValueError(f"{what}: {t.dtype}, {dtype} expected")


def _need(t, what: str, elements: int, dtype: str | None) -> int:
    """The pointer of a dense tensor of at least `elements` of a type (None: any of 8 bytes)."""
    if dtype:
        _typed(t, what, dtype)
    elif t.element_size() != 8:
        raise ValueError(f"{what}: elements of {t.element_size()} bytes, 8 expected")
    if elements and (not t.is_contiguous() or t.numel() < elements):
        raise ValueError(f"{what}: {elements} contiguous elements expected, not {tuple(t.shape)} with strides {t.stride()}")
    return t.data_ptr()


def _memory(shape, strides) -> list:
    """The (stride, size) pairs of a layout, the longest stride first, dims that join joined."""
    dims = []
    for stride, size in sorted(((t, n) for n, t in zip(shape, strides) if n > 1), reverse=True):
        if dims and dims[-1][0] == stride * size:
            dims[-1] = (stride, dims[-1][1] * size)
        else:
            dims.append((stride, size))
    return dims


def _lies_as(t, shape, strides) -> bool:
    """Whether a tensor without all of a layout's elements in a row has them where the layout says:
    it is the layout (or wider along some of its dims), or the same memory in another
    order or number of dims, or a plain row that starts at its first element."""
    have, at = list(t.shape), list(t.stride())
    while len(have) > len(shape) and have[0] == 1:
        have, at = have[1:], at[1:]
    count = math.prod(shape)
    if len(have) <= 1 and t.is_contiguous():
        return t.numel() != count
    rest = len(shape) - len(have)
    if rest >= 0 and all(n == 1 for n in shape[:rest]):
        if all(n <= 1 or (h >= n and a == s) for h, a, n, s in zip(have, at, shape[rest:], strides[rest:])):
            return True
        if tuple(have) == tuple(shape[rest:]):
            return False
    return _memory(have, at) == _memory(shape, strides)


def _need_layout(t, what: str, elements: int, dtype: str, shape, strides) -> int:
    """The pointer of a tensor in which the plan's layout, `elements` from its first to its last, lies."""
    _typed(t, what, dtype)
    own = t.is_contiguous() and t.numel() >= elements or t.stride() == strides and t.shape == shape
    if elements and not own:
        if _room(t) < elements:
            raise ValueError(f"{what}: {_room(t)} elements behind the pointer, {elements} needed")
        if not _lies_as(t, shape, strides):
            raise ValueError(f"{what}: {tuple(t.shape)} with strides {t.stride()}, the plan says {shape} with {strides}")
    return t.data_ptr()


def _positions(positions, queries: int):
    if positions is None:
        return None
    return _need(positions, "positions", queries, "i32")


def _bytes(workspace) -> int:
    if not workspace.is_contiguous():
        raise ValueError("workspace: not contiguous")
    return workspace.numel() * workspace.element_size()


def position_bias_async(plan: BiasPlan, table, out, *, positions=None, stream=None) -> None:
    """Launch a position bias on device tensors.  `table` and `positions` are dense;
    `out` starts at the bias's first element and lies as the plan's strides say
    (a tensor of the bias's shape with these strides, or the memory around it)."""
    _check(lib().dcf_position_bias_async(
        plan.ref, _need(table, "table", plan.entries, plan.table_dtype),
        _positions(positions, plan.desc.queries),
        _need_layout(out, "out", plan.out_elements, plan.dtype, *plan.out_layout), _own_stream(stream, out)))


def position_bias_grad_workspace(plan: BiasPlan) -> int:
    """Bytes of device workspace that a gradient call of this plan needs."""
    return plan.workspace


def position_bias_grad_async(plan: BiasPlan, grad, out, workspace, *, positions=None, stream=None) -> None:
    """Launch the table gradient on device tensors: `grad` lies as the plan's
    strides say, `out` is the dense [num_buckets, heads] gradient, `workspace`
    uint8 (may be empty when position_bias_grad_workspace says 0)."""
    _check(lib().dcf_position_bias_grad_async(
        plan.ref, _need_layout(grad, "grad", plan.grad_elements, plan.dtype, *plan.grad_layout),
        _positions(positions, plan.desc.queries),
        _need(out, "out", plan.entries, "f64" if plan.dtype == "f64" else "f32"), workspace.data_ptr(),
        _bytes(workspace), _own_stream(stream, out)))


class OrthPlan:
    """The sizes, strides and coefficients of one orthogonalisation: a
    dcf_orth_desc that calls reuse.  Validated when made."""

    def __init__(self, desc: OrthDesc, dtype: str, out_dtype: str):
        self.desc, self.dtype, self.out_dtype = desc, dtype, out_dtype
        self.ref = ctypes.byref(desc)
        d = desc

        def span(row, batch):
            if not (d.rows and d.cols and d.batch):
                return 0
            row = row or d.cols
            return (d.rows - 1) * row + d.cols + (d.batch - 1) * (batch or d.rows * row)

        def layout(row, batch):
            row = row or d.cols
            return (d.batch, d.rows, d.cols), (batch or d.rows * row, row, 1)
        self.in_layout, self.out_layout = layout(d.row_stride, d.batch_stride), layout(d.out_row_stride, d.out_batch_stride)
        self.in_elements = span(d.row_stride, d.batch_stride)
        self.out_elements = span(d.out_row_stride, d.out_batch_stride)
        ws = ctypes.c_size_t(0)
        _check(lib().dcf_orthogonalize_workspace(self.ref, ctypes.byref(ws)))
        self.workspace = ws.value


def orthogonalize_plan(dtype: str, rows: int, cols: int, *, batch: int = 1, steps: int = 5, coef=ORTH_COEF,
                       eps: float = 1e-7, out_dtype: str | None = None, row_stride: int = 0, batch_stride: int = 0,
                       out_row_stride: int = 0, out_batch_stride: int = 0) -> OrthPlan:
    """Describe a Newton-Schulz orthogonalisation (dcf_orth_desc,
    include/dcfold.h).  `coef` is one (a, b, c) for every step, or one per step."""
    for name, v in (("rows", rows), ("cols", cols), ("batch", batch)):
        if not 0 <= v < 1 << 31:
            raise ValueError(f"{name} {v} out of range")
    for name, v in (("row_stride", row_stride), ("batch_stride", batch_stride), ("out_row_stride", out_row_stride),
                    ("out_batch_stride", out_batch_stride)):
        if not -(1 << 62) < v < 1 << 62:
            raise ValueError(f"{name} {v} out of range")
    if not 0 <= steps <= ORTH_MAX_STEPS:
        raise ValueError(f"steps must be 0 .. {ORTH_MAX_STEPS}")
    per_step = [coef] * steps if len(coef) == 0 or not hasattr(coef[0], "__len__") else list(coef)
    if len(per_step) != steps or any(len(c) != 3 for c in per_step):
        raise ValueError("coef is three numbers, or three for each step")
    out_dtype = out_dtype or dtype
    desc = OrthDesc(DTYPES[dtype], DTYPES[out_dtype], steps, 0, batch, rows, cols, row_stride, batch_stride,
                    out_row_stride, out_batch_stride, eps)
    for i, c in enumerate(per_step):
        for j in range(3):
            desc.coef[i][j] = float(c[j])
    return OrthPlan(desc, dtype, out_dtype)


def orthogonalize(plan: OrthPlan, x, *, out: np.ndarray | None = None) -> Fold:
    """Orthogonalise [batch, rows, cols] on host buffers."""
    d = plan.desc
    a = as_storage(x, plan.dtype)
    n = d.batch * d.rows * d.cols
    if len(a) != n:
        raise ValueError(f"input has {len(a)} elements, {n} expected")
    out = _host_out(out, n, plan.out_dtype)
    res = Result()
    _check(lib().dcf_orthogonalize(plan.ref, _ptr(a), _ptr(out), ctypes.byref(res)))
    return Fold(bool(res.folded), bool(res.is_splat), int(res.first_fail_index), out.reshape(d.batch, d.rows, d.cols))


def orthogonalize_workspace(plan: OrthPlan) -> int:
    """Bytes of device workspace that a call of this plan needs."""
    return plan.workspace


def orthogonalize_async(plan: OrthPlan, x, out, workspace, status, *, stream=None) -> None:
    """Launch an orthogonalisation on device tensors, which lie as the plan's strides
    say; `out` may be `x`.
    `status` (16 bytes, reset first) takes a kernel's error report."""
    _check(lib().dcf_orthogonalize_async(
        plan.ref, _need_layout(x, "x", plan.in_elements, plan.dtype, *plan.in_layout),
        _need_layout(out, "out", plan.out_elements, plan.out_dtype, *plan.out_layout), workspace.data_ptr(),
        _bytes(workspace), _need(status, "status", 2, None), _own_stream(stream, out)))


# -------------------------------------------- operators on 8-bit integers

QUANT_RUN = 128                                        # rows of a run that shares a scale for each column
QUANT_ALONG = {"rows": 0, "columns": 1}
INT8_MAX_DEPTH = 131071
CHECKPOINT_ACCUMULATE = 1


def _rows(rows: int, cols: int, stride: int) -> tuple:
    """A matrix as (elements from its first to its last, shape, strides)."""
    stride = stride or cols
    return (rows - 1) * stride + cols if rows and cols else 0, (rows, cols), (stride, 1)


def _torch_type(dtype: str):
    if not _TORCH_TYPES:
        _load_torch_types()
    return _TORCH_TYPES[dtype]


def _at(t, what: str, dtype: str, rows: tuple) -> int:
    """The pointer of a tensor in which a matrix of _rows lies; one with exactly its shape and strides needs no
    further look."""
    if t.dtype is _torch_type(dtype) and t.stride() == rows[2] and t.shape == rows[1]:
        return t.data_ptr()
    return _need_layout(t, what, rows[0], dtype, *rows[1:])


def _floats(t, what: str, elements: int) -> int:
    """The pointer of a dense f32 tensor of at least `elements`."""
    if t.dtype is _torch_type("f32") and t.is_contiguous() and t.numel() >= elements:
        return t.data_ptr()
    return _need(t, what, elements, "f32")


def _fits(limit: int, **sizes) -> None:
    for name, v in sizes.items():
        if not 0 <= v < limit:
            raise ValueError(f"{name} {v} out of range")


def _vector(t, what: str, elements: int):
    return None if t is None else _floats(t, what, elements)


class QuantPlan:
    """The sizes, type and strides of a matrix and its 8-bit form: a
    dcf_quant_desc that calls reuse."""

    def __init__(self, desc: QuantDesc, dtype: str):
        self.desc, self.dtype = desc, dtype
        self.ref = ctypes.byref(desc)
        self.values = _rows(desc.rows, desc.cols, desc.row_stride)
        self.levels = _rows(desc.rows, desc.cols, desc.q_row_stride)
        self.scale_shape = (desc.rows,) if desc.along == 0 else (-(-desc.rows // QUANT_RUN), desc.cols)
        self.scales = math.prod(self.scale_shape)
        self.quantize, self.dequantize = lib().dcf_quantize_async, lib().dcf_dequantize_async


def quantize_plan(dtype: str, rows: int, cols: int, *, along: str = "rows", row_stride: int = 0,
                  q_row_stride: int = 0) -> QuantPlan:
    """Describe a matrix [rows, cols] of f16, bf16 or f32 and its 8-bit form
    (dcf_quant_desc, include/dcfold.h).

    `along` "rows" has a scale for each row, [rows]; "columns" one for each
    column of each run of 128 rows, [ceil(rows / 128), cols]: a checkpoint of
    activations.  Strides are in elements, 0 is dense.
    """
    _fits(1 << 31, rows=rows, cols=cols)
    _fits(1 << 62, row_stride=row_stride, q_row_stride=q_row_stride)
    if dtype not in ("f16", "bf16", "f32"):
        raise ValueError(f"dtype {dtype}: f16, bf16 or f32 expected")
    return QuantPlan(QuantDesc(DTYPES[dtype], QUANT_ALONG[along], rows, cols, row_stride, q_row_stride), dtype)


def quantize(plan: QuantPlan, x) -> tuple:
    """(Fold of int8 [rows, cols], f32 scales) of a matrix on host buffers."""
    d = plan.desc
    a = as_storage(x, plan.dtype)
    if len(a) != d.rows * d.cols:
        raise ValueError(f"input has {len(a)} elements, {d.rows * d.cols} expected")
    q, scale, res = np.empty((d.rows, d.cols), np.int8), np.empty(plan.scale_shape, np.float32), Result()
    _check(lib().dcf_quantize(plan.ref, _ptr(a), _ptr(q), _ptr(scale), ctypes.byref(res)))
    return Fold(bool(res.folded), bool(res.is_splat), int(res.first_fail_index), q), scale


def dequantize(plan: QuantPlan, q, scale, *, out: np.ndarray | None = None) -> Fold:
    """The values [rows, cols] that whole numbers and scales stand for, on host buffers."""
    d = plan.desc
    n = d.rows * d.cols
    a, s = _host_array(q, "q", n, np.int8), _host_array(scale, "scale", plan.scales, np.float32)
    out = _host_out(out, n, plan.dtype)
    res = Result()
    _check(lib().dcf_dequantize(plan.ref, _ptr(a), _ptr(s), _ptr(out), ctypes.byref(res)))
    return Fold(bool(res.folded), bool(res.is_splat), int(res.first_fail_index), out.reshape(d.rows, d.cols))


def _host_array(x, what: str, n: int, dtype) -> np.ndarray:
    a = np.ascontiguousarray(x).reshape(-1)
    if a.dtype != dtype or a.size != n:
        raise ValueError(f"{what}: {a.size} elements of {a.dtype}, {n} of {np.dtype(dtype)} expected")
    return a


def quantize_async(plan: QuantPlan, x, q, scale, *, stream=None) -> None:
    """Launch a quantisation on device tensors: `x` and the int8 `q` lie as the
    plan's strides say, the f32 `scale` is dense, of the plan's scale_shape."""
    _check(plan.quantize(plan.ref, _at(x, "x", plan.dtype, plan.values), _at(q, "q", "i8", plan.levels),
                         _floats(scale, "scale", plan.scales), _own_stream(stream, q)))


def dequantize_async(plan: QuantPlan, q, scale, out, *, stream=None) -> None:
    """Launch the reading back of what quantize_async wrote, into `out` as the plan's strides say."""
    _check(plan.dequantize(plan.ref, _at(q, "q", "i8", plan.levels), _floats(scale, "scale", plan.scales),
                           _at(out, "out", plan.dtype, plan.values), _own_stream(stream, out)))


class Int8Plan:
    """The sizes, types and strides of one 8-bit product: a dcf_int8_desc that
    calls reuse.  Validated when made."""

    def __init__(self, desc: Int8Desc, a_dtype: str, out_dtype: str):
        self.desc, self.a_dtype, self.out_dtype = desc, a_dtype, out_dtype
        self.ref = ctypes.byref(desc)
        self.a = _rows(desc.tokens, desc.depth, desc.a_row_stride)
        self.b = _rows(desc.channels, desc.depth, desc.b_row_stride)
        self.out = _rows(desc.tokens, desc.channels, desc.out_row_stride)
        ws = ctypes.c_size_t(0)
        _check(lib().dcf_int8_matmul_workspace(self.ref, ctypes.byref(ws)))
        self.workspace = ws.value
        self.tokens, self.channels, self.call = desc.tokens, desc.channels, lib().dcf_int8_matmul_async


def int8_matmul_plan(tokens: int, channels: int, depth: int, *, a_dtype: str = "i8", out_dtype: str = "bf16",
                     a_row_stride: int = 0, b_row_stride: int = 0, out_row_stride: int = 0) -> Int8Plan:
    """Describe the product of tokens [tokens, depth] and an int8 weight
    [channels, depth] (dcf_int8_desc, include/dcfold.h).

    Tokens are i8 with a scale each, or f16, bf16 or f32, which the call
    quantises by rows.  The result [tokens, channels] is f16, bf16 or f32, or,
    of i8 tokens, the i32 sums.  Strides are in elements, 0 is dense.
    """
    _fits(1 << 31, tokens=tokens, channels=channels, depth=depth)
    _fits(1 << 62, a_row_stride=a_row_stride, b_row_stride=b_row_stride, out_row_stride=out_row_stride)
    return Int8Plan(Int8Desc(DTYPES[a_dtype], DTYPES[out_dtype], tokens, channels, depth, a_row_stride, b_row_stride,
                             out_row_stride), a_dtype, out_dtype)


def int8_matmul(plan: Int8Plan, a, b, *, a_scale=None, b_scale=None, bias=None, out: np.ndarray | None = None) -> Fold:
    """The product [tokens, channels] on host buffers."""
    d = plan.desc
    x = as_storage(a, plan.a_dtype)
    if len(x) != d.tokens * d.depth:
        raise ValueError(f"a has {len(x)} elements, {d.tokens * d.depth} expected")
    w = _host_array(b, "b", d.channels * d.depth, np.int8)
    given = [None if v is None else _host_array(v, what, n, np.float32)
             for v, what, n in ((a_scale, "a_scale", d.tokens), (b_scale, "b_scale", d.channels), (bias, "bias", d.channels))]
    sa, sb, add = (None if v is None else _ptr(v) for v in given)
    out = _host_out(out, d.tokens * d.channels, plan.out_dtype)
    res = Result()
    _check(lib().dcf_int8_matmul(plan.ref, _ptr(x), sa, _ptr(w), sb, add, _ptr(out), ctypes.byref(res)))
    return Fold(bool(res.folded), bool(res.is_splat), int(res.first_fail_index), out.reshape(d.tokens, d.channels))


def int8_matmul_workspace(plan: Int8Plan) -> int:
    """Bytes of device workspace that a call of this plan needs."""
    return plan.workspace


def int8_matmul_async(plan: Int8Plan, a, b, out, workspace, status, *, a_scale=None, b_scale=None, bias=None,
                      stream=None) -> None:
    """Launch an 8-bit product on device tensors: `a`, the int8 weight `b` and
    `out` lie as the plan's strides say; `a_scale` [tokens] (of i8 tokens),
    `b_scale` and `bias` [channels] are dense f32.  `status` (16 bytes, reset
    first) takes a kernel's error report."""
    _check(plan.call(
        plan.ref, _at(a, "a", plan.a_dtype, plan.a), _vector(a_scale, "a_scale", plan.tokens),
        _at(b, "b", "i8", plan.b), _vector(b_scale, "b_scale", plan.channels), _vector(bias, "bias", plan.channels),
        _at(out, "out", plan.out_dtype, plan.out), workspace.data_ptr(), _bytes(workspace),
        _need(status, "status", 2, None), _own_stream(stream, out)))


class CheckpointPlan:
    """The sizes, types and strides of one weight gradient from a checkpoint: a
    dcf_checkpoint_desc that calls reuse.  Validated when made."""

    def __init__(self, desc: CheckpointDesc, dtype: str, out_dtype: str):
        self.desc, self.dtype, self.out_dtype = desc, dtype, out_dtype
        self.ref = ctypes.byref(desc)
        self.grad = _rows(desc.tokens, desc.channels, desc.grad_row_stride)
        self.levels = _rows(desc.tokens, desc.depth, desc.q_row_stride)
        self.out = _rows(desc.channels, desc.depth, desc.out_row_stride)
        self.scale_shape = -(-desc.tokens // QUANT_RUN), desc.depth
        self.scales = math.prod(self.scale_shape)
        ws = ctypes.c_size_t(0)
        _check(lib().dcf_checkpoint_grad_workspace(self.ref, ctypes.byref(ws)))
        self.workspace = ws.value
        self.call = lib().dcf_checkpoint_grad_async


def checkpoint_grad_plan(dtype: str, tokens: int, channels: int, depth: int, *, out_dtype: str = "f32",
                         grad_row_stride: int = 0, q_row_stride: int = 0, out_row_stride: int = 0,
                         accumulate: bool = False) -> CheckpointPlan:
    """Describe the gradient [channels, depth] of a weight from the f16 or bf16
    gradient [tokens, channels] of its layer's output and the checkpoint
    [tokens, depth] of its input, quantised along columns (dcf_checkpoint_desc,
    include/dcfold.h).  Strides are in elements, 0 is dense.  `accumulate` adds
    to what a f32 result holds.
    """
    _fits(1 << 31, tokens=tokens, channels=channels, depth=depth)
    _fits(1 << 62, grad_row_stride=grad_row_stride, q_row_stride=q_row_stride, out_row_stride=out_row_stride)
    flags = CHECKPOINT_ACCUMULATE if accumulate else 0
    return CheckpointPlan(CheckpointDesc(DTYPES[dtype], DTYPES[out_dtype], flags, 0, tokens, channels, depth,
                                         grad_row_stride, q_row_stride, out_row_stride), dtype, out_dtype)


def checkpoint_grad(plan: CheckpointPlan, grad, q, scale, *, out: np.ndarray | None = None) -> Fold:
    """The gradient [channels, depth] on host buffers.  With an accumulating plan `out` is added to."""
    d = plan.desc
    g = as_storage(grad, plan.dtype)
    if len(g) != d.tokens * d.channels:
        raise ValueError(f"gradient has {len(g)} elements, {d.tokens * d.channels} expected")
    if out is None and d.flags & CHECKPOINT_ACCUMULATE:
        raise ValueError("an accumulating plan needs `out`")
    a, s = _host_array(q, "q", d.tokens * d.depth, np.int8), _host_array(scale, "scale", plan.scales, np.float32)
    out = _host_out(out, d.channels * d.depth, plan.out_dtype)
    res = Result()
    _check(lib().dcf_checkpoint_grad(plan.ref, _ptr(g), _ptr(a), _ptr(s), _ptr(out), ctypes.byref(res)))
    return Fold(bool(res.folded), bool(res.is_splat), int(res.first_fail_index), out.reshape(d.channels, d.depth))


def checkpoint_grad_workspace(plan: CheckpointPlan) -> int:
    """Bytes of device workspace that a call of this plan needs."""
    return plan.workspace


def checkpoint_grad_async(plan: CheckpointPlan, grad, q, scale, out, workspace, status, *, stream=None) -> None:
    """Launch a weight gradient on device tensors: `grad`, the int8 `q` and `out`
    lie as the plan's strides say, the f32 `scale` is dense, of the plan's
    scale_shape.  `status` (16 bytes, reset first) takes a kernel's error report."""
    _check(plan.call(
        plan.ref, _at(grad, "grad", plan.dtype, plan.grad), _at(q, "q", "i8", plan.levels),
        _floats(scale, "scale", plan.scales), _at(out, "out", plan.out_dtype, plan.out), workspace.data_ptr(),
        _bytes(workspace), _need(status, "status", 2, None), _own_stream(stream, out)))
