"""The operators on 8-bit integers, stated in numpy: whole numbers and scales
from their definitions in 64 bits, results in 64 bits and, where a result is
defined to the bit, in the f32 steps that define it."""
import numpy as np

RUN = 128
LEAST = 2.0 ** -119


def levels(x: np.ndarray, top: np.ndarray):
    """(whole numbers, f32 scales) of f64 values, `top` the largest magnitudes beside them."""
    with np.errstate(all="ignore"):
        fine = np.isfinite(top)
        some = fine & (top >= LEAST)
        factor = np.where(some, np.float32(127) / top.astype(np.float32), np.float32(0)).astype(np.float64)
        scale = np.where(some, top.astype(np.float32) / np.float32(127), np.float32(0))
        scale = np.where(fine, scale, np.float32(np.nan)).astype(np.float32)
        # a product of two 24-bit values is exact in 64 bits, and rint takes ties to even
        q = np.where(fine, np.rint(np.where(fine, x, 0) * factor), 0)
    return q.astype(np.int8), scale


def largest(x: np.ndarray, axis: int) -> np.ndarray:
    return np.max(np.abs(x), axis=axis, keepdims=True, initial=0)      # NaN wins


def quantize(x: np.ndarray, along: str):
    """x f64 [rows, cols] -> int8 q, f32 scales in the operator's shape."""
    if along == "rows":
        q, s = levels(x, largest(x, 1))
        return q, s[:, 0]
    parts = [levels(x[r:r + RUN], largest(x[r:r + RUN], 0)) for r in range(0, len(x), RUN)]
    if not parts:
        return np.zeros(x.shape, np.int8), np.zeros((0, x.shape[1]), np.float32)
    return np.concatenate([q for q, _ in parts]), np.concatenate([s for _, s in parts])


def spread(scale: np.ndarray, rows: int, along: str) -> np.ndarray:
    """A scale for every value."""
    return scale[:, None] if along == "rows" else np.repeat(scale, RUN, 0)[:rows]


def values(q: np.ndarray, scale: np.ndarray, along: str) -> np.ndarray:
    """What is read back, as f32."""
    with np.errstate(all="ignore"):
        return q.astype(np.float32) * spread(scale, len(q), along).astype(np.float32)


def matmul(a, a_scale, b, b_scale, bias) -> np.ndarray:
    """The f32 result of int8 a, b (i32 sums where there are no scales)."""
    sums = a.astype(np.int64) @ b.astype(np.int64).T
    if a_scale is None:
        return sums
    with np.errstate(all="ignore"):
        out = sums.astype(np.float32) * a_scale[:, None] * b_scale[None, :]
        return out if bias is None else out + bias[None, :]


def grad(g: np.ndarray, q: np.ndarray, scale: np.ndarray):
    """(result, sum of magnitudes) in 64 bits of f64 g and int8 q."""
    with np.errstate(all="ignore"):
        x = q.astype(np.float64) * spread(scale, len(q), "columns").astype(np.float64)
        return g.T @ x, np.abs(g).T @ np.abs(x)
