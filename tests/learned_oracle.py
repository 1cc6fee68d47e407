"""Plain 64-bit statements of the operators on learned tensors, from their
definitions (include/dcfold.h), and the bounds their tests compare with."""
import math

import numpy as np

U32 = 2.0 ** -24          # half a step of f32
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": U32, "f64": 2.0 ** -53}


def bucket(d: int, num_buckets: int, max_distance: int, bidirectional: bool) -> int:
    """The bucket of d = key - query in whole numbers alone."""
    half = num_buckets // 2 if bidirectional else num_buckets
    base = half if bidirectional and d > 0 else 0
    n = abs(d) if bidirectional else max(-d, 0)
    e = half // 2
    if half == 1:
        return base
    if n < e:
        return base + n
    m, k = half - e, 0
    # the largest k <= m with n^m e^k >= D^k e^m
    while k < m and n ** m * e ** (k + 1) >= max_distance ** (k + 1) * e ** m:
        k += 1
    return base + min(half - 1, e + k)


def starts(num_buckets: int, max_distance: int, bidirectional: bool) -> list[int]:
    """The first distance of each bucket of one direction."""
    half = num_buckets // 2 if bidirectional else num_buckets
    e = half // 2
    m, out = half - e, list(range(min(e + 1, half)))
    for k in range(1, m if half > 1 else 0):
        low, high = e, max_distance          # the smallest n with n^m e^k >= D^k e^m
        while low < high:
            mid = (low + high) // 2
            if mid ** m * e ** k >= max_distance ** k * e ** m:
                high = mid
            else:
                low = mid + 1
        out.append(low)
    return out


def buckets(q_pos, keys: int, num_buckets: int, max_distance: int, bidirectional: bool) -> np.ndarray:
    """[queries, keys] of bucket numbers."""
    d = np.arange(keys, dtype=np.int64)[None, :] - np.asarray(q_pos, np.int64)[:, None]
    begin = np.array(starts(num_buckets, max_distance, bidirectional), np.int64)
    n = np.abs(d) if bidirectional else np.maximum(-d, 0)
    return np.searchsorted(begin, n, side="right") - 1 + np.where(d > 0, num_buckets // 2 if bidirectional else 0, 0)


def positions(queries: int, first: int, given=None) -> np.ndarray:
    return np.asarray(given, np.int64) if given is not None else first + np.arange(queries, dtype=np.int64)


def masked(q_pos, keys: int) -> np.ndarray:
    return np.arange(keys, dtype=np.int64)[None, :] > np.asarray(q_pos, np.int64)[:, None]


def bias_grad(g: np.ndarray, ids: np.ndarray, num_buckets: int, hidden=None):
    """(gradient, sum of magnitudes), both [num_buckets, heads], of g [batch, heads, queries, keys]."""
    g = g.astype(np.float64)
    if hidden is not None:
        g = np.where(hidden, 0.0, g)
    heads = g.shape[1]
    out, mag = np.zeros((num_buckets, heads)), np.zeros((num_buckets, heads))
    for h in range(heads):
        s, a = g[:, h].sum(0).reshape(-1), np.abs(g[:, h]).sum(0).reshape(-1)
        out[:, h] = np.bincount(ids.reshape(-1), s, num_buckets)
        mag[:, h] = np.bincount(ids.reshape(-1), a, num_buckets)
    return out, mag


def bias_grad_bound(mag, batch: int, queries: int, keys: int, vector: int, half_step: float) -> np.ndarray:
    """A sum's rounding error: every value passes at most as many additions
    as its lane makes (a lane has one vector in 32 of a row) and the joins
    of lanes, warps and splits, each off by half a step of the partial sum."""
    additions = batch * queries * (keys / 32 + 2 * vector) + 1024
    return additions * half_step * mag + 1e-300


def newton_schulz(g: np.ndarray, coef, eps: float, wobble=None) -> np.ndarray:
    """The iteration on [rows, cols] in 64 bits.  `wobble(x, y)` may return
    an error to add to the product x y."""
    x = g.astype(np.float64)
    turned = x.shape[0] > x.shape[1]
    if turned:
        x = x.T
    x = x / (math.sqrt(float((x * x).sum())) + eps)
    eye = np.eye(x.shape[0])

    def times(p, q):
        r = p @ q
        return r if wobble is None else r + wobble(p, q)

    for a, b, c in coef:
        gram = times(x, x.T)
        x = times(a * eye + b * gram + c * times(gram, gram), x)
    return x.T if turned else x


def orth_tolerance(g: np.ndarray, coef, eps: float, seed: int = 0) -> float:
    """Relative error (2-norm) that the split products may leave.

    A product of two values kept in 22 bits and without its lo lo term is off
    by at most 3 * 2^-22 of its magnitude, and a 32-bit sum of k of them by some
    sqrt(k) roundings (2^-23 each, the tensor core's adder may truncate).
    How the steps amplify that depends on the singular values, so it is taken
    from the iteration itself: the 64-bit iteration with every element of
    every product moved at random within that bound, the worst of three,
    times four.  The bound is on the sum of magnitudes, the true errors
    largely cancel: a correct kernel is well inside."""
    rng = np.random.default_rng(seed)
    want = newton_schulz(g, coef, eps)
    norm = np.linalg.norm(want)
    if not norm:
        return 0.0

    def wobble(p, q):
        size = (3 * 2.0 ** -22 + math.sqrt(p.shape[1]) * 2.0 ** -23) * (np.abs(p) @ np.abs(q))
        return rng.uniform(-1, 1, size.shape) * size
    return 4 * max(np.linalg.norm(newton_schulz(g, coef, eps, wobble) - want) / norm for _ in range(3))


def orth_quantum(g: np.ndarray, coef, eps: float, seed: int = 0) -> float:
    """Error (2-norm) that the planes' smallest step may leave.

    X, A and B are kept at powers of two that bring a bound on their singular values
    to 2^13; a plane's smallest step is 2^-24 there, so every element is off by up to
    half of that, 2^(e - 38) with the bound below 2^e, however small it is.  The bounds start
    from norm / (norm + eps) where that is below a half, else from 1, and follow
    the step's polynomial.  Its effect is taken as in orth_tolerance: the iteration with every
    element moved at random within that, the worst of three, times four."""
    rng = np.random.default_rng(seed)
    x0 = g.astype(np.float64)
    x0 = x0.T if x0.shape[0] > x0.shape[1] else x0
    norm = math.sqrt(float((x0 * x0).sum()))
    share = norm / (norm + eps) if norm else 1.0
    eye, want = np.eye(x0.shape[0]), newton_schulz(x0, coef, eps)

    def moved(v, bound):
        return v + rng.uniform(-1, 1, v.shape) * 2.0 ** (math.frexp(max(bound, 2.0 ** -120))[1] - 38)

    def run():
        x, s = x0 / (norm + eps), share if share < 0.5 else 1.0
        for a, b, c in coef:
            t = np.linspace(0, s, 10001) ** 2
            x = moved(x, s)
            gram = moved(x @ x.T, s * s)
            x = moved(a * eye + b * gram + c * gram @ gram, float(np.abs(a + t * (b + t * c)).max())) @ x
            s = float((np.sqrt(t) * np.abs(a + t * (b + t * c))).max())
        return x
    return 4 * max(np.linalg.norm(run() - want) for _ in range(3)) if norm else 0.0


def whole_values(shape, seed: int) -> np.ndarray:
    """1 .. 7 at random: exact in every type, and any sum of them below 2^24 is exact in
    f32 whatever its order, so that a sum that lacks, repeats or misplaces one element differs."""
    return np.random.default_rng(seed).integers(1, 8, shape).astype(np.float64)
