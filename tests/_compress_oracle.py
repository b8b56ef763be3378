"""Plain 64-bit implementations of the cache-compression operators, for the
tests: the 4-bit page format, attention over stored values, accumulated key
weights and eviction.  Written from the operators' definitions on numpy arrays;
nothing of the package under test is used.  Test infrastructure only."""
from __future__ import annotations

import numpy as np

GRID = np.array([(m / 8) * 2.0 ** -14 if e == 0 else (1 + m / 8) * 2.0 ** (e - 15)
                 for e in range(29) for m in range(8)][:226])
SCALES = np.concatenate([GRID, np.full(30, np.nan)])  # every scale byte's value


def scale_bytes(top: np.ndarray) -> np.ndarray:
    """Scale byte of each group's largest magnitude (fp64, may be inf/nan)."""
    y = top / 7.0
    hi = np.clip(np.searchsorted(GRID, y), 1, len(GRID) - 1)
    lo = hi - 1
    up, down = GRID[hi] - y, y - GRID[lo]
    pick = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    pick = np.where(y >= GRID[-1], len(GRID) - 1, pick)
    return np.where(np.isfinite(top), pick, 255).astype(np.uint8)


def quantise(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(codes in -7..7 [..., D], scale bytes [..., D / 16]) of rows."""
    g = x.astype(np.float64).reshape(*x.shape[:-1], -1, 16)
    b = scale_bytes(np.abs(g).max(-1) if not np.isnan(g).any() else np.abs(np.where(np.isnan(g), np.inf, g)).max(-1))
    s = SCALES[b][..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(s > 0, np.rint(g / s), 0.0)
    c = np.clip(np.nan_to_num(c), -7, 7)
    return c.reshape(x.shape).astype(np.int8), b


def stored(x: np.ndarray) -> np.ndarray:
    """What rows read back as."""
    c, b = quantise(x)
    return (c.reshape(*x.shape[:-1], -1, 16) * SCALES[b][..., None]).reshape(x.shape)


def pack_pages(x: np.ndarray, values: bool) -> np.ndarray:
    """[n, H, bs, D] rows as uint8 pages [n, H, bs, D * 9 / 16]."""
    n, H, bs, D = x.shape
    c, b = quantise(x)
    u = (c.astype(np.int16) + 8).astype(np.uint8)
    codes = u[..., 0::2] | (u[..., 1::2] << 4)
    scales = b.transpose(0, 1, 3, 2) if values else b
    return np.concatenate([codes.reshape(n, H, -1), scales.reshape(n, H, -1)], -1).reshape(n, H, bs, D * 9 // 16)


def rows_of(pool: np.ndarray, ids, n: int) -> np.ndarray:
    """Rows 0..n-1 [n, H, D] of a sequence with block ids ``ids``."""
    bs = pool.shape[2]
    if n == 0:
        return np.zeros((0, pool.shape[1], pool.shape[3]))
    x = pool[np.asarray(ids[: -(-n // bs)])]
    return x.transpose(0, 2, 1, 3).reshape(-1, pool.shape[1], pool.shape[3])[:n]


def softmax_rows(q: np.ndarray, K: np.ndarray, cur: int, scale: float, hidden=()) -> tuple[np.ndarray, float]:
    """Weights [H, T, n] of queries q [H, T, D] over keys K [n, H, D], and the
    largest sum of |q_d k_d| scale over d (for error bounds)."""
    H, T, D = q.shape
    n = K.shape[0]
    z = np.einsum("htd,nhd->htn", q, K) * scale
    size = float(np.einsum("htd,nhd->htn", np.abs(q), np.abs(K)).max(initial=0.0) * scale)
    t = np.arange(T)[:, None]
    j = np.arange(n)[None]
    seen = j < np.minimum(n, n - cur + t + 1)
    for k in hidden:
        seen = seen & (j != k)
    z = np.where(seen, z, -np.inf)
    top = z.max(-1, initial=-np.inf, keepdims=True)
    p = np.where(seen, np.exp(z - np.where(np.isfinite(top), top, 0)), 0.0)
    s = p.sum(-1, keepdims=True)
    return p / np.where(s > 0, s, 1), size


def evict(w: np.ndarray, keep: int, recent: int) -> np.ndarray:
    """Kept positions (ascending) of one head with key weights w [n]."""
    n = len(w)
    k = min(keep, n)
    sure = min(recent, k)
    if n <= keep:
        return np.arange(n)
    order = sorted(range(n - sure), key=lambda j: (0 if np.isnan(w[j]) else 1, -w[j] if not np.isnan(w[j]) else 0, j))
    return np.array(sorted(order[: k - sure]) + list(range(n - sure, n)))


# ------------------------------------------------------------ error bounds
# Rounding errors, in units of the relative precision u = 2^-22 (two units of
# fp32's last place: a tensor-core accumulation truncates, and an operand
# split in two 11-bit halves keeps 22 bits):
#   logit: (D + 8) u S, S = the largest sum over d of |q_d k_d| scale (and log2 e
#          for the base change enters both sides alike);
#   weight exp(logit - max) and its normaliser: twice that, the hardware
#          exponential's 2^-22 and the sum's n 2^-23;
#   output: the weights' relative error times max|v|, for the sums of both
#          numerator and denominator, and half a step of the output type.
U = 2.0 ** -22


def weight_error(D: int, size: float, n: int) -> float:
    """Relative error of a softmax weight over n keys."""
    return 2 * (D + 8) * U * max(size, 1.0) + (n + 8) * U / 2 + 4 * U


def output_bound(ref: np.ndarray, half_step: float, D: int, size: float, n: int, vmax: float) -> np.ndarray:
    return half_step * np.abs(ref) + 2 * weight_error(D, size, n) * vmax + 2.0 ** -25
