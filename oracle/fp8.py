"""Block-scaled e4m3 in numpy, in 64 bits: what the kernels of
nanopointllm_b200.fp8 compute, from the definitions."""
from __future__ import annotations

import numpy as np

BLOCK = 128

# The finite e4m3 values from 0 up: 0, 7 subnormals of step 2^-9, then 8 steps
# a binade up to 448 (the code after it is NaN).
_POSITIVE = np.array([m * 2.0 ** -9 for m in range(8)] +
                     [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:-1])


def round_e4m3(x: np.ndarray) -> np.ndarray:
    """Nearest e4m3 values (ties to the even code), saturating; NaN stays."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(np.nan_to_num(x, nan=0.0)), 448.0)
    hi = np.clip(np.searchsorted(_POSITIVE, a), 0, len(_POSITIVE) - 1)
    lo = np.maximum(hi - 1, 0)
    up = _POSITIVE[hi] - a
    down = a - _POSITIVE[lo]
    pick = np.where(up < down, hi, np.where(down < up, lo, np.where(hi % 2 == 0, hi, lo)))
    out = np.copysign(_POSITIVE[pick], x)
    return np.where(np.isnan(x), np.nan, out)


def half_step_e4m3(x: np.ndarray) -> np.ndarray:
    """The most that rounding x to e4m3 may move it: half a step of its
    binade, half of the subnormals' step below 2^-6."""
    e = np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6)))
    return 2.0 ** (e - 4)


def block_scales(v: np.ndarray, block_rows: int) -> np.ndarray:
    """[R, K] -> scales [ceil(R / block_rows), ceil(K / 128)] in v's precision:
    max(max |v| / 448, 2^-126)."""
    r, k = v.shape
    rb, kb = -(-r // block_rows), -(-k // BLOCK)
    pad = np.zeros((rb * block_rows, kb * BLOCK), v.dtype)
    pad[:r, :k] = np.abs(v)
    a = pad.reshape(rb, block_rows, kb, BLOCK).max((1, 3))
    return np.maximum(a / v.dtype.type(448), v.dtype.type(2.0 ** -126))


def spread(scale: np.ndarray, block_rows: int, shape: tuple[int, int]) -> np.ndarray:
    """A block's scale for each of its elements."""
    return np.repeat(np.repeat(scale, block_rows, 0), BLOCK, 1)[:shape[0], :shape[1]]


def quant_fp32(v: np.ndarray, block_rows: int) -> tuple[np.ndarray, np.ndarray]:
    """The quantiser's own fp32 steps on fp32 values: (code values, scales)."""
    v = v.astype(np.float32)
    with np.errstate(all="ignore"):
        s = block_scales(v, block_rows)
        return round_e4m3(v * spread(np.float32(1) / s, block_rows, v.shape)), s


def rmsnorm(s: np.ndarray, w: np.ndarray, eps: float) -> np.ndarray:
    s, w = s.astype(np.float64), w.astype(np.float64)
    return s / np.sqrt((s * s).mean(-1, keepdims=True) + eps) * w


def silu_mul(g: np.ndarray, u: np.ndarray) -> np.ndarray:
    g = g.astype(np.float64)
    return g / (1.0 + np.exp(-g)) * u.astype(np.float64)


def linear(qa, sa, qw, sw, bias=None, residual=None):
    """(exact values [M, N], sum of the magnitudes of what is added up)."""
    a = qa.astype(np.float64) * spread(sa.astype(np.float64), 1, qa.shape)
    w = qw.astype(np.float64) * spread(sw.astype(np.float64), BLOCK, qw.shape)
    v, mag = a @ w.T, np.abs(a) @ np.abs(w).T
    for t in (bias, residual):
        if t is not None:
            v, mag = v + t.astype(np.float64), mag + np.abs(t.astype(np.float64))
    return v, mag
