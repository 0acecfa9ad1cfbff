"""Plain numpy statements of the block-scaled 8-bit format: the codes as their
definition has them (f32, each quotient and product rounded once), everything
else in 64 bits."""

from __future__ import annotations

import numpy as np

GROUP = 128
TINY = np.float32(448.0 * 2.0 ** -126)


def groups(n: int) -> int:
    return -(-n // GROUP)


def decode(codes: np.ndarray) -> np.ndarray:
    """E4M3FN bytes -> f64."""
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b >= 128, -v, v)[codes]


def encode(x: np.ndarray) -> np.ndarray:
    """f32 of magnitude 464 or less, or NaN -> E4M3FN bytes, nearest even."""
    a = np.abs(x.astype(np.float64))
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.clip(np.floor(np.log2(np.where(a > 0, a, 1.0))), -6, 8)
        e = np.where(a >= 2.0 ** (e + 1), e + 1, np.where((a < 2.0 ** e) & (e > -6), e - 1, e))
        n = np.rint(a / 2.0 ** (e - 3))  # in eighths of 2^e; half to even
    up = n == 16
    e, n = np.where(up, e + 1, e), np.where(up, 8, n)
    code = np.where(n < 8, n, (e + 7) * 8 + n - 8)
    code = np.where(np.isnan(x), 127, code).astype(np.uint8)
    return code | (np.signbit(x).astype(np.uint8) << 7)


def _scaled(amax: np.ndarray):
    amax = np.maximum(amax.astype(np.float32), TINY)
    return np.float32(448) / amax, amax / np.float32(448)


def quantize_rows(x: np.ndarray):
    """f32 [T, K] -> codes u8 [T, K], scales f32 [T, groups]."""
    T, K = x.shape
    v = np.zeros((T, groups(K) * GROUP), np.float32)
    v[:, :K] = x
    v = v.reshape(T, -1, GROUP)
    up, scales = _scaled(np.where(np.isfinite(v), np.abs(v), 0).max(-1))
    v = np.where(np.isinf(v), np.float32(np.nan), v)
    return encode(v * up[..., None]).reshape(T, -1)[:, :K].copy(), scales


def quantize_weight(w: np.ndarray):
    """f32 [N, K] -> codes u8 [N, K], scales f32 [groups(N), groups(K)]."""
    N, K = w.shape
    v = np.zeros((groups(N) * GROUP, groups(K) * GROUP), np.float32)
    v[:N, :K] = w
    v = v.reshape(groups(N), GROUP, groups(K), GROUP)
    up, scales = _scaled(np.where(np.isfinite(v), np.abs(v), 0).max((1, 3)))
    v = np.where(np.isinf(v), np.float32(np.nan), v)
    codes = encode(v * up[:, None, :, None]).reshape(groups(N) * GROUP, -1)
    return codes[:N, :K].copy(), scales


def row_values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    return decode(codes) * np.repeat(scales.astype(np.float64), GROUP, 1)[:, :codes.shape[1]]


def weight_values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    return row_values(codes, np.repeat(scales, GROUP, 0)[:codes.shape[0]])


def product(x, w):
    """x w^T in 64 bits and the sum of its terms' magnitudes, of (codes,
    scales) pairs."""
    a, b = row_values(*x), weight_values(*w)
    return a @ b.T, np.abs(a) @ np.abs(b).T


def gated(g: np.ndarray, u: np.ndarray, limit: float) -> np.ndarray:
    if limit > 0:
        g, u = np.minimum(g, limit), np.clip(u, -limit, limit)
    with np.errstate(over="ignore"):
        return g / (1 + np.exp(-g)) * u


def add_rms_norm(x, residual, weight, eps):
    """(y, h) in 64 bits of f32 arrays; h unrounded."""
    h = x.astype(np.float64) + (0 if residual is None else residual.astype(np.float64))
    y = h / np.sqrt(np.mean(h * h, -1, keepdims=True) + eps)
    return (y if weight is None else y * weight.astype(np.float64)), h
