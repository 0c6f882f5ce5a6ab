"""numpy (64-bit) restatement of the microscaled formats of ``metallora_b200.quant``.

Written from the definition, by arithmetic on the values (``frexp``, division,
``rint``); the kernels work on the bits of the exponents instead.
"""
from __future__ import annotations

import numpy as np

FP4_GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def _blocks(x: np.ndarray):
    x = np.asarray(x, np.float64)
    rows, k = x.shape
    pad = (-k) % 32
    v = np.pad(x, ((0, 0), (0, pad))).reshape(rows, -1, 32)
    amax = np.max(np.abs(v), axis=-1)          # NaN if the block holds one
    bad = ~np.isfinite(amax)
    safe = np.where(bad | (amax == 0), 1.0, amax)
    e = np.frexp(safe)[1] - 1                  # floor(log2)
    e = np.where(amax == 0, -1000, e)
    return np.where(bad[..., None], 0.0, v), e, bad, k


def mxfp4(x: np.ndarray):
    """(values [rows, K], scale bytes [rows, ceil(K/32)]) of MXFP4."""
    v, e, bad, k = _blocks(x)
    e = np.maximum(e - 2, -127)
    s = np.exp2(e.astype(np.float64))[..., None]
    u = np.abs(v / s)
    # nearest grid value, ties to the even code
    d = np.abs(u[..., None] - FP4_GRID)
    best = d.min(-1, keepdims=True)
    tied = d == best
    order = np.array([0, 2, 4, 6, 1, 3, 5, 7])  # even codes first
    code = order[np.argmax(tied[..., order], axis=-1)]
    out = np.copysign(FP4_GRID[code], v) * s
    out = np.where(bad[..., None], np.nan, out)
    return out.reshape(len(v), -1)[:, :k], np.where(bad, 255, e + 127).astype(np.uint8)


def mxint8(x: np.ndarray):
    """(values, codes [rows, K], scale bytes [rows, ceil(K/32)]) of MXINT8."""
    v, e, bad, k = _blocks(x)
    e = np.maximum(e, -127)
    s = np.exp2(e.astype(np.float64))[..., None]
    q = np.clip(np.rint(64.0 * (v / s)), -127, 127)
    out = np.where(bad[..., None], np.nan, q / 64.0 * s)
    rows = len(v)
    return (out.reshape(rows, -1)[:, :k], q.reshape(rows, -1)[:, :k].astype(np.int8),
            np.where(bad, 255, e + 127).astype(np.uint8))


def unpack_fp4(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """Values of packed codes [rows, K/2] (low nibble = even feature)."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(len(codes), -1)
    v = FP4_GRID[c & 7] * np.where(c & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return v * np.repeat(s, 32, axis=-1)[:, : v.shape[1]]
