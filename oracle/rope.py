"""CPU oracle for per-head RMSNorm and rotary position embedding (test infrastructure only).

For a head x of D elements at position p, with row p of the ``[positions, R]`` cos/sin table
holding R/2 cosines c and R/2 sines s:

    y = x / sqrt(mean(x^2) + eps) * w                     (only with a weight)
    (y_i, y_j) -> (y_i c_n - y_j s_n, y_j c_n + y_i s_n),  n < R/2

with ``(i, j) = (n, n + R/2)``, or ``(2n, 2n + 1)`` when interleaved; elements R..D pass.
Everything is evaluated in float64.
"""
from __future__ import annotations

import numpy as np


def norm_rope(x, weight, positions, cos_sin, eps: float, interleaved: bool):
    """``x [T, H, D]`` -> (values [T, H, D], size [T, H, D]): size is |y_i c| + |y_j s|, what a
    rotated element's rounding errors are relative to."""
    y = np.asarray(x, np.float64)
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    out, size = y.copy(), np.abs(y)
    half = cos_sin.shape[1] // 2
    rows = np.asarray(cos_sin, np.float64)[np.asarray(positions, np.int64)]
    for n in range(half):
        i, j = (2 * n, 2 * n + 1) if interleaved else (n, n + half)
        c, s = rows[:, n, None], rows[:, half + n, None]
        out[..., i] = y[..., i] * c - y[..., j] * s
        out[..., j] = y[..., j] * c + y[..., i] * s
        size[..., i] = np.abs(y[..., i] * c) + np.abs(y[..., j] * s)
        size[..., j] = np.abs(y[..., j] * c) + np.abs(y[..., i] * s)
    return out, size
