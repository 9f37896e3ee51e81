"""Rotary positions in float64 numpy (oracle; test infrastructure only), from the definition."""

from __future__ import annotations

import numpy as np


def rotate(x, positions, inv_freq, axis_of_pair=None, interleaved=False, scaling=1.0, weight=None, eps=1e-6):
    """x [B, Q, H, D] -> float64 [B, Q, H, D]; positions [axes, B, Q]; pair i turns by positions[axis_of_pair[i]] *
    inv_freq[i]: (a, b) -> scaling (a cos t - b sin t, a sin t + b cos t)."""
    x = np.asarray(x, dtype=np.float64)
    if weight is not None:
        x = x / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + np.float64(np.float32(eps))) * np.asarray(weight, dtype=np.float64)
    out = x.copy()
    half = len(inv_freq)
    for i in range(half):
        first, second = (2 * i, 2 * i + 1) if interleaved else (i, half + i)
        axis = 0 if axis_of_pair is None else axis_of_pair[i]
        # Angles of far positions keep their fraction of a turn: extended precision, reduced before the sine.
        t = np.asarray(positions[axis], dtype=np.longdouble) * np.longdouble(inv_freq[i])
        c, s = np.cos(t).astype(np.float64)[..., None], np.sin(t).astype(np.float64)[..., None]
        a, b = x[..., first], x[..., second]
        out[..., first] = np.float64(np.float32(scaling)) * (a * c - b * s)
        out[..., second] = np.float64(np.float32(scaling)) * (a * s + b * c)
    return out


def spread(x, inv_freq, interleaved=False, scaling=1.0, weight=None, eps=1e-6):
    """For each channel of x the sum of its pair's magnitudes after the norm (and its own, where it is not rotated): what
    the rotation's roundings are relative to."""
    x = np.asarray(x, dtype=np.float64)
    if weight is not None:
        x = x / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + np.float64(np.float32(eps))) * np.asarray(weight, dtype=np.float64)
    out = np.abs(x)
    half = len(inv_freq)
    for i in range(half):
        first, second = (2 * i, 2 * i + 1) if interleaved else (i, half + i)
        out[..., first] = out[..., second] = abs(scaling) * (np.abs(x[..., first]) + np.abs(x[..., second]))
    return out
