"""Masked, shaped attention over a paged cache in float64 numpy (oracle; test infrastructure only), from the definition."""

from __future__ import annotations

import numpy as np


def visible(length, queries, prefix=0, starts=None, window=None):
    """[Q, length] bool and [Q, length] distances: query i sits at length - Q + i."""
    j = np.arange(length)[None, :]
    p = (length - queries + np.arange(queries))[:, None]
    near = j <= p
    if window is not None:
        near &= p - j < window
    if starts is not None:
        near &= j >= np.asarray(starts)[:, None]
    return near | (j < prefix), np.abs(p - j)


def attend(q, k, v, table, lens, scale, softcap=None, slopes=None, window=None, prefix=None, starts=None):
    """q [B, Q, Hq, D]; k, v float64 pools [NB, P, Hkv, D]; table [B, blocks]. Returns (out, lse, spread, slack): spread is the
    weighted mean of |v|, slack [B, Q, Hq] what float32 may do to a score (see the tests' tolerances)."""
    q = np.asarray(q, dtype=np.float64)
    b, n, hq, d = q.shape
    page, hkv = k.shape[1:3]
    g = hq // hkv
    out, lse = np.zeros(q.shape), np.full((b, n, hq), -np.inf)
    spread, slack = np.zeros(q.shape), np.zeros((b, n, hq))
    for i in range(b):
        length = int(lens[i])
        if length == 0:
            continue
        pages = np.asarray(table[i][: -(-length // page)])
        seen, far = visible(length, n, 0 if prefix is None else int(prefix[i]), None if starts is None else starts[i], window)
        for h in range(hq):
            kk = k[pages, :, h // g].reshape(-1, d)[:length]
            vv = v[pages, :, h // g].reshape(-1, d)[:length]
            for r in range(n):
                s = seen[r]
                if not s.any():
                    continue
                with np.errstate(invalid="ignore", over="ignore"):
                    t = kk[s] @ q[i, r, h] * scale
                    size = np.abs(kk[s]) @ np.abs(q[i, r, h]) * abs(scale)
                    t0 = np.abs(t).max()
                    bias = 0.0
                    if softcap is not None:
                        t = softcap * np.tanh(t / softcap)
                    if slopes is not None:
                        bias = float(slopes[h]) * far[r][s]
                        t = t - bias
                    m = t.max()
                    w = np.exp(t - m)
                    out[i, r, h] = w @ vv[s] / w.sum()
                    spread[i, r, h] = w @ np.abs(vv[s]) / w.sum()
                    lse[i, r, h] = m + np.log(w.sum())
                    # Products and sums of 128 terms, the cap's cancellation, the bias's two roundings, the exponent's.
                    slack[i, r, h] = (130 * 2.0**-24 * size.max() + (0 if softcap is None else min(softcap, 256) * 2.0**-21)
                                      + (t0 + np.abs(bias).max() + np.abs(t).max()) * 2.0**-22)
    return out, lse, spread, slack
