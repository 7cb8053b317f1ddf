"""What sample_tokens must give, row by row in 64 bits on the host."""

from __future__ import annotations

import numpy as np


def sample_row(x, u, temp, top_k, top_p, min_p):
    """(token, probability) of one row of logits (float64 array; the settings as 32 bits hold them)."""
    x = np.where(np.isnan(x), -np.inf, x)
    if not temp > 0:
        return int(np.argmax(x)), 1.0
    order = np.argsort(-x, kind="stable")
    ranked = x[order]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(ranked == ranked[0], 1.0, np.exp((ranked - ranked[0]) / np.float64(temp)))
    w = np.nan_to_num(w, nan=0.0)
    n = len(w) if top_k <= 0 else min(top_k, len(w))
    mass = np.cumsum(w[:n].astype(np.longdouble))
    before = mass - w[:n]
    if top_p < 1:
        n = min(n, max(1, int(np.searchsorted(before, max(top_p, 0.0) * mass[-1], side="right"))))
    if min_p > 0:
        n = min(n, max(1, int((w >= min_p).sum())))
    kept = mass[n - 1]
    u = min(max(u, 0.0), 1.0 - 2.0 ** -24) if u == u else 0.0
    at = min(n - 1, int(np.searchsorted(mass[:n], u * kept, side="right")))
    return int(order[at]), float(w[at] / kept)


def sample_rows(logits, uniforms, temp, top_k, top_p, min_p):
    """Tokens and probabilities of (rows, vocab) logits; settings are numbers or arrays of rows."""
    rows = logits.shape[0]
    x = logits.double().cpu().numpy()
    u = uniforms.double().cpu().numpy()

    def each(p, kind=np.float32):
        p = p.cpu().numpy() if hasattr(p, "cpu") else np.full(rows, p, dtype=kind)
        return p.astype(np.float64) if kind == np.float32 else p

    settings = list(zip(u, each(temp), each(top_k, np.int32), each(top_p), each(min_p)))
    got = [sample_row(x[r], *settings[r]) for r in range(rows)]
    return np.array([g[0] for g in got]), np.array([g[1] for g in got])
