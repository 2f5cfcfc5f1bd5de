"""Log probabilities of tokens, entropy and top alternatives in 64 bits from
the definition, and how far an fp32 result may be off.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py): the checker for
npl_token_logprobs.
"""
from __future__ import annotations

import numpy as np


def token_logprobs(logits, ids, top_k):
    """logits [n, V] (any float type), ids [n]. Returns (logprobs, entropy,
    top_ids, top_logprobs, tol): tol [n] bounds the absolute error of the three
    computed results (the entropy's in units of its own bound, see below).

    With d = max - x >= 0 (exact in fp32 up to half a step), an fp32 kernel has
    e^-d to a factor of 1 + (d + 4) 2^-23 (the argument's two roundings and 2
    ulp for the exponential), and each of the two sums to V' 2^-24 of its
    terms, where V' <= V / 256 + 64 bounds the additions that a term passes
    through: sums of a thread's words, of threads, of CTAs. Weighted with p the exponentials' factor
    is at most (E[d] + 4) 2^-23. ln S is off by the sum's relative error and an
    ulp of itself; ln p by that and half an ulp of d and of the result; the
    entropy ln S + E[d] by ln S's error and E[d] times the errors of both sums
    and of the terms, (E[d^2] + 6 E[d]) 2^-23 among them.
    """
    x = np.asarray(logits, np.float64)
    n, v = x.shape
    ids = np.asarray(ids)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = x.max(1, keepdims=True)
        d = m - x
        e = np.exp(-d)
        s = e.sum(1, keepdims=True)
        ls = np.log(s)
        p = e / s
        dz = np.where(np.isinf(d) & (x == -np.inf) & np.isfinite(m), 0.0, d)
        mean_d = (p * dz).sum(1)
        mean_d2 = (p * dz * dz).sum(1)
        entropy = ls[:, 0] + mean_d
        lp = -d - ls
        bad = ~np.isfinite(m[:, 0]) | np.isnan(x).any(1)
        lp[bad], entropy[bad] = np.nan, np.nan
        safe = np.clip(ids, 0, v - 1)
        got = lp[np.arange(n), safe]
        got = np.where(ids == -1, 0.0, np.where((ids < 0) | (ids >= v), np.nan, got))
        # stable descending order of the values; NaN first
        key = np.where(np.isnan(x), np.inf, x)
        tie = np.isnan(x)
        order = np.lexsort((np.broadcast_to(np.arange(v), x.shape), -key, ~tie), axis=1)[:, :top_k]
        top_lp = np.take_along_axis(lp, order, 1)
        depth = v / 256 + 64
        rel = (mean_d + 4) * 2.0 ** -23 + depth * 2.0 ** -24
        tol_ls = rel + np.abs(ls[:, 0]) * 2.0 ** -23 + 2.0 ** -23
        ent_tol = tol_ls + (mean_d2 + 6 * mean_d) * 2.0 ** -23 + mean_d * (rel + depth * 2.0 ** -24) + \
            np.abs(entropy) * 2.0 ** -23
    return got, entropy, order, top_lp, tol_ls, ent_tol


def value_tol(tol_ls, d_and_value):
    """Tolerance of a log probability whose magnitude is ``d_and_value``."""
    return tol_ls + np.where(np.isfinite(d_and_value), np.abs(d_and_value), 0.0) * 2 * 2.0 ** -23
