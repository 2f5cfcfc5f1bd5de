"""Attention over the paged pool under a tree's mask or a sliding window with
sinks, in 64 bits from the definition, and how far a right result may be off.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py): the checker for
npl_paged_tree_attention and npl_paged_window_attention.
"""
from __future__ import annotations

import numpy as np

# half a step of the type, relative to the value
HALF_STEP = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def tree_seen(mask_rows, n, ctx):
    """bool [n, ctx]: what n drafts see of their sequence's ctx keys."""
    seen = np.ones((n, ctx), bool)
    seen[:, ctx - n:] = np.asarray(mask_rows)[:, :n] != 0
    return seen


def window_seen(n, ctx, window, sinks):
    pos = np.arange(ctx - n, ctx)[:, None]
    key = np.arange(ctx)[None]
    return (key <= pos) & ((key > pos - window) | (key < sinks))


def attention(q, k_cache, v_cache, block_tables, context_lens, q_lens, q_offsets, scale, groups, seen_of, dtype):
    """q [total_q, H, D], caches [num_blocks, block_size, Hkv, D] (any float
    type); seen_of(b) gives bool [q_len, ctx]. Returns (out, tol) float64
    [total_q, H, D]; rows of no sequence are NaN in both.

    tol bounds |result - out| of a kernel that sums in fp32, rounds the
    probabilities to ``dtype`` and the output once. With u half a step of the
    type, n visible keys, A = sum p |v| and out = sum p v:
      * each score: D fp32 accumulations of exact products, each off by at most
        2^-23 (truncation) of sum |q||k| * scale, and two fp32 steps of the
        score itself: e_s; p changes by the factor 1 + 2 e_s (numerator and sum)
        and 2^-21 for exp2 and the scaling of both;
      * p rounded to the type: u A; p below the type's normal numbers (fp16,
        p scaled so that the largest is 2^6 or more): 2^-31 |v| a key at most;
      * fp32 sums over keys, in any order: 2 n 2^-24 A;
      * the output's rounding: u |out|, and 2^-25 where fp16 is subnormal.
    """
    q, kc, vc = (np.asarray(a, np.float64) for a in (q, k_cache, v_cache))
    total, H, D = q.shape
    bs = kc.shape[1]
    u = HALF_STEP[dtype]
    out = np.full((total, H, D), np.nan)
    tol = np.full((total, H, D), np.nan)
    for b in range(len(q_lens)):
        n, ctx, off = int(q_lens[b]), int(context_lens[b]), int(q_offsets[b])
        if n <= 0:
            continue
        if ctx == 0:
            out[off:off + n] = tol[off:off + n] = 0.0
            continue
        seen = seen_of(b)
        any_row = seen.any(0)
        keys = np.arange(ctx)
        blk = np.where(any_row, np.asarray(block_tables[b])[np.minimum(keys // bs, len(block_tables[b]) - 1)], 0)
        k, v = kc[blk, keys % bs], vc[blk, keys % bs]  # [ctx, Hkv, D]
        k[~any_row], v[~any_row] = 0.0, 0.0
        for h in range(H):
            kh, vh, qh = k[:, h // groups], v[:, h // groups], q[off:off + n, h]
            with np.errstate(invalid="ignore", over="ignore"):
                s = np.where(seen, qh @ kh.T * scale, -np.inf)
                mx = s.max(1, keepdims=True, initial=-np.inf)
                p = np.where(seen, np.exp(s - np.where(np.isfinite(mx), mx, 0.0)), 0.0)
                l = p.sum(1, keepdims=True)
                p = p / np.where(l == 0, 1.0, l)
                clean = np.isfinite(vh).all(1)
                o = p[:, clean] @ vh[clean]
                for j in np.nonzero(~clean)[0]:  # such keys reach the rows that see them only
                    o = o + np.where(seen[:, j:j + 1], p[:, j:j + 1] * vh[j], 0.0)
                va = np.where(np.isfinite(vh), np.abs(vh), 0.0)
                A = p @ va
                prod = np.abs(qh) @ np.abs(np.where(np.isfinite(kh), kh, 0.0)).T * scale
                es = D * 2.0 ** -23 * np.where(seen, prod, 0).max(1, keepdims=True)
                es = es + 2 * 2.0 ** -23 * np.where(seen & np.isfinite(s), np.abs(s), 0).max(1, keepdims=True)
                cnt = seen.sum(1, keepdims=True)
                t = A * (2 * es + 2.0 ** -21 + u + 2 * cnt * 2.0 ** -24) + u * np.abs(o)
                if dtype == "float16":
                    t = t + cnt * 2.0 ** -31 * va.max(initial=0.0) + 2.0 ** -25
            out[off:off + n, h], tol[off:off + n, h] = o, t
    return out, tol
