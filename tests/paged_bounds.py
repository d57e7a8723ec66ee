"""Bounds of the attention over a paged cache, column by column: what a row without weight holds, or a row
that a query does not see, excuses nothing in the columns of the others."""
import math

import numpy as np

# half a step of the type, relative to the value
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}


def column_bounds(case, q, q_seq, group, causal, new_rows=None):
    """Largest |error| of every value of A.  With p the probabilities, v a column of the values seen:

      half a step of the type for every probability, and for the sum:  u (sum p |v| + |A|)
      fp32 products and sums of `count` keys:                           eps (count + 16) sum p |v|
      a score's error ds moves its p by the factor 1 + ds, and the sum: 2 ds sum p |v|

    and what lies below the types' normal numbers: 2^-25 of an fp16 result.  Probabilities of unpacked fp16 pages
    are fp16 numbers that carry 2^7 at least, the largest of a row being 1: half of their smallest step is
    2^-32 of it, whatever the row's value.  Others have the exponents of fp32: below 2^-118 they may be 0."""
    n_batch, heads, head = case.n_batch, case.heads, case.head
    q = q.float().numpy().astype(np.float64).reshape(heads, group, n_batch, q_seq, head)
    bound = np.zeros(q.shape)
    u, eps = HALF_STEP[case.dtype], 2.0 ** -24
    lost = 2.0 ** -32 if case.dtype == "fp16" and not case.packed else 2.0 ** -118
    for n in range(n_batch):
        k, ok = case.rows(n, 0)
        v, _ = case.rows(n, 1)
        length = k.shape[1]
        given = q_seq if new_rows is None else max(0, min(q_seq, new_rows[n]))
        for j in range(given):
            seen = ok.copy()
            if causal:
                seen &= np.arange(length) <= length - given + j
            if not seen.any():
                continue
            count = int(seen.sum())
            for h in range(heads):
                kk, vv, qq = k[h][seen], v[h][seen], q[h, :, n, j]
                s = qq @ kk.T / math.sqrt(head)
                w = np.exp(s - s.max(axis=1, keepdims=True))
                p = w / w.sum(axis=1, keepdims=True)
                ds = (eps * (head + 8) * (np.abs(qq) @ np.abs(kk).T) / math.sqrt(head)
                      + 8 * eps * (1 + np.abs(s))).max(axis=1, keepdims=True)
                pv = p @ np.abs(vv)
                bound[h, :, n, j] = (u + 2 * ds + eps * (count + 16)) * pv + u * np.abs(p @ vv) \
                    + lost * p.max(axis=1, keepdims=True) * np.abs(vv).sum(axis=0)[None, :] \
                    + (2.0 ** -25 if case.dtype == "fp16" else 2.0 ** -133)
    return bound.reshape(-1, q_seq, head)
