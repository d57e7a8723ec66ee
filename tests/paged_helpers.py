"""A paged cache in numpy, in 64 bits, and the tolerances of what is compared with it."""
import math

import numpy as np
import torch

TORCH_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


class Case:
    """Pools, table and lengths of random sequences; every page that no sequence has, every
    row behind a sequence's last and every spare byte of a pool holds `junk`."""

    def __init__(self, seed, dtype, packed, n_batch, heads, head, page_rows, lens, max_pages=None,
                 spread=0, junk=float("nan"), scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.packed, self.head, self.heads = dtype, packed, head, heads
        self.page_rows, self.n_batch = page_rows, n_batch
        self.lens = list(lens)
        pages_of = [-(-max(0, l) // page_rows) for l in lens]
        self.max_pages = max(1, max(pages_of)) if max_pages is None else max_pages
        self.n_pages = max(1, sum(pages_of)) + 3
        order = torch.randperm(self.n_pages, generator=g).tolist()
        self.table = torch.full((n_batch, self.max_pages), -1, dtype=torch.int32)
        used = 0
        for n, count in enumerate(pages_of):
            count = min(count, self.max_pages)
            self.table[n, :count] = torch.tensor(order[used:used + count], dtype=torch.int32)
            used += count
        held = torch.float8_e4m3fn if packed else TORCH_DT[dtype]
        shape = (self.n_pages, 2, heads, page_rows, head)
        if packed:
            pool = (scale * torch.randn(shape, generator=g)).clamp(-400, 400).to(held)
        else:
            pool = (scale * torch.randn(shape, generator=g)).to(held)
        scales = torch.randint(119, 131, shape[:4], generator=g).to(torch.uint8)
        there = torch.zeros(self.n_pages, page_rows, dtype=torch.bool)
        for n in range(n_batch):
            for p in range(pages_of[n]):
                there[self.table[n, p], :max(0, min(page_rows, lens[n] - p * page_rows))] = True
        self.there = there
        pool = pool.float()
        pool[~there[:, None, None].expand(shape[:4])] = junk
        self.pool, self.scales = pool.to(held), scales
        self.spread = spread

    def device(self):
        """K and V as the two halves of one pool (strided pages) where spread, else apart."""
        pool, scales = self.pool.cuda(), self.scales.cuda()
        self.dpool, self.dscales = pool, scales
        if self.spread:
            k, v = pool[:, 0], pool[:, 1]
            ks, vs = scales[:, 0], scales[:, 1]
        else:
            k, v = pool[:, 0].contiguous(), pool[:, 1].contiguous()
            ks, vs = scales[:, 0].contiguous(), scales[:, 1].contiguous()
        self.k, self.v = k, v
        self.ks, self.vs = (ks, vs) if self.packed else (None, None)
        self.dtable = self.table.cuda()
        self.dlens = torch.tensor(self.lens, dtype=torch.int32).cuda()
        return self

    def values(self, which, pool=None, scales=None):
        """The pool's values in 64 bits: [n_pages, heads, page_rows, head]."""
        x = (self.pool if pool is None else pool)[:, which].float().numpy().astype(np.float64)
        if self.packed:
            s = (self.scales if scales is None else scales)[:, which].numpy().astype(np.float64)
            x = x * np.exp2(s - 127.0)[..., None]
        return x

    def rows(self, n, which, count=None):
        """Rows of sequence n: [heads, rows, head] in 64 bits; and which of them have a page."""
        count = max(0, min(self.lens[n], self.max_pages * self.page_rows)) if count is None else count
        x = self.values(which)
        out = np.zeros((self.heads, count, self.head))
        ok = np.zeros(count, bool)
        for r in range(count):
            page = int(self.table[n, r // self.page_rows])
            if 0 <= page < self.n_pages:
                out[:, r] = x[page, :, r % self.page_rows]
                ok[r] = True
        return out, ok


def attend(case, q, q_seq, group, causal, new_rows=None):
    """A, lse in 64 bits of q [entries * group, q_seq, head] (a CPU tensor)."""
    n_batch, heads, head = case.n_batch, case.heads, case.head
    q = q.float().numpy().astype(np.float64).reshape(heads, group, n_batch, q_seq, head)
    A = np.zeros(q.shape)
    lse = np.full(q.shape[:4], -np.inf)
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
            for h in range(heads):
                with np.errstate(invalid="ignore", over="ignore"):
                    s = q[h, :, n, j] @ k[h][seen].T / math.sqrt(head)
                    top = s.max(axis=1, keepdims=True)
                    w = np.exp(s - top)
                    total = w.sum(axis=1, keepdims=True)
                    lse[h, :, n, j] = (np.log(total) + top)[:, 0]
                    A[h, :, n, j] = (w / total) @ v[h][seen]
    return A.reshape(-1, q_seq, head), lse.reshape(-1, q_seq)


def attend_bounds(case, q, q_seq, group, causal, new_rows=None):
    """Largest |error| of every value of A and of lse.

    With p the probabilities: products and sums in fp32 of n keys and `head` products err by
    at most a few roundings each; what dominates in 16 bit is the rounding of every
    probability (half a step u of its type, relative) and of the output (half a step):
    |dA| <= u sum p |v| + u |A|, at p near the type's smallest normal numbers an absolute 2^-25
    of the largest term beside it.  The score errs by eps32 * (head + 4) * sum |q||k| / sqrt(head),
    which moves p, and so A by twice that times sum p |v|, and lse by once that."""
    n_batch, heads, head = case.n_batch, case.heads, case.head
    q = q.float().numpy().astype(np.float64).reshape(heads, group, n_batch, q_seq, head)
    bound_a, bound_l = np.zeros(q.shape), np.zeros(q.shape[:4])
    u = {"bf16": 2.0 ** -9, "fp16": 2.0 ** -12, "fp32": 2.0 ** -24}[case.dtype] * 2     # relative to the value
    # (a probability is rounded to the tile type whatever the pages hold, in bf16 times the power
    # of two of its value row, which moves no bit of it: half a step, u, again)
    up = u
    eps = 2.0 ** -24
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
            for h in range(heads):
                kk, vv, qq = k[h][seen], v[h][seen], q[h, :, n, j]
                s = qq @ kk.T / math.sqrt(head)
                w = np.exp(s - s.max(axis=1, keepdims=True))
                p = w / w.sum(axis=1, keepdims=True)
                ds = (eps * (head + 8) * (np.abs(qq) @ np.abs(kk).T) / math.sqrt(head)
                      + 8 * eps * (1 + np.abs(s))).max(axis=1, keepdims=True)
                pv = p @ np.abs(vv)
                count = seen.sum()
                small = 0.0 if case.dtype != "fp16" and not case.packed else 2.0 ** -25 * count
                a = np.abs(p @ vv)
                bound_a[h, :, n, j] = (up + 2 * ds + eps * (count + 16)) * pv + u * a \
                    + small * p.max(axis=1, keepdims=True) * np.abs(vv).max(axis=0)[None, :] + 2.0 ** -25
                bound_l[h, :, n, j] = (ds + eps * (count + 16) + 4 * eps * (1 + np.abs(s).max(axis=1, keepdims=True)))[:, 0]
    return bound_a.reshape(-1, q_seq, head), bound_l.reshape(-1, q_seq)


def quantised(x):
    """The definition of an 8-bit row, for x [.., head] in 64 bits: (values, bytes)."""
    a = np.abs(x).max(axis=-1)
    bad = ~np.isfinite(a)
    k = np.full(a.shape, -126, np.int64)
    ok = ~bad & (a > 0)
    m, e = np.frexp(a[ok])
    k[ok] = np.maximum(np.where(m > 0.875, e - 8, e - 9), -126)
    k[bad] = 0
    with np.errstate(invalid="ignore"):
        y = x * np.exp2(-k.astype(np.float64))[..., None]
        # e4m3: three bits behind the point from 2^-6 on, steps of 2^-9 below
        step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -60))), -6) - 3)
        code = np.rint(y / step) * step
    code[bad] = np.nan
    return code * np.exp2(k.astype(np.float64))[..., None], (k + 127).astype(np.uint8)
