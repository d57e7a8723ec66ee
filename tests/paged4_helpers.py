"""Pages of 4-bit codes in numpy, in 64 bits, and what eviction and received weights are by definition."""
import math

import numpy as np
import torch

from . import paged_helpers as P

CODES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
F4 = torch.float4_e2m1fn_x2


def quantised4(x):
    """The definition of 4-bit rows, for x [.., head] in 64 bits: (codes [.., head/2], bytes [.., head/32])."""
    b = x.reshape(x.shape[:-1] + (-1, 32))
    a = np.abs(b).max(axis=-1)
    bad = ~np.isfinite(a)
    k = np.full(a.shape, -125, np.int64)
    ok = ~bad & (a > 0)
    # the smallest k with a <= 7 * 2^k: 7 = 0.875 * 2^3; from -125 to 125
    m, e = np.frexp(a[ok])
    k[ok] = np.clip(np.where(m > 0.875, e - 2, e - 3), -125, 125)
    with np.errstate(invalid="ignore"):
        y = np.abs(b) * np.exp2(-k.astype(np.float64))[..., None]
        far = np.abs(y[..., None] - CODES)
    # the nearest code; of two equally near ones the even
    best = np.where(np.isnan(far), np.inf, far).min(axis=-1, keepdims=True)
    near = far == best
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(axis=-1), even.argmax(axis=-1), near.argmax(axis=-1))
    code = (code + 8 * np.signbit(b)).astype(np.uint8)
    code[bad] = 0
    code = code.reshape(x.shape[:-1] + (-1, 2))
    byte = np.where(bad, 255, k + 127).astype(np.uint8)
    return code[..., 0] + 16 * code[..., 1], byte


def values4(codes, scales):
    """What codes [.., head/2] and bytes [.., head/32] stand for, in 64 bits."""
    table = np.concatenate([CODES, -CODES])
    x = np.stack([table[codes & 15], table[codes >> 4]], axis=-1).reshape(codes.shape[:-1] + (-1, 32))
    s = scales.astype(np.float64)
    s = np.where(s == 255, np.nan, np.exp2(s - 127.0))
    return (x * s[..., None]).reshape(codes.shape[:-1] + (-1,))


class Case4(P.Case):
    """A P.Case in 4 bits: every page that no sequence has and every row behind a sequence's last holds NaN
    (bytes of 255 over codes of all kinds)."""

    def __init__(self, seed, dtype, n_batch, heads, head, page_rows, lens, max_pages=None, spread=0, scale=1.0):
        super().__init__(seed, dtype, True, n_batch, heads, head, page_rows, lens, max_pages, spread)
        g = torch.Generator().manual_seed(seed + 77)
        x = scale * torch.randn(self.n_pages, 2, heads, page_rows, head, generator=g, dtype=torch.float64)
        codes, scales = quantised4(x.numpy())
        gone = ~self.there.numpy()[:, None, None].repeat(2, 1).repeat(heads, 2)
        codes[gone] = torch.randint(0, 256, (int(gone.sum()), head // 2), generator=g).numpy()
        scales[gone] = 255
        self.pool, self.scales = torch.from_numpy(codes), torch.from_numpy(scales)

    def device(self):
        pool, scales = self.pool.cuda(), self.scales.cuda()
        self.dpool, self.dscales = pool, scales
        both = [t[:, i] if self.spread else t[:, i].contiguous() for t in (pool, scales) for i in (0, 1)]
        self.k, self.v, self.ks, self.vs = both
        self.k, self.v = self.k.view(F4), self.v.view(F4)
        self.dtable = self.table.cuda()
        self.dlens = torch.tensor(self.lens, dtype=torch.int32).cuda()
        return self

    def values(self, which, pool=None, scales=None):
        return values4((self.pool if pool is None else pool)[:, which].numpy(),
                       (self.scales if scales is None else scales)[:, which].numpy())


def free_first_page(case):
    """Page 0, which entries of the table that are no pages are read as, belongs to no sequence any more: it changes
    places with a page that belongs to none."""
    spare = next(p for p in range(case.n_pages) if not bool(case.there[p].any()))
    swap = torch.arange(case.n_pages)
    swap[0], swap[spare] = spare, 0
    case.pool, case.scales, case.there = case.pool[swap], case.scales[swap], case.there[swap]
    real = (case.table >= 0) & (case.table < case.n_pages)
    case.table = torch.where(real, swap[case.table.clamp(0, case.n_pages - 1).long()].to(torch.int32), case.table)


def in_the_rest(case, byte):
    """`byte` as the power of two of every row that no sequence has."""
    case.scales[~case.there[:, None, None].expand(case.scales.shape[:4])] = byte
    return case


def make(seed, dtype, bits, n_batch, heads, head, page_rows, lens, **kw):
    """A case whose pages hold `bits` bits (4, 8, or the tile type's)."""
    if bits == 4:
        return Case4(seed, dtype, n_batch, heads, head, page_rows, lens, **kw)
    return P.Case(seed, dtype, bits == 8, n_batch, heads, head, page_rows, lens, **kw)


KINDS = [("bf16", 16), ("fp16", 16), ("fp32", 32), ("bf16", 8), ("fp16", 8), ("bf16", 4), ("fp16", 4)]


def received(case, q, lse, q_seq, group, causal, new_rows=None):
    """What every row receives, [heads, n_batch, rows] by sequence (a list), and a bound of its error.

    A term exp(s - lse) errs by its exponent's error: that of the score, eps (head + 8) |q||k| / sqrt(head) for
    products and sums in fp32, a few roundings of s, lse and their logarithmic units; and the sum of `count` terms
    by eps (count + 8) of it."""
    n_batch, heads, head = case.n_batch, case.heads, case.head
    q = q.double().numpy().reshape(heads, group, n_batch, q_seq, head)
    lse = lse.double().numpy().reshape(heads, group, n_batch, q_seq)
    eps, out = 2.0 ** -24, []
    for n in range(n_batch):
        k, ok = case.rows(n, 0)
        length = k.shape[1]
        given = q_seq if new_rows is None else max(0, min(q_seq, new_rows[n]))
        total, bound = np.zeros((heads, length)), np.zeros((heads, length))
        for j in range(given):
            seen = ok.copy()
            if causal:
                seen &= np.arange(length) <= length - given + j
            for h in range(heads):
                for g in range(group):
                    if np.isneginf(lse[h, g, n, j]):
                        continue
                    with np.errstate(invalid="ignore", over="ignore"):
                        s = (k[h][seen] @ q[h, g, n, j]) / math.sqrt(head)
                        size = (np.abs(k[h][seen]) @ np.abs(q[h, g, n, j])) / math.sqrt(head)
                        p = np.exp(s - lse[h, g, n, j])
                        ds = eps * (head + 8) * size + 8 * eps * (2 + np.abs(s) + abs(lse[h, g, n, j]))
                    total[h, seen] += p
                    bound[h, seen] += 2 * ds * p + eps * (given * group + 16) * p
        out.append((total, bound + 2.0 ** -120))
    return out


def chosen(weights, length, keep, recent):
    """The rows that stay of a sequence of `length` rows with these weights [columns], in 64 bits."""
    if length <= keep:
        return np.arange(length)
    old = max(0, length - recent)
    w = np.where(np.isnan(weights[:old]), np.inf, weights[:old])
    order = np.lexsort((np.arange(old), ~np.isnan(weights[:old]), -w))
    return np.sort(np.concatenate([order[:keep - (length - old)], np.arange(old, length)])).astype(np.int64)
