"""Attention over a paged cache whose value rows differ much in size: no row costs another bits that it has no
weight against."""
import numpy as np
import pytest
import torch

from . import paged_helpers as P
from .paged_bounds import column_bounds
from .test_gpu_paged_attention import _queries, _run

pytestmark = pytest.mark.gpu
TYPES = ["bf16", "fp16"]


def _check(c, q, q_seq, group, causal=True, new_rows=None):
    print("ranges", c.dtype, c.packed, c.n_batch, c.heads, group, c.head, c.lens, q_seq, causal, flush=True)
    c.device()
    A, lse = _run(c, q, group, causal, new_rows)
    want, want_l = P.attend(c, q, q_seq, group, causal, new_rows)
    bound = column_bounds(c, q, q_seq, group, causal, new_rows)
    _, bound_l = P.attend_bounds(c, q, q_seq, group, causal, new_rows)
    dead = np.isneginf(want_l)
    off = np.abs(A.double().cpu().numpy() - want)
    print("worst: %.2f of the bound" % (off / bound)[~dead].max(), flush=True)
    assert np.all(off[~dead] <= bound[~dead])
    assert np.all(np.abs(lse.double().cpu().numpy()[~dead] - want_l[~dead]) <= bound_l[~dead])
    return A, lse


def _row(c, n, pos):
    """Page and place in it of a sequence's row."""
    return int(c.table[n, pos // c.page_rows]), pos % c.page_rows


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("q_seq,group", [(4, 3), (5, 6), (9, 4)])
def test_a_row_that_is_not_seen_costs_no_bits(dtype, head, q_seq, group):
    """The newest token's values are 2^26 times the others', and more: the tokens before it have the bits they
    have beside an ordinary row."""
    c = P.Case(60, dtype, True, 3, 2, head, 16, [300, 70, q_seq])
    c.scales[:, 1] = 109
    q = _queries(61, c, q_seq, group)
    results = []
    for byte in (109, 135, 254):
        for n, length in enumerate(c.lens):
            page, at = _row(c, n, length - 1)
            c.scales[page, 1, :, at] = byte
        if byte == 254:
            c.device()
            A, lse = _run(c, q, group)
        else:
            A, lse = _check(c, q, q_seq, group)
        results.append((A[:, :-1].clone(), lse.clone()))
    for A, lse in results[1:]:
        assert torch.equal(A, results[0][0]) and torch.equal(lse, results[0][1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("small", [102, 106, 110])
@pytest.mark.parametrize("score", [-25.0, -12.0, -3.0])
def test_a_large_row_of_little_weight(dtype, head, small, score):
    """One row near the largest fp16 value among 1000 small ones, with a weight of e^-25 to e^-3; half of the columns
    it has zeros in."""
    c = P.Case(62, dtype, True, 1, 1, head, 64, [1000])
    c.scales[:] = 127
    c.scales[:, 1] = small
    x = c.pool.float()
    x[:, 0] *= 0.125
    x[:, 1] = (100.0 * x[:, 1]).clamp(-400.0, 400.0)
    page, at = _row(c, 0, 613)
    x[page, 0, 0, at] = score / head ** 0.5
    x[page, 1, 0, at] = 200.0
    x[page, 1, 0, at, ::2] = 0.0
    c.pool = x.to(c.pool.dtype)
    c.scales[page, 1, 0, at] = 135
    g = torch.Generator().manual_seed(63)
    q = (1.0 + 0.03125 * torch.randn(8, 2, head, generator=g)).to(P.TORCH_DT[dtype])
    _check(c, q, 2, 8)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,q_seq,group", [([1500], 3, 2), ([400, 77, 19], 4, 8), ([700, 30], 16, 4)])
def test_rows_of_all_sizes(dtype, lens, q_seq, group):
    """Powers of two over the whole range of fp16 values; rows of some sizes have zeros in some columns, so that
    small rows decide there."""
    g = torch.Generator().manual_seed(64)
    c = P.Case(65, dtype, True, len(lens), 2, 64, 16, lens)
    c.scales[:, 1] = torch.randint(96, 133, c.scales[:, 1].shape, generator=g).to(torch.uint8)
    x = c.pool.float()
    size = c.scales[:, 1].int()[..., None]
    x[:, 1] = torch.where(size > 96 + torch.arange(64) * 37 // 64, 0.0, x[:, 1])
    x[~c.there[:, None, None].expand(x.shape[:4])] = float("nan")
    c.pool = x.to(c.pool.dtype)
    _check(c, _queries(66, c, q_seq, group), q_seq, group)


@pytest.mark.parametrize("dtype,packed", [("bf16", False), ("fp32", False), ("bf16", True)])
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("q_seq,group", [(1, 1), (2, 12), (5, 12)])
def test_large_values_behind_small_scores(dtype, packed, head, q_seq, group):
    """A few keys late in the sequence score a little more than those before them, less than makes the running
    maximum worth replacing, and have values of 2^124: their sum is a number of the type."""
    n_batch, heads, length = 8, 24, 1024
    c = P.Case(67, dtype, packed, n_batch, heads, head, 128, [length] * n_batch, spread=0)
    c.scales[:] = 127
    x = c.pool.float()
    x[:, 0] = 0.0
    for n in range(n_batch):
        for pos in (length - 301, length - 200, length - 99):
            page, at = _row(c, n, pos)
            # a score of 4.85, so a probability of 2^7 times the others'
            x[page, 0, :, at] = 4.85 / head ** 0.5
            big = 1.0 + 0.25 * (torch.arange(head) % 4)
            x[page, 1, :, at] = 64.0 * big if packed else 2.0 ** 124 * big
            c.scales[page, 1, :, at] = 127 + 118
    c.pool = x.to(c.pool.dtype)
    values = [c.values(which) for which in range(2)]
    c.values = lambda which: values[which]          # (once, not for every sequence)
    q = torch.ones(heads * group * n_batch, q_seq, head).to(P.TORCH_DT[dtype])
    A, _ = _check(c, q, q_seq, group)
    assert float(A.float().min()) > 2.0 ** 121
