"""Attention over a paged cache within bounds that every column has for itself: each form, equal lengths of more
(sequence, head) pairs than workgroups, pages behind 2^32 elements."""
import pytest
import torch

from nntile_amd import hip_sdpa as h
from . import paged_helpers as P
from .test_gpu_paged_attention import KINDS, _queries, _run
from .test_gpu_paged_value_ranges import _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,packed", KINDS)
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("q_seq,group,causal", [(1, 4, True), (4, 8, True), (4, 8, False), (16, 4, True), (43, 3, True)])
def test_every_form(dtype, packed, head, q_seq, group, causal):
    c = P.Case(90, dtype, packed, 3, 2, head, 16, [700, 64, 333], spread=1)
    _check(c, _queries(91, c, q_seq, group), q_seq, group, causal)


@pytest.mark.parametrize("dtype,packed", KINDS)
@pytest.mark.parametrize("n_batch,heads", [(60, 10), (70, 8)])
@pytest.mark.parametrize("q_seq,group", [(1, 2), (4, 8)])
def test_more_equal_units_than_workgroups(dtype, packed, n_batch, heads, q_seq, group):
    """Every sequence has as many blocks, and there are more units than places: even runs of blocks, none of which
    counts a unit's begin."""
    assert n_batch * heads > 512
    length = 600 if packed else 300
    c = P.Case(92, dtype, packed, n_batch, heads, 64, 64, [length] * n_batch)
    values = [c.values(which) for which in range(2)]
    c.values = lambda which: values[which]          # (once, not for every sequence)
    _check(c, _queries(93, c, q_seq, group), q_seq, group)


@pytest.mark.parametrize("dtype,packed", KINDS)
def test_pages_behind_32_bits(dtype, packed):
    """Pools of more than 2^32 elements: pages at their end give the bits that they give in a small pool."""
    page_rows, head, heads, group, q_seq = 1024, 128, 8, 2, 3
    c = P.Case(94, dtype, packed, 2, heads, head, page_rows, [1500, 333]).device()
    q = _queries(95, c, q_seq, group)
    want, want_l = _run(c, q, group)
    n_pages = 2 ** 32 // (page_rows * head * heads) + 5
    print("large pool", dtype, packed, n_pages, flush=True)
    places = torch.tensor([n_pages - 1, n_pages // 2 + 1, n_pages - 2, 0, n_pages - 3, 7], device="cuda")
    table = torch.full((2, 2), -1, dtype=torch.int32, device="cuda")

    def spread(x):
        if x is None:
            return None
        y = torch.empty((n_pages,) + tuple(x.shape[1:]), dtype=x.dtype, device="cuda")
        at = 0
        for n in range(2):
            for p in range(2):
                page = int(c.table[n, p])
                if page >= 0:
                    # (as bytes: e4m3 tensors have no copy by index)
                    y[int(places[at])].view(torch.uint8).copy_(x[page].contiguous().view(torch.uint8))
                    table[n, p] = places[at]
                    at += 1
        return y

    k, v, ks, vs = (spread(x) for x in (c.k, c.v, c.ks, c.vs))
    qd = q.cuda()
    lse = torch.full(q.shape[:2], float("nan"), device="cuda")
    A = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    ws = torch.zeros(h.paged_workspace_bytes(qd, 2, group), dtype=torch.uint8, device="cuda")
    h.sdpa_fwd_paged(k, v, table, c.dlens, qd, lse, A, h.MASK_CAUSAL, group, ws, k_scales=ks, v_scales=vs, flags=h.OVERWRITE)
    torch.cuda.synchronize()
    assert torch.equal(A, want) and torch.equal(lse, want_l)
