"""Attention over a paged cache against the formula in 64 bits, value by value."""
import numpy as np
import pytest
import torch

from nntile_amd import hip_sdpa as h
from . import paged_helpers as P

pytestmark = pytest.mark.gpu
KINDS = [("bf16", False), ("fp16", False), ("fp32", False), ("bf16", True), ("fp16", True)]


def _queries(seed, c, q_seq, group, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    q = scale * torch.randn(c.heads * group * c.n_batch, q_seq, c.head, generator=g)
    return q.to(P.TORCH_DT[c.dtype])


def _run(c, q, group, causal=True, new_rows=None, flags=h.OVERWRITE, lse=None, A=None, ws=None):
    qd = q.cuda()
    if lse is None:
        lse = torch.full(q.shape[:2], float("nan"), device="cuda")
        A = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    nr = None if new_rows is None else torch.tensor(new_rows, dtype=torch.int32).cuda()
    if ws is None:
        # whatever lies in it must not matter
        ws = torch.full((h.paged_workspace_bytes(qd, c.n_batch, group),), 255, dtype=torch.uint8, device="cuda")
    h.sdpa_fwd_paged(c.k, c.v, c.dtable, c.dlens, qd, lse, A, h.MASK_CAUSAL if causal else h.MASK_NONE, group,
                     ws, k_scales=c.ks, v_scales=c.vs, new_rows=nr, flags=flags)
    torch.cuda.synchronize()
    return A, lse


def _check(c, q_seq, group, causal=True, new_rows=None, seed=21, qscale=1.0):
    print("attend", c.dtype, c.packed, c.n_batch, c.heads, group, c.head, c.page_rows, c.lens, q_seq, causal,
          new_rows, flush=True)
    c.device()
    q = _queries(seed, c, q_seq, group, qscale)
    A, lse = _run(c, q, group, causal, new_rows)
    want, want_l = P.attend(c, q, q_seq, group, causal, new_rows)
    bound, bound_l = P.attend_bounds(c, q, q_seq, group, causal, new_rows)
    A, lse = A.double().cpu().numpy(), lse.double().cpu().numpy()
    dead = np.isneginf(want_l)
    assert np.array_equal(np.isneginf(lse), dead)
    assert np.all(A[dead] == 0)
    with np.errstate(invalid="ignore"):
        off, off_l = np.abs(A - want), np.abs(lse - want_l)
    off_l[dead] = 0
    assert np.all(np.isfinite(off)) and np.all(np.isfinite(off_l))
    print("worst: A %.2f, lse %.2f of the bound" % ((off / np.maximum(bound, 1e-30))[~dead].max(initial=0),
                                                     (off_l / np.maximum(bound_l, 1e-30)).max(initial=0)), flush=True)
    assert np.all(off[~dead] <= bound[~dead]) and np.all(off_l[~dead] <= bound_l[~dead])


@pytest.mark.parametrize("dtype,packed", KINDS)
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("lens,q_seq,group,page_rows", [
    ([1], 1, 1, 16), ([17], 1, 4, 16), ([63, 64, 65], 1, 4, 32), ([300, 5, 0, 129], 2, 3, 16),
    ([257, 40], 5, 4, 64), ([700], 16, 4, 128), ([90, 33], 7, 8, 16), ([20, 130], 9, 1, 256)])
def test_small(dtype, packed, head, lens, q_seq, group, page_rows):
    _check(P.Case(20, dtype, packed, len(lens), 2, head, page_rows, lens, spread=q_seq % 2), q_seq, group)


@pytest.mark.parametrize("dtype,packed", KINDS)
@pytest.mark.parametrize("lens,q_seq,group", [([3000, 1, 500, 2047], 1, 4), ([1500], 3, 12), ([4000], 20, 4)])
def test_long(dtype, packed, lens, q_seq, group):
    _check(P.Case(22, dtype, packed, len(lens), 1, 128, 64, lens), q_seq, group)


@pytest.mark.parametrize("dtype,packed", KINDS)
def test_many_sequences(dtype, packed):
    """More sequences than threads of a workgroup, many of them empty."""
    lens = [(37 * i * i) % 90 if i % 3 else 0 for i in range(600)]
    _check(P.Case(23, dtype, packed, 600, 1, 64, 16, lens), 1, 2)


@pytest.mark.parametrize("dtype,packed", KINDS)
@pytest.mark.parametrize("causal", [True, False])
def test_padded_and_missing(dtype, packed, causal):
    """Sequences that bring fewer tokens, none, or more than they have rows; pages that are
    none; a length past the table and one below 0."""
    c = P.Case(24, dtype, packed, 7, 2, 64, 16, [70, 3, 200, 48, 64, 0, 33], max_pages=13)
    c.table[0, 1] = -1
    c.table[2, 3] = c.n_pages
    c.table[2, 12] = -2 ** 31
    c.table[6, :3] = -1
    c.lens[5] = -3
    _check(c, 6, 4, causal, [6, 6, 2, 0, 9, 6, 6])


@pytest.mark.parametrize("dtype,packed", KINDS)
def test_running_pair(dtype, packed):
    """Without OVERWRITE: merged into (lse, A); rows that see nothing keep theirs."""
    c = P.Case(25, dtype, packed, 3, 2, 128, 32, [90, 0, 700], spread=1).device()
    q = _queries(26, c, 3, 2)
    want, want_l = P.attend(c, q, 3, 2, True)
    bound, bound_l = P.attend_bounds(c, q, 3, 2, True)
    g = torch.Generator().manual_seed(27)
    A0 = torch.randn(q.shape, generator=g).to(q.dtype)
    lse0 = 4 + torch.randn(q.shape[:2], generator=g)
    lse0[0, 0] = float("-inf")
    A0[0, 0] = float("nan")         # not read
    A, lse = _run(c, q, 2, flags=0, lse=lse0.cuda().clone(), A=A0.cuda().clone())
    old, old_l = A0.double().numpy(), lse0.double().numpy()
    dead = np.isneginf(want_l)
    A, lse = A.double().cpu().numpy(), lse.double().cpu().numpy()
    assert np.array_equal(A[dead], old[dead]) and np.array_equal(lse[dead], old_l[dead])
    with np.errstate(invalid="ignore"):
        merged_l = np.logaddexp(old_l, want_l)
        w = np.exp(want_l - merged_l)[..., None]
        merged = np.where(w == 1.0, want, w * want + (1 - w) * np.nan_to_num(old))
    u = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -23}[dtype]
    live = ~dead
    # the row's own bounds, what a shift of lse does to the weights, one rounding of the result
    slack = bound + (bound_l[..., None] + 2.0 ** -20) * (np.abs(want) + np.abs(np.nan_to_num(old))) + u * np.abs(merged)
    assert np.all(np.abs(A - merged)[live] <= slack[live])
    assert np.all(np.abs(lse - merged_l)[live] <= (bound_l + 2.0 ** -20)[live])


@pytest.mark.parametrize("dtype,packed", KINDS)
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_no_numbers_among_the_newest_values(dtype, packed, head, value):
    """V of a drafted token is no number: the tokens before it do not notice, the later ones do."""
    if packed and value == value:
        pytest.skip("e4m3 has no infinity")
    c = P.Case(28, dtype, packed, 2, 2, head, 16, [150, 38])
    for n, at in ((0, 147), (1, 36)):
        page = int(c.table[n, at // 16])
        x = c.pool.float()
        x[page, 1, :, at % 16, 3] = value
        c.pool = x.to(c.pool.dtype)
    c.device()
    q_seq, group = 6, 3
    q = _queries(29, c, q_seq, group)
    A, lse = _run(c, q, group)
    want, want_l = P.attend(c, q, q_seq, group, True)
    A = A.double().cpu().numpy()
    odd = ~np.isfinite(want)
    assert odd.any() and not odd.all() and odd[..., 3].any() and not odd[..., 4].any()
    assert np.array_equal(~np.isfinite(A), odd)
    # (8-bit rows reach 4 * 2^3 = 32 here, of which half a bf16 step alone is 0.06: no fixed
    # tolerance, but the bound of every value, which the formula gives column by column)
    with np.errstate(invalid="ignore"):
        bound, _ = P.attend_bounds(c, q, q_seq, group, True)
        off = np.abs(A - want)
    assert np.all(off[~odd] <= bound[~odd])
    assert np.all(np.isfinite(lse.cpu().numpy()))


@pytest.mark.parametrize("dtype,packed", KINDS)
def test_nan_in_a_visible_key(dtype, packed):
    """... makes the rows that see it NaN, and no others."""
    c = P.Case(30, dtype, packed, 2, 1, 64, 16, [400, 400])
    page = int(c.table[0, 398 // 16])
    x = c.pool.float()
    x[page, 0, 0, 398 % 16, 5] = float("nan")
    c.pool = x.to(c.pool.dtype)
    c.device()
    q = _queries(31, c, 4, 2)
    A, lse = _run(c, q, 2)
    A, lse = A.cpu().reshape(2, 2, 4, 64).isnan(), lse.cpu().reshape(2, 2, 4).isnan()
    sees = torch.tensor([False, False, True, True])     # rows 396 .. 399
    for g in range(2):
        assert torch.equal(lse[g, 0], sees) and not lse[g, 1].any()
        assert torch.equal(A[g, 0].all(-1), sees) and torch.equal(A[g, 0].any(-1), sees) and not A[g, 1].any()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_values_of_very_different_scales(dtype):
    """8-bit rows whose powers of two differ by 2^40 in the values, rows of zeros among them."""
    c = P.Case(32, dtype, True, 2, 1, 128, 16, [300, 77])
    c.scales[:, 1] = torch.where(torch.rand(c.scales[:, 1].shape, generator=torch.Generator().manual_seed(3)) < 0.5,
                                 100, 140 if dtype == "bf16" else 127).to(torch.uint8)
    x = c.pool.float()
    x[:, 1, :, ::5] = 0
    x[~c.there[:, None, None].expand(x.shape[:4])] = float("nan")
    c.pool = x.to(c.pool.dtype)
    c.scales[:, 1, :, ::5] = 1
    _check(c, 2, 4)
    # all values small: nothing of them is lost
    c.scales[:, 1] = 70 if dtype == "bf16" else 110
    c.device()
    q = _queries(33, c, 2, 4)
    A, _ = _run(c, q, 4)
    want, _ = P.attend(c, q, 2, 4, True)
    size = np.abs(want).max()
    # (fp16: the result itself has an absolute step of 2^-24 below 2^-14)
    tol = 2.0 ** -7 * size + (2.0 ** -24 if dtype == "fp16" else 0)
    assert np.abs(A.double().cpu().numpy() - want).max() <= tol


def test_same_bits_every_time():
    c = P.Case(34, "bf16", False, 5, 4, 128, 64, [5000, 1, 900, 3333, 64]).device()
    q = _queries(35, c, 4, 4)
    first = _run(c, q, 4)
    ws = torch.zeros(h.paged_workspace_bytes(q, 5, 4), dtype=torch.uint8, device="cuda")
    for _ in range(5):
        again = _run(c, q, 4, ws=ws)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
