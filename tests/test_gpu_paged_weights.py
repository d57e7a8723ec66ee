"""What cached rows receive of attention, against the definition in 64 bits."""
import numpy as np
import pytest
import torch

from nntile_amd import hip_sdpa as h
from . import paged4_helpers as F
from . import paged_helpers as P

pytestmark = pytest.mark.gpu


def _run(c, q, lse, weights, group, causal, new_rows=None, decay=1.0, stream=None):
    given = torch.tensor(new_rows, dtype=torch.int32).cuda() if new_rows is not None else None
    out = weights.cuda()
    h.paged_attn_weights(c.k, c.dtable, c.dlens, q.cuda(), lse.cuda(), out, h.MASK_CAUSAL if causal else h.MASK_NONE,
                         group, k_scales=c.ks, new_rows=given, decay=decay, stream=stream)
    torch.cuda.synchronize()
    return out.cpu()


def _check(c, q, lse, before, after, q_seq, group, causal, new_rows, decay):
    rows = F.received(c, q, lse, q_seq, group, causal, new_rows)
    before, after = before.double().numpy(), after.double().numpy()
    for n, (total, bound) in enumerate(rows):
        for hd in range(c.heads):
            e, length = n + c.n_batch * hd, total.shape[1]
            old = np.zeros(length) if decay == 0 else float(np.float32(decay)) * before[e, :length]
            want = old + total[hd]
            # (a rounding of the product and the sum)
            room = bound[hd] + 2.0 ** -23 * np.abs(old) + 2.0 ** -24 * np.abs(want)
            assert np.all(np.abs(after[e, :length] - want) <= room), (n, hd)
            assert np.array_equal(after[e, length:], before[e, length:], equal_nan=True)


@pytest.mark.parametrize("dtype,bits", F.KINDS)
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("q_seq,group", [(1, 1), (1, 4), (9, 1), (5, 4), (1, 33), (16, 4), (13, 5), (30, 5)])
def test_weights(dtype, bits, head, q_seq, group):
    """Rows in one block of 16 up to several stages of 64; lengths about every border of a block."""
    print("weights", dtype, bits, head, q_seq, group, flush=True)
    lens = [0, q_seq, 16, 63, 64, 65, 257] if q_seq % 2 else [300, max(1, q_seq - 1), 128]
    causal = q_seq % 3 != 0
    new_rows = None if q_seq % 5 else [max(0, q_seq - i) for i in range(len(lens))]
    decay = {0: 1.0, 1: 0.75, 2: 0.0}[(q_seq + group) % 3]
    c = F.make(q_seq + group, dtype, bits, len(lens), 2, head, 16 if group % 2 else 64, lens).device()
    g = torch.Generator().manual_seed(3)
    q = torch.randn(2 * group * c.n_batch, q_seq, head, generator=g).to(P.TORCH_DT[dtype])
    lse = torch.from_numpy(P.attend(c, q, q_seq, group, causal, new_rows)[1]).float()
    columns = c.max_pages * c.page_rows + 5
    weights = torch.rand(2 * c.n_batch, columns, generator=g)
    if decay == 0.0:
        weights[:, ::3] = float("nan")
    for n in range(c.n_batch):
        weights[n::c.n_batch, c.lens[n]:] = float("nan")        # left as it is
    after = _run(c, q, lse, weights, group, causal, new_rows, decay)
    _check(c, q, lse, weights, after, q_seq, group, causal, new_rows, decay)


def test_weights_of_one_step_add_up_to_the_queries():
    c = F.make(5, "bf16", 16, 3, 2, 128, 16, [100, 40, 9]).device()
    q = torch.randn(24, 2, 128).to(torch.bfloat16)
    A, lse = torch.empty(24, 2, 128, dtype=torch.bfloat16, device="cuda"), torch.empty(24, 2, device="cuda")
    ws = torch.zeros(h.paged_workspace_bytes(q, 3, 4), dtype=torch.uint8, device="cuda")
    h.sdpa_fwd_paged(c.k, c.v, c.dtable, c.dlens, q.cuda(), lse, A, h.MASK_CAUSAL, 4, ws, flags=h.OVERWRITE)
    w = _run(c, q, lse, torch.zeros(6, c.max_pages * 16), 4, True)
    # 4 heads times 2 tokens; a probability errs by a few 2^-20 of itself
    assert torch.allclose(w.double().sum(dim=1), torch.full((6,), 8.0, dtype=torch.float64), rtol=2.0 ** -18, atol=0)


@pytest.mark.parametrize("dtype,bits", F.KINDS)
@pytest.mark.parametrize("group", [2, 20])
def test_what_a_query_does_not_see_does_not_count(dtype, bits, group):
    """NaN in keys that nobody sees - of padded tokens, of pages that are none, behind the last row - and queries whose lse
    is -inf."""
    q_seq, lens = 4, [70, 33]
    c = F.make(7, dtype, bits, 2, 1, 64, 16, lens)
    c.table[0, 1] = -1
    c.device()
    g = torch.Generator().manual_seed(4)
    q = torch.randn(group * 2, q_seq, 64, generator=g).to(P.TORCH_DT[dtype])
    new_rows = [2, 0]
    lse = torch.from_numpy(P.attend(c, q, q_seq, group, True, new_rows)[1]).float()
    lse[1] = float("inf")           # (of sequence 1, which brings nothing)
    lse.view(group, 2, q_seq)[0, 0, 0] = float("-inf")
    q.view(group, 2, q_seq, 64)[0, 0, 0] = 3e4
    q.view(group, 2, q_seq, 64)[:, 0, 2:] = float("nan")        # (padding)
    q.view(group, 2, q_seq, 64)[:, 1] = float("inf")
    weights = torch.rand(2, c.max_pages * 16, generator=g)
    after = _run(c, q, lse, weights, group, True, new_rows, 0.5)
    assert torch.equal(after[1, :33], weights[1, :33] * 0.5)
    assert torch.equal(after[0, 16:32], weights[0, 16:32] * 0.5)
    q.view(group, 2, q_seq, 64)[:, 1] = 0
    q.view(group, 2, q_seq, 64)[:, 0, 2:] = 0
    _check(c, q, lse, weights, after, q_seq, group, True, new_rows, 0.5)


@pytest.mark.parametrize("dtype,bits", F.KINDS)
def test_a_seen_key_that_is_no_number(dtype, bits):
    """Its own weight is NaN, no other."""
    lens = [90]
    c = F.make(8, dtype, bits, 1, 1, 128, 16, lens)
    page = int(c.table[0, 2])
    if bits == 4:
        c.scales[page, 0, 0, 5, 1] = 255
        c.pool[page, 0, 0, 5, 16:32] = 0
    else:
        c.pool[page, 0, 0, 5, 9] = float("nan")
    c.device()
    q = torch.randn(3, 1, 128).to(P.TORCH_DT[dtype])
    after = _run(c, q, torch.zeros(3, 1), torch.zeros(1, c.max_pages * 16), 3, True)
    assert torch.isnan(after[0]).nonzero().flatten().tolist() == [37]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("q_seq,group", [(1, 4), (5, 4), (10, 16)])
def test_four_bit_keys_of_sizes_far_apart(dtype, head, q_seq, group):
    """Powers of two that fp16 has no exponents for, beside usual ones: in one block of 32 values of a sequence, in all."""
    c = F.make(12, dtype, 4, 2, 2, head, 64, [300, 200])
    g = torch.Generator().manual_seed(13)
    size = torch.randint(127 - 30, 127 + 15, c.scales[:, 0].shape, generator=g).to(torch.uint8)
    there = c.there[:, None, :, None].expand(size.shape).clone()
    for page in set(c.table[0].tolist()) - {-1}:
        there[page] = False
    c.scales[:, 0] = torch.where(there, size, c.scales[:, 0])
    c.scales[int(c.table[0, 1]), 0, 1, 6, 1] = 127 - 17
    c.device()
    q = (2.0 ** -7 * torch.randn(4 * group, q_seq, head, generator=g)).to(P.TORCH_DT[dtype])
    lse = torch.from_numpy(P.attend(c, q, q_seq, group, True, None)[1]).float()
    weights = torch.rand(4, c.max_pages * 64, generator=g)
    after = _run(c, q, lse, weights, group, True, None, 0.5)
    _check(c, q, lse, weights, after, q_seq, group, True, None, 0.5)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("group", [3, 16, 37])
def test_a_seen_key_that_is_infinite(dtype, group):
    """Scores of -inf: a weight of 0, and none that the rows which fill up a block of 16 make NaN."""
    c = F.make(11, dtype, 32 if dtype == "fp32" else 16, 1, 1, 64, 16, [90])
    page = int(c.table[0, 2])
    q = torch.randn(group, 1, 64)
    q[:, 0, 9] = -0.5 - torch.rand(group)
    q = q.to(P.TORCH_DT[dtype])
    rest = torch.arange(c.max_pages * 16) != 37
    runs = []
    for key in (1.0, float("inf")):
        c.pool[page, 0, 0, 5, 9] = key
        c.device()
        runs.append(_run(c, q, torch.full((group, 1), 2.0), torch.zeros(1, c.max_pages * 16), group, True)[0])
    assert torch.equal(runs[0][rest], runs[1][rest])
    assert float(runs[0][37]) > 0 and float(runs[1][37]) == 0


@pytest.mark.parametrize("dtype,bits", F.KINDS)
@pytest.mark.parametrize("q_seq,n_batch", [(1, 150), (40, 70)])
def test_weights_of_many_sequences(dtype, bits, q_seq, n_batch):
    """More sequences than a wavefront has lanes, empty ones among them, more blocks than workgroups; the same bits twice."""
    print("many", dtype, bits, q_seq, flush=True)
    lens = [0 if i % 5 == 4 else q_seq + (37 * i) % 330 for i in range(n_batch)]
    c = F.make(9, dtype, bits, n_batch, 2, 64, 32, lens).device()
    g = torch.Generator().manual_seed(6)
    q = torch.randn(4 * n_batch, q_seq, 64, generator=g).to(P.TORCH_DT[dtype])
    weights = torch.rand(2 * n_batch, c.max_pages * 32, generator=g)
    lse = torch.full((4 * n_batch, q_seq), 3.0)
    a = _run(c, q, lse, weights, 2, True, None, 0.25)
    b = _run(c, q, lse, weights, 2, True, None, 0.25, stream=torch.cuda.Stream())
    assert torch.equal(a.view(torch.int32), b.view(torch.int32))
    _check(c, q, lse, weights, a, q_seq, 2, True, None, 0.25)


@pytest.mark.parametrize("dtype,bits", F.KINDS)
@pytest.mark.parametrize("q_seq,group,given", [(5, 28, 5), (1, 129, 1), (3, 90, 2), (4, 40, 3)])
@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
def test_a_first_query_that_counts_nothing(dtype, bits, q_seq, group, given, fill):
    """More query rows than are staged at a time, some that only fill up a block of 16 or are padding, and a first one
    whose lse is -inf over a query that is no number: no key receives anything of it."""
    print("first", dtype, bits, q_seq, group, given, fill, flush=True)
    lens = [600, 300]               # (more than one block of keys that every query sees)
    c = F.make(14, dtype, bits, 2, 1, 64, 64, lens).device()
    g = torch.Generator().manual_seed(15)
    q = torch.randn(group * 2, q_seq, 64, generator=g).to(P.TORCH_DT[dtype])
    new_rows = [given, q_seq]
    lse = torch.from_numpy(P.attend(c, q, q_seq, group, True, new_rows)[1]).float()
    q.view(group, 2, q_seq, 64)[0, 0, 0] = fill
    lse.view(group, 2, q_seq)[0, 0, 0] = float("-inf")
    weights = torch.rand(2, c.max_pages * 64, generator=g)
    after = _run(c, q, lse, weights, group, True, new_rows, 0.5)
    _check(c, q, lse, weights, after, q_seq, group, True, new_rows, 0.5)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("q_seq,group", [(1, 4), (2, 16), (5, 28)])
def test_four_bit_rows_that_are_none_do_not_choose_the_arithmetic(dtype, head, q_seq, group):
    """The same bits whatever lies behind the last rows, in pages that no sequence has and in a page that a bad entry of the
    table is read as."""
    c = F.Case4(16, dtype, 2, 2, head, 16, [300, 77])
    c.table[0, 3], c.table[1, 2] = -1, c.n_pages
    F.free_first_page(c)
    g = torch.Generator().manual_seed(17)
    q = torch.randn(4 * group, q_seq, head, generator=g).to(P.TORCH_DT[dtype])
    lse = torch.from_numpy(P.attend(c, q, q_seq, group, True, None)[1]).float()
    runs = [_run(F.in_the_rest(c, byte).device(), q, lse, torch.zeros(4, c.max_pages * 16), group, True)
            for byte in (127, 1, 252, 255)]
    for other in runs[1:]:
        assert torch.equal(runs[0].view(torch.int32), other.view(torch.int32))
    _check(c, q, lse, torch.zeros(4, c.max_pages * 16), runs[0], q_seq, group, True, None, 1.0)
