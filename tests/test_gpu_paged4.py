"""Pages of 4-bit codes: rows written, read back and attended over, against their definitions in 64 bits."""
import numpy as np
import pytest
import torch

from nntile_amd import hip_sdpa as h
from . import paged4_helpers as F
from . import paged_bounds
from . import paged_helpers as P

pytestmark = pytest.mark.gpu

LARGEST = {"bf16": 3.3e38, "fp16": 65504.0}


def _bits(t):
    return t.view(torch.uint8)


def _values(seed, dtype, shape):
    """Values with what a block may hold: sizes of all kinds, zeros, ties, subnormal numbers, the largest."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g, dtype=torch.float64)
    b = x.view(-1, 32)
    kind = torch.arange(b.shape[0]) % 9
    spread = 30 if dtype == "fp16" else 200
    b[kind == 1] *= torch.exp2(torch.randint(-spread // 2, spread // 3, (int((kind == 1).sum()), 1), generator=g).double())
    b[kind == 2] = 0.0
    b[kind == 3] = torch.randint(-28, 29, (int((kind == 3).sum()), 32), generator=g).double() / 4.0      # ties, and 7 among them
    b[kind == 4] *= 2.0 ** (-133 if dtype == "bf16" else -22)
    b[kind == 5, 3] = LARGEST[dtype]
    b[kind == 6] = torch.where(torch.rand(b[kind == 6].shape, generator=g) < 0.9, -0.0, b[kind == 6])
    b[kind == 7] = 1.0
    return x.clamp(-LARGEST[dtype], LARGEST[dtype]).to(P.TORCH_DT[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("rows,page_rows,new_rows", [(1, 16, None), (19, 16, None), (70, 64, [70, 0, 5, 69]), (3, 32, [9, -2, 1, 3])])
def test_rows_written(dtype, head, rows, page_rows, new_rows):
    """Codes and bytes of the new rows bit for bit; every other byte of the pool stays."""
    print("write", dtype, head, rows, page_rows, new_rows, flush=True)
    lens = [200, 70, 71, 130]
    c = F.Case4(3, dtype, 4, 3, head, page_rows, lens, spread=1).device()
    k, v = _values(1, dtype, (12, rows, head)), _values(2, dtype, (12, rows, head))
    if rows > 2:
        k[0, 2, 5], v[1, 1, 40], v[1, 2, 41] = float("inf"), float("nan"), float("-inf")
    given = torch.tensor(new_rows, dtype=torch.int32).cuda() if new_rows else None
    h.paged_kv_append(k.cuda(), v.cuda(), c.k, c.v, c.dtable, c.dlens, c.ks, c.vs, new_rows=given)
    torch.cuda.synchronize()
    want, want_s = c.pool.numpy().copy(), c.scales.numpy().copy()
    for which, x in ((0, k), (1, v)):
        codes, size = F.quantised4(x.double().numpy().reshape(3, 4, rows, head))
        for n in range(4):
            count = rows if new_rows is None else max(0, min(rows, new_rows[n]))
            for r in range(count):
                row = lens[n] - count + r
                if row >= 0:
                    page = int(c.table[n, row // page_rows])
                    want[page, which, :, row % page_rows] = codes[:, n, r]
                    want_s[page, which, :, row % page_rows] = size[:, n, r]
    assert np.array_equal(c.dscales.cpu().numpy(), want_s)
    assert np.array_equal(c.dpool.cpu().numpy(), want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("first,rows", [(0, 230), (13, 1), (100, 64), (250, 40)])
def test_rows_read(dtype, head, first, rows):
    print("read", dtype, head, first, rows, flush=True)
    c = F.Case4(4, dtype, 4, 3, head, 16, [0, 1, 100, 230], scale=3.0)
    # all bytes that stand for something, all codes
    g = torch.Generator().manual_seed(9)
    c.scales[c.there[:, None, None].expand(c.scales.shape[:4])] = torch.randint(
        1, 253, (int(c.there.sum()) * 6, head // 32), generator=g).to(torch.uint8)
    c.table[3, 2] = -1
    c.table[2, 1] = c.n_pages
    c.device()
    k = torch.full((12, rows, head), 7.0, dtype=P.TORCH_DT[dtype], device="cuda")
    v = torch.full_like(k, 7.0)
    h.paged_kv_read(c.k, c.v, c.dtable, c.dlens, k, v, first=first, k_scales=c.ks, v_scales=c.vs)
    for which, x in ((0, k), (1, v)):
        x = x.double().cpu().numpy().reshape(3, 4, rows, head)
        for n in range(4):
            want, ok = c.rows(n, which)
            want = want.clip(-65504.0, 65504.0) if dtype == "fp16" else want
            want = torch.from_numpy(want[:, first:first + rows]).to(P.TORCH_DT[dtype]).double().numpy()
            assert np.array_equal(x[:, n, :want.shape[1]], want)
            assert not x[:, n, want.shape[1]:].any()


def test_a_block_that_is_no_number():
    """NaN in, NaN out, its 32 values only."""
    c = F.Case4(5, "bf16", 1, 1, 128, 16, [2]).device()
    x = torch.randn(1, 2, 128).to(torch.bfloat16)
    x[0, 0, 40] = float("inf")
    y = torch.empty_like(x, device="cuda")
    h.paged_kv_append(x.cuda(), x.cuda(), c.k, c.v, c.dtable, c.dlens, c.ks, c.vs)
    h.paged_kv_read(c.k, c.v, c.dtable, c.dlens, y, torch.empty_like(y), k_scales=c.ks, v_scales=c.vs)
    nan = torch.zeros(1, 2, 128, dtype=torch.bool)
    nan[0, 0, 32:64] = True
    assert torch.equal(y.isnan().cpu(), nan)


def _attend(c, q, group, causal, new_rows=None, ws=None, flags=h.OVERWRITE, A=None, lse=None, stream=None):
    A = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda") if A is None else A
    lse = torch.full(q.shape[:2], float("nan"), device="cuda") if lse is None else lse
    ws = torch.full((h.paged_workspace_bytes(q, c.n_batch, group),), 0x5a, dtype=torch.uint8, device="cuda") if ws is None else ws
    given = torch.tensor(new_rows, dtype=torch.int32).cuda() if new_rows is not None else None
    h.sdpa_fwd_paged(c.k, c.v, c.dtable, c.dlens, q.cuda(), lse, A, h.MASK_CAUSAL if causal else h.MASK_NONE, group, ws,
                     k_scales=c.ks, v_scales=c.vs, new_rows=given, flags=flags, stream=stream)
    return A, lse


def _check(c, q, q_seq, group, causal, new_rows, A, lse):
    want, want_l = P.attend(c, q, q_seq, group, causal, new_rows)
    _, bound_l = P.attend_bounds(c, q, q_seq, group, causal, new_rows)
    bound = paged_bounds.column_bounds(c, q, q_seq, group, causal, new_rows)
    dead = np.isneginf(want_l)
    got, got_l = A.double().cpu().numpy(), lse.double().cpu().numpy()
    assert np.array_equal(np.isneginf(got_l), dead)
    assert np.all(np.abs(got - want) <= bound), np.max(np.abs(got - want) / bound)
    assert np.all(np.abs(got_l - want_l)[~dead] <= bound_l[~dead])


LENS = [[0], [1], [15, 16, 17], [0, 63, 64, 65, 200], [1000, 3, 0, 257]]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("q_seq,group", [(1, 1), (1, 4), (4, 4), (1, 17), (8, 4), (3, 11), (16, 4), (20, 4)])
@pytest.mark.parametrize("lens", LENS)
def test_attention(dtype, head, q_seq, group, lens):
    print("attend", dtype, head, q_seq, group, lens, flush=True)
    causal = (q_seq + len(lens)) % 3 != 0
    c = F.Case4(q_seq * 10 + len(lens), dtype, len(lens), 2, head, 16 if len(lens) % 2 else 128, lens).device()
    g = torch.Generator().manual_seed(11)
    q = torch.randn(2 * group * c.n_batch, q_seq, head, generator=g).to(P.TORCH_DT[dtype])
    new_rows = None if len(lens) != 4 else [q_seq, q_seq // 2, 0, max(1, q_seq - 1)]
    A, lse = _attend(c, q, group, causal, new_rows)
    _check(c, q, q_seq, group, causal, new_rows, A, lse)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("n_batch,heads,q_seq,group,length", [(40, 2, 1, 4, 300), (3, 1, 2, 40, 900), (130, 1, 1, 16, 70),
                                                              (20, 8, 8, 4, 130)])
def test_attention_of_many_units(dtype, head, n_batch, heads, q_seq, group, length):
    """More units than a wavefront scans, several row groups of a head, units that end inside a share."""
    print("units", dtype, head, n_batch, heads, q_seq, group, flush=True)
    lens = [max(q_seq, (length * (i % 7 + 1)) // 7) for i in range(n_batch)]
    c = F.Case4(21, dtype, n_batch, heads, head, 32, lens).device()
    q = torch.randn(heads * group * n_batch, q_seq, head, generator=torch.Generator().manual_seed(12)).to(P.TORCH_DT[dtype])
    A, lse = _attend(c, q, group, True)
    _check(c, q, q_seq, group, True, None, A, lse)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_attention_merged_into_what_is_there(dtype):
    """Without OVERWRITE: the running pair, and rows that see nothing stay."""
    c = F.Case4(31, dtype, 3, 2, 128, 16, [90, 0, 33]).device()
    q = torch.randn(12, 2, 128).to(P.TORCH_DT[dtype])
    fresh_A, fresh_l = _attend(c, q, 2, True)
    old_A, old_l = torch.randn(12, 2, 128).to(P.TORCH_DT[dtype]).cuda(), torch.randn(12, 2).cuda()
    A, lse = _attend(c, q, 2, True, flags=0, A=old_A.clone(), lse=old_l.clone())
    dead = torch.isneginf(fresh_l)
    assert torch.equal(_bits(A[dead]), _bits(old_A[dead])) and torch.equal(lse[dead], old_l[dead])
    both = torch.logaddexp(fresh_l.double(), old_l.double())
    assert torch.allclose(lse.double()[~dead], both[~dead], rtol=0, atol=2e-6)
    want = (fresh_A.double() * torch.exp(fresh_l.double() - both)[..., None]
            + old_A.double() * torch.exp(old_l.double() - both)[..., None])
    # half a step of the result, and of the fresh one, which was rounded, too
    u = paged_bounds.HALF_STEP[dtype]
    size = fresh_A.double().abs() + old_A.double().abs()
    assert bool(((A.double() - want).abs() <= 2.1 * u * size + 2.0 ** -24)[~dead].all())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("q_seq,group", [(4, 1), (12, 2), (16, 4)])
def test_rows_that_are_no_numbers(dtype, head, q_seq, group):
    """A NaN block of a newer token does not reach the tokens in front of it; the tokens from there on get it, in its 32
    columns where it is a value, in all where it is a key."""
    lens = [100, 130]
    c = F.Case4(41, dtype, 2, 1, head, 16, lens)
    at = [lens[0] - q_seq + 2, lens[1] - q_seq + 1]       # sequence 0: a value's first block; 1: a key's
    for n, which in ((0, 1), (1, 0)):
        page = int(c.table[n, at[n] // 16])
        c.scales[page, which, 0, at[n] % 16, 0] = 255
        c.pool[page, which, 0, at[n] % 16, :16] = 0
    c.device()
    q = torch.randn(2 * group, q_seq, head, generator=torch.Generator().manual_seed(13)).to(P.TORCH_DT[dtype])
    A, lse = _attend(c, q, group, True)
    A, lse = A.cpu().view(group, 2, q_seq, head), lse.cpu().view(group, 2, q_seq)
    want = torch.zeros(group, 2, q_seq, head, dtype=torch.bool)
    want[:, 0, 2:, :32] = True
    want[:, 1, 1:] = True
    assert torch.equal(A.isnan(), want)
    want_l = torch.zeros(group, 2, q_seq, dtype=torch.bool)
    want_l[:, 1, 1:] = True
    assert torch.equal(lse.isnan(), want_l)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("q_seq,group", [(1, 4), (8, 4), (16, 4)])
def test_blocks_of_sizes_far_apart(dtype, q_seq, group):
    """Values whose blocks' powers of two lie 2^200 apart: every column within its own bound; an old value that is no
    number reaches its columns of every token, past 64 keys of whole steps."""
    c = F.Case4(51, dtype, 2, 2, 128, 64, [700, 500])
    g = torch.Generator().manual_seed(52)
    top = 100 if dtype == "bf16" else 8
    size = torch.randint(127 - top, 127 + top, c.scales[:, 1].shape, generator=g).to(torch.uint8)
    size[..., 3] = 127 + top
    c.scales[:, 1] = torch.where(c.there[:, None, :, None].expand(size.shape), size, c.scales[:, 1])
    if dtype == "bf16":
        page = int(c.table[0, 1])
        c.scales[page, 1, 1, 7, 2] = 255
        c.pool[page, 1, 1, 7, 32:48] = 0
    c.device()
    q = torch.randn(2 * group * 2, q_seq, 128, generator=g).to(P.TORCH_DT[dtype])
    A, lse = _attend(c, q, group, True)
    if dtype == "bf16":
        bad = torch.zeros(2, group, 2, q_seq, 128, dtype=torch.bool)
        bad[1, :, 0, :, 64:96] = True
        bad = bad.view(A.shape)
        assert torch.equal(A.isnan().cpu(), bad)
        c.scales[page, 1, 1, 7, 2] = 1
        A[bad.cuda()] = torch.from_numpy(P.attend(c, q, q_seq, group, True)[0]).to(A.dtype)[bad].cuda()
    _check(c, q, q_seq, group, True, None, A, lse)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("q_seq,group", [(1, 4), (5, 4), (10, 6)])
def test_keys_of_sizes_far_apart(dtype, head, q_seq, group):
    """Keys' powers of two that fp16 has no exponents for, beside usual ones: in one block of 32 values of a sequence, in
    all blocks of the other."""
    c = F.Case4(55, dtype, 2, 2, head, 64, [900, 500])
    g = torch.Generator().manual_seed(56)
    size = torch.randint(127 - 30, 127 + 15, c.scales[:, 0].shape, generator=g).to(torch.uint8)
    there = c.there[:, None, :, None].expand(size.shape).clone()
    for page in set(c.table[0].tolist()) - {-1}:
        there[page] = False
    c.scales[:, 0] = torch.where(there, size, c.scales[:, 0])
    c.scales[int(c.table[0, 3]), 0, 1, 6, 1] = 127 - 17
    c.device()
    q = (2.0 ** -7 * torch.randn(4 * group, q_seq, head, generator=g)).to(P.TORCH_DT[dtype])
    A, lse = _attend(c, q, group, True)
    _check(c, q, q_seq, group, True, None, A, lse)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("byte", [191, 192, 252])
def test_the_largest_values_of_a_row_without_weight(dtype, head, byte):
    """A row that every query sees, with a score of some -1000 and values of 6 * 2^(byte - 127), among rows of usual ones:
    it leaves them as they are."""
    c = F.Case4(53, dtype, 1, 1, head, 64, [900])
    page = int(c.table[0, 2])
    c.pool[page, :, 0, 11] = 0x77          # 6 everywhere
    c.scales[page, 0, 0, 11] = 127 + 6
    c.scales[page, 1, 0, 11] = byte
    c.device()
    q = -torch.rand(16, 1, head, generator=torch.Generator().manual_seed(54)).to(P.TORCH_DT[dtype])
    A, lse = _attend(c, q, 16, True)
    _check(c, q, 1, 16, True, None, A, lse)


def test_a_table_with_entries_that_are_no_pages():
    c = F.Case4(61, "bf16", 2, 2, 64, 16, [100, 90])
    c.table[0, 2], c.table[1, 5], c.table[1, 0] = -1, c.n_pages, 1 << 30
    c.device()
    q = torch.randn(8, 3, 64).to(torch.bfloat16)
    A, lse = _attend(c, q, 2, True)
    _check(c, q, 3, 2, True, None, A, lse)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_the_same_bits_on_any_workspace_and_stream(dtype):
    c = F.Case4(71, dtype, 5, 2, 128, 16, [700, 40, 0, 513, 64]).device()
    q = torch.randn(40, 2, 128).to(P.TORCH_DT[dtype])
    A, lse = _attend(c, q, 4, True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for i in range(3):
        ws = torch.randint(0, 256, (h.paged_workspace_bytes(q, 5, 4),), dtype=torch.uint8, device="cuda")
        side.wait_stream(torch.cuda.current_stream())
        B, other = _attend(c, q, 4, True, ws=ws, stream=side if i == 1 else None)
        torch.cuda.synchronize()
        assert torch.equal(_bits(A), _bits(B)) and torch.equal(_bits(lse), _bits(other))


def test_pages_behind_four_gigabytes():
    """Codes and bytes whose offsets pass 32 bits: a pool of few pages far apart."""
    stride, apart = (1 << 31) + 4096, (1 << 30) + 64
    pool = torch.zeros(3 * stride, dtype=torch.uint8, device="cuda")
    scales = torch.ones(5 * apart, dtype=torch.uint8, device="cuda")
    k = pool.as_strided((3, 2, 16, 32), (stride, 512, 32, 1)).view(F.F4)
    v = pool[4096 - 1024:].as_strided((3, 2, 16, 32), (stride, 512, 32, 1)).view(F.F4)
    ks, vs = (scales[i * 4096:].as_strided((3, 2, 16, 2), (2 * apart, 32, 2, 1)) for i in (0, 1))
    c = F.Case4(81, "bf16", 1, 2, 64, 16, [40])
    c.table = torch.tensor([[2, 0, 1]], dtype=torch.int32)
    c.dtable, c.dlens = c.table.cuda(), torch.tensor([40], dtype=torch.int32).cuda()
    x, y = (torch.randn(2, 40, 64).to(torch.bfloat16) for _ in range(2))
    h.paged_kv_append(x.cuda(), y.cuda(), k, v, c.dtable, c.dlens, ks, vs)
    a, b = torch.empty_like(x, device="cuda"), torch.empty_like(x, device="cuda")
    h.paged_kv_read(k, v, c.dtable, c.dlens, a, b, k_scales=ks, v_scales=vs)
    for got, put in ((a, x), (b, y)):
        assert np.array_equal(got.double().cpu().numpy(), F.values4(*F.quantised4(put.double().numpy())))
    c.k, c.v, c.ks, c.vs = k, v, ks, vs
    q = torch.randn(4, 1, 64).to(torch.bfloat16)
    A, lse = _attend(c, q, 2, True)
    rows = [t.double().cpu().numpy() for t in (a, b)]
    c.rows = lambda n, which, count=None: (rows[which], np.ones(40, bool))
    _check(c, q, 1, 2, True, None, A, lse)
    # (the pages of the second tensor begin where those of the first end)
    assert pool[:stride].count_nonzero() > 0 and pool[2 * stride:2 * stride + 4096].count_nonzero() > 0


class Step:
    """A generation step over 4-bit pages that can be captured: append, attention, the weights received."""

    def __init__(self, dtype, ws):
        self.c = F.Case4(91, dtype, 3, 2, 128, 16, [40, 7, 90], max_pages=20).device()
        spare = torch.arange(self.c.n_pages, self.c.n_pages + 60, dtype=torch.int32)
        pool, scales = self.c.dpool, self.c.dscales
        self.pool = torch.cat([pool, torch.zeros(60, *pool.shape[1:], dtype=torch.uint8, device="cuda")])
        self.scales = torch.cat([scales, torch.ones(60, *scales.shape[1:], dtype=torch.uint8, device="cuda")])
        table = self.c.table.clone()
        table[table < 0] = spare[:int((table < 0).sum())]
        self.table, self.lens = table.cuda(), torch.tensor([40, 7, 90], dtype=torch.int32).cuda()
        t = P.TORCH_DT[dtype]
        self.k, self.v = (torch.zeros(6, 5, 128, dtype=t, device="cuda") for _ in range(2))
        self.q = torch.zeros(24, 5, 128, dtype=t, device="cuda")
        self.A, self.lse = torch.zeros_like(self.q), torch.zeros(24, 5, device="cuda")
        self.given = torch.zeros(3, dtype=torch.int32, device="cuda")
        self.weights, self.ws = torch.zeros(6, 320, device="cuda"), ws

    def feed(self, i):
        g = torch.Generator().manual_seed(1000 + i)
        for t in (self.k, self.v, self.q):
            t.copy_(torch.randn(t.shape, generator=g).to(t.dtype))
        self.given.copy_(torch.tensor([5, i % 6, (3 * i) % 6], dtype=torch.int32))

    def step(self, stream=None):
        pages = [self.pool[:, i].view(F.F4) for i in (0, 1)]
        scales = dict(k_scales=self.scales[:, 0], v_scales=self.scales[:, 1])
        with torch.cuda.stream(stream):
            self.lens.add_(self.given)
        h.paged_kv_append(self.k, self.v, *pages, self.table, self.lens, new_rows=self.given, stream=stream, **scales)
        h.sdpa_fwd_paged(*pages, self.table, self.lens, self.q, self.lse, self.A, h.MASK_CAUSAL, 4, self.ws,
                         new_rows=self.given, flags=h.OVERWRITE, stream=stream, **scales)
        h.paged_attn_weights(pages[0], self.table, self.lens, self.q, self.lse, self.weights, h.MASK_CAUSAL, 4,
                             k_scales=scales["k_scales"], new_rows=self.given, decay=0.9, stream=stream)

    def same(self, other):
        return all(torch.equal(_bits(getattr(self, n)), _bits(getattr(other, n)))
                   for n in ("A", "lse", "weights", "pool", "scales", "lens"))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_a_captured_step_replayed(dtype):
    """One captured step, replayed while the lengths grow, beside eager work on the same workspace."""
    ws = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
    eager, graphed, alone = Step(dtype, torch.zeros_like(ws)), Step(dtype, ws), Step(dtype, ws)
    graph = torch.cuda.CUDAGraph()
    for i in range(8):
        for s in (eager, graphed, alone):
            s.feed(i)
        eager.step()
        if i == 2:
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                graphed.step()
        if i < 2:
            graphed.step()
        else:
            graph.replay()
        alone.step()
        torch.cuda.synchronize()
        assert eager.same(graphed) and eager.same(alone)


def test_steps_on_two_streams():
    want = [Step(t, torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")) for t in ("bf16", "fp16")]
    steps = [Step(t, torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")) for t in ("bf16", "fp16")]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(4):
        for s in want:
            s.feed(i)
            s.step()
        for s, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                stream.wait_stream(torch.cuda.default_stream())
                s.feed(i)
            s.step(stream=stream)
        torch.cuda.synchronize()
        for a, b in zip(want, steps):
            assert a.same(b)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_the_largest_values_stay_finite(dtype):
    """Blocks of the type's largest value: what comes back is 6 * 2^125 of bf16, the largest value of fp16 again."""
    c = F.Case4(101, dtype, 1, 1, 64, 16, [1]).device()
    top = torch.finfo(P.TORCH_DT[dtype]).max
    x = torch.full((1, 1, 64), top, dtype=P.TORCH_DT[dtype])
    y, z = torch.empty_like(x, device="cuda"), torch.empty_like(x, device="cuda")
    h.paged_kv_append(x.cuda(), -x.cuda(), c.k, c.v, c.dtable, c.dlens, c.ks, c.vs)
    h.paged_kv_read(c.k, c.v, c.dtable, c.dlens, y, z, k_scales=c.ks, v_scales=c.vs)
    want = 6.0 * 2.0 ** 125 if dtype == "bf16" else 65504.0
    assert y.double().unique().tolist() == [want] and z.double().unique().tolist() == [-want]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("q_seq,group,causal", [(1, 4, True), (1, 32, True), (8, 4, True), (5, 28, False)])
def test_rows_that_are_none_do_not_choose_the_arithmetic(dtype, head, q_seq, group, causal):
    """The same bits whatever lies behind the last rows, in pages that no sequence has and in a page that a bad entry of the
    table is read as."""
    c = F.Case4(111, dtype, 2, 2, head, 16, [700, 77])
    c.table[0, 3], c.table[1, 2] = -1, c.n_pages
    F.free_first_page(c)
    q = torch.randn(4 * group, q_seq, head, generator=torch.Generator().manual_seed(112)).to(P.TORCH_DT[dtype])
    runs = [_attend(F.in_the_rest(c, byte).device(), q, group, causal) for byte in (127, 1, 252, 255)]
    for A, lse in runs[1:]:
        assert torch.equal(_bits(A), _bits(runs[0][0])) and torch.equal(_bits(lse), _bits(runs[0][1]))
    _check(c, q, q_seq, group, causal, None, *runs[0])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("q_seq,group", [(4, 1), (8, 4), (16, 4), (40, 2)])
def test_newer_tokens_do_not_choose_the_arithmetic(dtype, head, q_seq, group):
    """The same bits of every token whatever powers of two the keys and values of the newer ones have."""
    lens = [700, 77]
    c = F.Case4(113, dtype, 2, 1, head, 64, lens)
    q = torch.randn(2 * group, q_seq, head, generator=torch.Generator().manual_seed(114)).to(P.TORCH_DT[dtype])
    want = [t.cpu() for t in _attend(c.device(), q, group, True)]
    _check(c, q, q_seq, group, True, None, *want)
    # (from the newest token on backwards: what has been changed stays)
    for token in range(q_seq - 1, 0, -max(1, q_seq // 4)):
        for n, length in enumerate(lens):
            row = length - q_seq + token
            c.scales[int(c.table[n, row // 64]), :, 0, row % 64] = 127 - 17
        got = [t.cpu() for t in _attend(c.device(), q, group, True)]
        _check(c, q, q_seq, group, True, None, *got)
        for a, b in zip(got, want):
            a, b = (t.view(group, 2, q_seq, -1)[:, :, :token] for t in (a, b))
            assert torch.equal(_bits(a.contiguous()), _bits(b.contiguous()))
