"""Eviction from a paged cache: which rows stay, and that they and nothing else move."""
import numpy as np
import pytest
import torch

from nntile_amd import hip_sdpa as h
from nntile_amd.kv_cache import PagedKVCache
from . import paged4_helpers as F
from . import paged_helpers as P

pytestmark = pytest.mark.gpu


def _bytes(t):
    return t.contiguous().view(torch.uint8).cpu().numpy()


def _weights(seed, c, kind):
    g = torch.Generator().manual_seed(seed)
    w = torch.exp(3 * torch.randn(c.heads * c.n_batch, c.max_pages * c.page_rows, generator=g) - 3)
    if kind == "ties":
        w = torch.randint(0, 4, w.shape, generator=g).float()
    elif kind == "zeros":
        w[:] = 0.0
    elif kind == "odd":
        # NaN, infinities, both zeros, numbers below zero and subnormal ones
        odd = torch.tensor([float("nan"), float("inf"), float("-inf"), 0.0, -0.0, -1.0, 1e-40, -1e-41, 1.0])
        w = odd[torch.randint(0, len(odd), w.shape, generator=g)]
    return w


def _expected(c, w, keep, recent):
    """kept, weights_out (columns below lens) and the pool after the call."""
    kept = np.full((c.heads * c.n_batch, keep), -1, np.int32)
    out = w.numpy().copy()
    pool, scales = c.pool.clone(), c.scales.clone()
    before, before_s = c.pool.clone(), c.scales.clone()
    for n in range(c.n_batch):
        length = max(0, min(c.lens[n], c.max_pages * c.page_rows))
        for hd in range(c.heads):
            e = n + c.n_batch * hd
            stay = F.chosen(w[e].numpy(), length, keep, recent)
            kept[e, :len(stay)] = stay
            out[e, :length] = 0.0
            out[e, :len(stay)] = w[e].numpy()[stay]
            for d, src in enumerate(stay):
                if d != src:
                    to, of = int(c.table[n, d // c.page_rows]), int(c.table[n, src // c.page_rows])
                    if 0 <= to < c.n_pages:
                        here = (to, slice(None), hd, d % c.page_rows)
                        if 0 <= of < c.n_pages:
                            there = (of, slice(None), hd, src % c.page_rows)
                            pool[here], scales[here] = before[there], before_s[there]
                        else:
                            pool[here], scales[here] = 0, 127
    return kept, out, pool, scales


def _run(c, w, keep, recent, in_place=True, stream=None):
    w = w.cuda()
    out = w if in_place else torch.full_like(w, 77.0)
    kept = torch.full((w.shape[0], keep), 99, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    h.paged_kv_evict(c.k, c.v, c.dtable, c.dlens, w, out, kept, recent, k_scales=c.ks, v_scales=c.vs, stream=stream)
    torch.cuda.synchronize()
    return kept.cpu().numpy(), out.cpu().numpy()


def _check(c, w, keep, recent, in_place=True):
    kept, out, pool, scales = _expected(c, w, keep, recent)
    got, got_w = _run(c, w, keep, recent, in_place)
    assert np.array_equal(got, kept)
    for n in range(c.n_batch):
        length = max(0, min(c.lens[n], c.max_pages * c.page_rows))
        for e in range(n, len(out), c.n_batch):
            assert np.array_equal(got_w[e, :length].view(np.int32), out[e, :length].view(np.int32))
            behind = w[e, length:].numpy() if in_place else np.full_like(out[e, length:], 77.0)
            assert np.array_equal(got_w[e, length:], behind, equal_nan=True)
    spread = c.spread
    c.spread = 1
    if spread:
        assert np.array_equal(_bytes(c.dpool), _bytes(pool))
        if c.packed:
            assert np.array_equal(_bytes(c.dscales), _bytes(scales))
    else:
        for got_t, which in ((c.k, 0), (c.v, 1)):
            assert np.array_equal(_bytes(got_t), _bytes(pool[:, which]))
        if c.packed:
            for got_t, which in ((c.ks, 0), (c.vs, 1)):
                assert np.array_equal(_bytes(got_t), _bytes(scales[:, which]))
    c.spread = spread


@pytest.mark.parametrize("dtype,bits", F.KINDS)
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("keep,recent,kind", [(50, 10, "any"), (1, 0, "any"), (1, 1, "any"), (64, 64, "odd"), (77, 0, "odd"),
                                              (63, 5, "ties"), (100, 40, "zeros"), (130, 1, "ties"), (500, 7, "any")])
def test_eviction(dtype, bits, head, keep, recent, kind):
    """Lengths about keep, empty and longer ones; a pool whose other bytes stay."""
    print("evict", dtype, bits, head, keep, recent, kind, flush=True)
    lens = [0, 1, keep - 1, keep, keep + 1, 200, 131]
    c = F.make(keep, dtype, bits, len(lens), 2, head, 16, lens, spread=keep % 2).device()
    _check(c, _weights(1, c, kind), keep, recent, in_place=keep % 3 != 0)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("length,keep,recent,kind", [(4096, 4095, 0, "ties"), (4097, 4096, 100, "any"), (5000, 100, 0, "odd"),
                                                     (9001, 8200, 1000, "any"), (40000, 33000, 5, "ties"),
                                                     (70001, 1001, 1000, "zeros")])
def test_long_sequences(bits, length, keep, recent, kind):
    """More rows than one step of the selection, and of the moves, takes."""
    print("long", bits, length, keep, recent, kind, flush=True)
    c = F.make(2, "bf16", bits, 2, 1, 64, 256, [length, length // 2]).device()
    _check(c, _weights(2, c, kind), keep, recent)


@pytest.mark.parametrize("dtype,bits,head", [("bf16", 4, 64), ("fp16", 4, 128), ("bf16", 8, 64), ("fp16", 16, 128), ("fp32", 32, 128)])
@pytest.mark.parametrize("first", [0, 1, 1023, 1024, 2047, 2049, 4100, 5890])
def test_rows_that_stay_where_they_are(dtype, bits, head, first):
    """One row goes, and the others behind it move by one; another head loses its last that may go."""
    c = F.make(21, dtype, bits, 1, 2, head, 64, [6000]).device()
    w = torch.ones(2, c.max_pages * c.page_rows)
    w[0, first] = 0.5
    _check(c, w, 5999, 100)


def test_many_entries():
    c = F.make(3, "bf16", 16, 300, 9, 64, 16, [i % 40 for i in range(300)]).device()
    _check(c, _weights(3, c, "any"), 16, 4)


@pytest.mark.parametrize("dtype,bits", F.KINDS)
def test_tables_with_entries_that_are_no_pages(dtype, bits):
    c = F.make(4, dtype, bits, 2, 2, 64, 16, [100, 90], junk=1.0) if bits != 4 else F.make(4, dtype, 4, 2, 2, 64, 16, [100, 90])
    c.table[0, 2], c.table[0, 5], c.table[1, 0], c.table[1, 3] = -1, c.n_pages, 1 << 30, -7
    c.device()
    _check(c, _weights(4, c, "any"), 60, 8)


def test_a_length_past_the_table_counts_for_its_rows():
    c = F.make(5, "bf16", 16, 2, 1, 64, 16, [80, 33]).device()
    c.lens = [500, -3]
    c.dlens = torch.tensor(c.lens, dtype=torch.int32).cuda()
    _check(c, _weights(5, c, "any"), 40, 8)


def test_the_same_on_another_stream_and_in_a_graph():
    """Captured once and replayed on caches that were put back, with eager work between."""
    c = F.make(6, "bf16", 4, 3, 2, 128, 16, [200, 50, 131], spread=1).device()
    w = _weights(6, c, "any")
    kept, out, pool, scales = _expected(c, w, 60, 9)
    fresh, fresh_s = c.dpool.clone(), c.dscales.clone()
    side = torch.cuda.Stream()
    got, got_w = _run(c, w, 60, 9, stream=side)
    assert np.array_equal(got, kept) and np.array_equal(_bytes(c.dpool), _bytes(pool))
    w_dev, out_dev = w.cuda(), torch.zeros_like(w, device="cuda")
    kept_dev = torch.zeros(6, 60, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h.paged_kv_evict(c.k, c.v, c.dtable, c.dlens, w_dev, out_dev, kept_dev, 9, k_scales=c.ks, v_scales=c.vs)
    for _ in range(4):
        c.dpool.copy_(fresh)
        c.dscales.copy_(fresh_s)
        kept_dev.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(kept_dev.cpu().numpy(), kept)
        assert np.array_equal(_bytes(c.dpool), _bytes(pool)) and np.array_equal(_bytes(c.dscales), _bytes(scales))
        torch.randn(1000, device="cuda").sum()


def test_pages_behind_four_gigabytes():
    stride = (1 << 31) + 64         # elements of 16 bits
    pool = torch.zeros(3 * stride, dtype=torch.bfloat16, device="cuda")
    k = pool.as_strided((3, 1, 16, 64), (stride, 1024, 64, 1))
    v = pool[4096:].as_strided((3, 1, 16, 64), (stride, 1024, 64, 1))
    x = torch.randn(2, 48, 64).to(torch.bfloat16).cuda()
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([48], dtype=torch.int32, device="cuda")
    h.paged_kv_append(x[:1], x[1:], k, v, table, lens)
    w = torch.rand(1, 48, device="cuda")
    kept = torch.zeros(1, 30, dtype=torch.int32, device="cuda")
    stay = F.chosen(w[0].double().cpu().numpy(), 48, 30, 3)
    h.paged_kv_evict(k, v, table, lens, w, w, kept, 3)
    a, b = torch.empty(1, 30, 64, dtype=torch.bfloat16, device="cuda"), torch.empty(1, 30, 64, dtype=torch.bfloat16, device="cuda")
    h.paged_kv_read(k, v, table, lens, a, b)
    assert kept[0].tolist() == stay.tolist()
    assert torch.equal(a[0], x[0][torch.from_numpy(stay).cuda()]) and torch.equal(b[0], x[1][torch.from_numpy(stay).cuda()])


# ---- PagedKVCache ---------------------------------------------------------------------

class Rows:
    """What a weighted PagedKVCache has to hold: rows by sequence and head, weights, in 64 bits."""

    def __init__(self, c, dtype):
        self.c, self.dtype = c, dtype
        self.rows = [[np.zeros((c.n_head_kv, 0, c.head)) for _ in range(c.n_batch)] for _ in (0, 1)]
        self.w = [np.zeros((c.n_head_kv, 0)) for _ in range(c.n_batch)]

    def append(self, k, v, counts):
        for mine, x in zip(self.rows, (k, v)):
            x = x.double().cpu().numpy().reshape(self.c.n_head_kv, self.c.n_batch, -1, self.c.head)
            x = F.values4(*F.quantised4(x)) if self.c.bits == 4 else P.quantised(x)[0] if self.c.bits == 8 else x
            for n, count in enumerate(counts):
                mine[n] = np.concatenate([mine[n], x[:, n, :count]], axis=1)
        for n, count in enumerate(counts):
            self.w[n] = np.concatenate([self.w[n], np.zeros((self.c.n_head_kv, count))], axis=1)

    def case(self):
        c = P.Case.__new__(P.Case)
        c.dtype, c.packed, c.head, c.heads, c.n_batch = self.dtype, self.c.packed, self.c.head, self.c.n_head_kv, self.c.n_batch
        c.lens = [x.shape[1] for x in self.w]
        c.rows = lambda n, which, count=None: (self.rows[which][n], np.ones(c.lens[n], bool))
        return c

    def check_attention(self, Q, lse, A, group, counts):
        want, want_l = P.attend(self.case(), Q.cpu(), Q.shape[1], group, True, counts)
        bound, bound_l = P.attend_bounds(self.case(), Q.cpu(), Q.shape[1], group, True, counts)
        dead = np.isneginf(want_l)
        got, got_l = A.double().cpu().numpy(), lse.double().cpu().numpy()
        assert np.array_equal(np.isneginf(got_l), dead) and np.all(np.abs(got - want) <= bound)
        assert np.all(np.abs(got_l - want_l)[~dead] <= bound_l[~dead])

    def observe(self, Q, lse, group, counts, decay):
        """The weights by the formula from the cache's own of before; then what the cache has."""
        after = self.c.weights.double().cpu().numpy().reshape(self.c.n_head_kv, self.c.n_batch, -1)
        for n, (total, bound) in enumerate(F.received(self.case(), Q.cpu(), lse.cpu(), Q.shape[1], group, True, counts)):
            old = float(np.float32(decay)) * self.w[n]
            want, length = old + total, total.shape[1]
            assert np.all(np.abs(after[:, n, :length] - want) <= bound + 2.0 ** -23 * np.abs(old) + 2.0 ** -24 * want)
            assert not after[:, n, length:].any()
            self.w[n] = after[:, n, :length].copy()

    def evict(self, kept, keep, recent):
        kept = kept.cpu().numpy().reshape(self.c.n_head_kv, self.c.n_batch, keep)
        for n in range(self.c.n_batch):
            length = self.w[n].shape[1]
            stay = [F.chosen(self.w[n][hd], length, keep, recent) for hd in range(self.c.n_head_kv)]
            for hd, rows in enumerate(stay):
                assert kept[hd, n].tolist() == rows.tolist() + [-1] * (keep - len(rows))
            for mine in self.rows:
                mine[n] = np.stack([mine[n][hd][rows] for hd, rows in enumerate(stay)])
            self.w[n] = np.stack([self.w[n][hd][rows] for hd, rows in enumerate(stay)])

    def check(self):
        assert self.c.lengths == [x.shape[1] for x in self.w] == self.c.lens.tolist()
        w = self.c.weights.double().cpu().numpy().reshape(self.c.n_head_kv, self.c.n_batch, -1)
        for n, mine in enumerate(self.w):
            assert np.array_equal(w[:, n, :mine.shape[1]], mine) and not w[:, n, mine.shape[1]:].any()
        for x, rows in zip(self.c.read(), self.rows):
            x = x.double().cpu().numpy().reshape(self.c.n_head_kv, self.c.n_batch, -1, self.c.head)
            for n, mine in enumerate(rows):
                assert np.array_equal(x[:, n, :mine.shape[1]], mine) and not x[:, n, mine.shape[1]:].any()


def _tiles(seed, c, rows, group, dtype):
    g = torch.Generator().manual_seed(seed)
    t = P.TORCH_DT[dtype]
    k, v = (torch.randn(c.n_head_kv * c.n_batch, rows, c.head, generator=g).to(t).cuda() for _ in range(2))
    Q = torch.randn(c.n_head_kv * group * c.n_batch, rows, c.head, generator=g).to(t).cuda()
    A = torch.full(Q.shape, float("nan"), dtype=t, device="cuda")
    return k, v, Q, torch.full(Q.shape[:2], float("nan"), device="cuda"), A


def _cache(dtype, bits, head, n_pages=24, n_batch=3, **kw):
    return PagedKVCache(n_pages, 16, n_batch, 200, 2, head, dtype=P.TORCH_DT[dtype], bits=bits if bits <= 8 else None,
                        weighted=True, **kw)


@pytest.mark.parametrize("dtype,bits", F.KINDS)
@pytest.mark.parametrize("head", [64, 128])
def test_a_served_batch_that_is_cut_down(dtype, bits, head):
    """Prompts, steps, a cut, steps, an end, another sequence on the same pages, a cut again."""
    print("serve", dtype, bits, head, flush=True)
    c = _cache(dtype, bits, head)
    mine, group = Rows(c, dtype), 2
    for i, (rows, counts, decay) in enumerate([(70, [70, 3, 0], 1.0), (1, None, 1.0), (40, [2, 40, 5], 0.5), ("evict", 33, 8),
                                               (1, None, 1.0), (9, [9, 0, 9], 0.0), ("release", 1, 0), (50, [0, 50, 1], 1.0),
                                               ("evict", 20, 20), ("evict", 20, 3), (1, None, 0.9), ("evict", 1, 0),
                                               (2, None, 1.0)]):
        if rows == "evict":
            keep, recent = counts, decay
            mine.evict(c.evict(keep, recent), keep, recent)
        elif rows == "release":
            c.release(counts)
            mine.w[counts] = mine.w[counts][:, :0]
            for x in mine.rows:
                x[counts] = x[counts][:, :0]
        else:
            k, v, Q, lse, A = _tiles(60 + i, c, rows, group, dtype)
            c.append_attend(k, v, Q, lse, A, group, new_rows=counts)
            mine.append(k, v, [rows] * 3 if counts is None else counts)
            mine.check_attention(Q, lse, A, group, counts)
            c.observe(Q, lse, group, new_rows=counts, decay=decay)
            mine.observe(Q, lse, group, counts, decay)
        mine.check()
        assert c.free_pages == 24 - sum(-(-n // 16) for n in c.lengths)
        held = [p for row in c.table.tolist() for p in row if p >= 0]
        assert len(set(held)) == len(held) == 24 - c.free_pages


def test_a_long_chunk_over_four_bits():
    """As many queries as go through the tile kernels, and their weights."""
    c = _cache("bf16", 4, 64, n_pages=40, n_batch=2)
    mine = Rows(c, "bf16")
    k, v, _, _, _ = _tiles(80, c, 30, 4, "bf16")
    c.append(k, v)
    mine.append(k, v, [30, 30])
    k, v, Q, lse, A = _tiles(81, c, 140, 4, "bf16")
    c.append_attend(k, v, Q, lse, A, 4)
    mine.append(k, v, [140] * 2)
    mine.check_attention(Q, lse, A, 4, None)
    c.observe(Q, lse, 4)
    mine.observe(Q, lse, 4, None, 1.0)
    mine.evict(c.evict(100, 16), 100, 16)
    mine.check()


def test_a_cache_on_a_stream_of_its_own():
    c, d = (_cache("bf16", 4, 128, n_batch=2) for _ in range(2))
    stream = torch.cuda.Stream()
    for i, counts in enumerate([[30, 7], [1, 30], None]):
        tiles = _tiles(90 + i, c, 30, 2, "bf16")
        other = [t.clone() for t in tiles]
        c.append_attend(*tiles, 2, new_rows=counts)
        c.observe(tiles[2], tiles[3], 2, new_rows=counts)
        stream.wait_stream(torch.cuda.current_stream())
        d.append_attend(*other, 2, new_rows=counts, stream=stream)
        d.observe(other[2], other[3], 2, new_rows=counts, stream=stream)
        a, b = c.evict(25, 5), d.evict(25, 5, stream=stream)
        if i == 1:
            c.release(0)
            d.release(0, stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(a, b) and c.lengths == d.lengths and torch.equal(c.weights, d.weights)
        for x, y in zip(tuple(tiles) + c.read(), tuple(other) + d.read(stream=stream)):
            torch.cuda.synchronize()
            assert torch.equal(x, y)


def test_what_a_cache_refuses():
    plain = PagedKVCache(4, 16, 1, 64, 1, 64)
    _, _, Q, lse, _ = _tiles(1, plain, 1, 1, "bf16")
    with pytest.raises(ValueError, match="without weights"):
        plain.observe(Q, lse, 1)
    with pytest.raises(ValueError, match="without weights"):
        plain.evict(8)
    c = PagedKVCache(4, 16, 1, 64, 1, 64, weighted=True)
    for keep, recent in ((0, 0), (-1, 0), (8, 9), (8, -1)):
        with pytest.raises(ValueError):
            c.evict(keep, recent)
    k, v, Q, lse, A = _tiles(2, c, 40, 1, "bf16")
    c.append_attend(k, v, Q, lse, A, 1)
    for decay in (-0.5, 1.5, float("nan")):
        with pytest.raises(h.SdpaError):
            c.observe(Q, lse, 1, decay=decay)
    with pytest.raises(ValueError):
        c.observe(Q, lse, 1, new_rows=[41])
    assert c.lengths == [40] and not c.weights.any()
