"""The paged cache as a program uses it: rotation, append and attention behind each other, captured and
replayed, on streams of their own, and `PagedKVCache`."""
import numpy as np
import pytest
import torch

from nntile_amd import hip_sdpa as h
from nntile_amd.kv_cache import PagedKVCache
from . import paged_helpers as P

pytestmark = pytest.mark.gpu
KINDS = [("bf16", False), ("fp16", False), ("fp32", False), ("bf16", True), ("fp16", True)]


class Server:
    """A few generation steps of three sequences through rope_axes, paged_kv_append and
    sdpa_fwd_paged, on tensors that stay where they are."""

    def __init__(self, dtype, packed, q_seq, group, head, ws=None, seed=50, n_batch=3, heads=2, max_pages=40):
        t = P.TORCH_DT[dtype]
        self.q_seq, self.group, self.head, self.n_batch, self.heads = q_seq, group, head, n_batch, heads
        g = torch.Generator().manual_seed(seed)
        n_pages = n_batch * max_pages
        shape = (n_pages, 2, heads, 16, head)
        self.pool = torch.zeros(shape, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) if packed \
            else torch.zeros(shape, dtype=t, device="cuda")
        scales = torch.ones(shape[:4], dtype=torch.uint8, device="cuda") if packed else None
        self.k_scales, self.v_scales = (scales[:, 0], scales[:, 1]) if packed else (None, None)
        self.table = torch.randperm(n_pages, generator=g).to(torch.int32).view(n_batch, max_pages).cuda()
        self.lens = torch.zeros(n_batch, dtype=torch.int32, device="cuda")
        self.step_rows = torch.tensor([q_seq, max(1, q_seq - 1), q_seq][:n_batch], dtype=torch.int32).cuda()
        self.positions = torch.zeros(3, n_batch, q_seq, dtype=torch.int64, device="cuda")
        self.freqs, self.axes = h.rope_axes_freqs(head, [head // 8, head // 8, head // 4])
        self.q = torch.empty(heads * group * n_batch, q_seq, head, dtype=t, device="cuda")
        self.k = torch.empty(heads * n_batch, q_seq, head, dtype=t, device="cuda")
        self.v = torch.empty_like(self.k)
        self.q_rot, self.k_rot = torch.empty_like(self.q), torch.empty_like(self.k)
        self.A = torch.empty_like(self.q)
        self.lse = torch.empty(self.q.shape[:2], dtype=torch.float32, device="cuda")
        need = h.paged_workspace_bytes(self.q, n_batch, group)
        self.ws = torch.empty(need, dtype=torch.uint8, device="cuda").fill_(0x5a) if ws is None else ws

    def step(self, stream=None):
        h.rope_axes(self.positions, self.freqs, self.axes, self.q, self.q_rot, self.k, self.k_rot, stream=stream)
        h.paged_kv_append(self.k_rot, self.v, self.pool[:, 0], self.pool[:, 1], self.table, self.lens,
                          self.k_scales, self.v_scales, new_rows=self.step_rows, stream=stream)
        h.sdpa_fwd_paged(self.pool[:, 0], self.pool[:, 1], self.table, self.lens, self.q_rot, self.lse, self.A,
                         h.MASK_CAUSAL, self.group, self.ws, k_scales=self.k_scales, v_scales=self.v_scales,
                         new_rows=self.step_rows, flags=h.OVERWRITE, stream=stream)

    def feed(self, i, seed=51):
        """Tokens of step i, at the place where a captured step reads them."""
        g = torch.Generator().manual_seed(seed + i)
        for t in (self.q, self.k, self.v):
            t.copy_(torch.randn(t.shape, generator=g))
        at = self.lens.long()[:, None] + torch.arange(self.q_seq, device="cuda")
        self.positions.copy_(at * torch.tensor([1, 2, 5], device="cuda")[:, None, None])
        self.lens += self.step_rows

    def result(self):
        return self.A.clone(), self.lse.clone()


def _rotated(x, s):
    """x [heads * n_batch, q_seq, head] turned in 64 bits."""
    x = x.double().cpu().numpy()
    pos = s.positions.cpu().numpy()
    f, ax = s.freqs.cpu().numpy(), s.axes.cpu().numpy()
    ang = np.stack([pos[ax, e % s.n_batch].T * f for e in range(x.shape[0])])
    a, b = x[..., 0::2], x[..., 1::2]
    y = np.empty_like(x)
    y[..., 0::2] = a * np.cos(ang) - b * np.sin(ang)
    y[..., 1::2] = a * np.sin(ang) + b * np.cos(ang)
    return y


@pytest.mark.parametrize("dtype,packed", KINDS)
@pytest.mark.parametrize("q_seq,group,head", [(1, 4, 64), (5, 3, 128), (12, 4, 64)])
def test_steps_of_generation(dtype, packed, q_seq, group, head):
    """The attention of every step, of the rows that the steps before wrote, against the formula; the
    rows of the pages against the rotation."""
    print("steps", dtype, packed, q_seq, group, head, flush=True)
    s = Server(dtype, packed, q_seq, group, head)
    c = P.Case(1, dtype, packed, 3, 2, head, 16, [0, 0, 0])
    c.n_pages, c.max_pages, c.table = s.pool.shape[0], s.table.shape[1], s.table.cpu()
    u = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}[dtype]
    for i in range(6):
        s.feed(i)
        s.step()
        torch.cuda.synchronize()
        c.pool = s.pool.cpu()
        if packed:
            c.scales = torch.stack([s.k_scales.cpu(), s.v_scales.cpu()], dim=1)
        c.lens = s.lens.tolist()
        given = s.step_rows.tolist()
        # the rotation's outputs: one rounding, and a few of fp32 sines
        turned = _rotated(s.k, s)
        size = np.abs(s.k.double().cpu().numpy())
        pair = np.repeat(size[..., 0::2] + size[..., 1::2], 2, axis=-1)
        assert np.all(np.abs(s.k_rot.double().cpu().numpy() - turned) <= u * np.abs(turned) + 2.0 ** -21 * pair
                      + (2.0 ** -25 if dtype == "fp16" else 0))
        # its rows in the pages: as they are, or as the definition of an 8-bit row has them
        new = s.k_rot.double().cpu().numpy().reshape(2, 3, q_seq, head)
        want_rows = P.quantised(new)[0] if packed else new
        for n in range(3):
            rows, _ = c.rows(n, 0)
            first = c.lens[n] - given[n]
            assert np.array_equal(rows[:, first:], want_rows[:, n, :given[n]])
        q = s.q_rot.cpu()
        want, want_l = P.attend(c, q, q_seq, group, True, given)
        bound, bound_l = P.attend_bounds(c, q, q_seq, group, True, given)
        dead = np.isneginf(want_l)
        A, lse = s.A.double().cpu().numpy(), s.lse.double().cpu().numpy()
        assert np.all(np.abs(A - want) <= bound) and np.array_equal(np.isneginf(lse), dead)
        assert np.all(np.abs(lse - want_l)[~dead] <= bound_l[~dead])


@pytest.mark.parametrize("dtype,packed", KINDS)
def test_a_captured_step_replayed(dtype, packed):
    """One captured step, replayed while the lengths grow, with eager work in between, bit for bit
    the eager steps."""
    eager, graphed = (Server(dtype, packed, 2, 4, 64) for _ in range(2))
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    for i in range(9):
        eager.feed(i)
        eager.step()
        graphed.feed(i)
        if i == 2:
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, stream=side):
                graphed.step()
            torch.cuda.synchronize()
        if i < 2:
            graphed.step()
        else:
            graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager.result(), graphed.result()):
            assert torch.equal(a, b)
        torch.randn(1000, device="cuda").sum()
    assert torch.equal(eager.pool.view(torch.uint8), graphed.pool.view(torch.uint8))


def test_graphs_of_several_shapes_on_one_workspace():
    """Two captured steps of other shapes, types and numbers of shares, replayed in turn on one
    workspace that an eager call uses as well."""
    ws = torch.full((64 << 20,), 0x33, dtype=torch.uint8, device="cuda")
    kinds = [("bf16", False, 1, 4, 128), ("fp16", True, 12, 3, 64), ("fp32", False, 5, 4, 64)]
    shared = [Server(*k, ws=ws) for k in kinds]
    alone = [Server(*k) for k in kinds]
    graphs = []
    for s in shared[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.step()
        graphs.append(g)
    torch.cuda.synchronize()
    for i in range(6):
        for j, (a, b) in enumerate(zip(shared, alone)):
            a.feed(i)
            b.feed(i)
            graphs[j].replay() if j < 2 else a.step()
            b.step()
        torch.cuda.synchronize()
        for a, b in zip(shared, alone):
            for x, y in zip(a.result(), b.result()):
                assert torch.equal(x, y)


@pytest.mark.parametrize("packed", [False, True])
def test_steps_on_two_streams(packed):
    """Two batches at once, each on a stream of its own that is not the current one."""
    kinds = [("bf16", packed, 1, 4, 128), ("bf16", packed, 6, 4, 128)]
    want = [Server(*k) for k in kinds]
    servers = [Server(*k) for k in kinds]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(5):
        for s in want:
            s.feed(i)
            s.step()
        for s, stream in zip(servers, streams):
            with torch.cuda.stream(stream):
                stream.wait_stream(torch.cuda.default_stream())
                s.feed(i)
            s.step(stream=stream)
        for stream in streams:
            torch.cuda.current_stream().wait_stream(stream)
        for a, b in zip(want, servers):
            for x, y in zip(a.result(), b.result()):
                assert torch.equal(x, y)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_rotation_in_place(dtype):
    a, b = Server(dtype, False, 7, 3, 64), Server(dtype, False, 7, 3, 64)
    a.feed(3)
    b.feed(3)
    h.rope_axes(a.positions, a.freqs, a.axes, a.q, a.q_rot, a.k, a.k_rot)
    h.rope_axes(b.positions, b.freqs, b.axes, b.q, b.q, b.k, b.k)
    torch.cuda.synchronize()
    assert torch.equal(a.q_rot, b.q) and torch.equal(a.k_rot, b.k)


# ---- PagedKVCache ---------------------------------------------------------------------

class Rows:
    """What a PagedKVCache has to hold, in 64 bits, and the formula over it."""

    def __init__(self, cache, dtype, packed):
        self.c, self.dtype, self.packed = cache, dtype, packed
        self.k = [np.zeros((cache.n_head_kv, 0, cache.head)) for _ in range(cache.n_batch)]
        self.v = [x.copy() for x in self.k]

    def append(self, k, v, counts):
        for mine, x in ((self.k, k), (self.v, v)):
            x = x.double().cpu().numpy().reshape(self.c.n_head_kv, self.c.n_batch, -1, self.c.head)
            x = P.quantised(x)[0] if self.packed else x
            for n, count in enumerate(counts):
                mine[n] = np.concatenate([mine[n], x[:, n, :count]], axis=1)

    def case(self):
        """The same as a Case of one page a sequence."""
        c = P.Case.__new__(P.Case)
        c.dtype, c.packed, c.head, c.heads, c.n_batch = self.dtype, self.packed, self.c.head, self.c.n_head_kv, self.c.n_batch
        c.lens = [x.shape[1] for x in self.k]
        c.rows = lambda n, which, count=None: ((self.v if which else self.k)[n], np.ones(c.lens[n], bool))
        return c

    def check(self, Q, lse, A, group, causal, counts=None):
        want, want_l = P.attend(self.case(), Q.cpu(), Q.shape[1], group, causal, counts)
        bound, bound_l = P.attend_bounds(self.case(), Q.cpu(), Q.shape[1], group, causal, counts)
        got, got_l = A.double().cpu().numpy(), lse.double().cpu().numpy()
        dead = np.isneginf(want_l)
        assert np.array_equal(np.isneginf(got_l), dead) and np.all(np.abs(got - want) <= bound)
        assert np.all(np.abs(got_l - want_l)[~dead] <= bound_l[~dead])
        k, v = self.c.read()
        assert torch.equal(k, self.c.k_partial) and torch.equal(v, self.c.v_partial)
        for x, mine in ((k, self.k), (v, self.v)):
            x = x.double().cpu().numpy().reshape(self.c.n_head_kv, self.c.n_batch, -1, self.c.head)
            for n, rows in enumerate(mine):
                assert np.array_equal(x[:, n, :rows.shape[1]], rows) and not x[:, n, rows.shape[1]:].any()


def _tiles(seed, c, rows, group, dtype):
    g = torch.Generator().manual_seed(seed)
    t = P.TORCH_DT[dtype]
    k, v = (torch.randn(c.n_head_kv * c.n_batch, rows, c.head, generator=g).to(t).cuda() for _ in range(2))
    Q = torch.randn(c.n_head_kv * group * c.n_batch, rows, c.head, generator=g).to(t).cuda()
    A = torch.full(Q.shape, float("nan"), dtype=t, device="cuda")
    return k, v, Q, torch.full(Q.shape[:2], float("nan"), device="cuda"), A


@pytest.mark.parametrize("dtype,packed", KINDS)
@pytest.mark.parametrize("head", [64, 128])
def test_a_served_batch(dtype, packed, head):
    """Sequences of lengths of their own grow, end, and others take their pages."""
    print("serve", dtype, packed, head, flush=True)
    c = PagedKVCache(24, 16, 3, 200, 2, head, dtype=P.TORCH_DT[dtype], packed=packed)
    mine, group = Rows(c, dtype, packed), 2
    for i, (rows, counts) in enumerate([(70, [70, 3, 0]), (1, None), (5, [2, 5, 5]), (40, [0, 40, 17]), (1, None),
                                        (-1, None), (33, [0, 33, 0]), (1, [1, 0, 1])]):
        if rows < 0:
            c.release(1)
            mine.k[1], mine.v[1] = mine.k[1][:, :0], mine.v[1][:, :0]
            assert c.lengths[1] == 0
            continue
        k, v, Q, lse, A = _tiles(60 + i, c, rows, group, dtype)
        c.append_attend(k, v, Q, lse, A, group, new_rows=counts)
        mine.append(k, v, [rows] * 3 if counts is None else counts)
        assert c.lengths == [x.shape[1] for x in mine.k] == c.lens.tolist()
        assert c.free_pages == 24 - sum(-(-n // 16) for n in c.lengths)
        mine.check(Q, lse, A, group, True, counts)


@pytest.mark.parametrize("dtype,packed", KINDS)
def test_a_refused_append_changes_nothing(dtype, packed):
    c = PagedKVCache(6, 16, 2, 80, 1, 64, dtype=P.TORCH_DT[dtype], packed=packed)        # 5 in use below
    mine = Rows(c, dtype, packed)
    k, v, Q, lse, A = _tiles(70, c, 40, 1, dtype)
    c.append(k, v, new_rows=[40, 30])
    mine.append(k, v, [40, 30])
    before = (c.free_pages, c.lens.tolist(), c.table.tolist())

    def unchanged():
        assert (c.free_pages, c.lens.tolist(), c.table.tolist()) == before and c.lengths == [40, 30]

    long = _tiles(71, c, 60, 1, dtype)
    with pytest.raises(h.SdpaError, match="sequence 0: 100 rows, max: 80"):
        c.append(long[0], long[1])
    unchanged()
    with pytest.raises(h.SdpaError, match="2 pages wanted, 1 free"):
        c.append(k, v, new_rows=[9, 3])         # 49 and 33 rows: a page more each, one is left
    unchanged()
    for bad in ([41, 0], [-1, 0], [1], [1, 1, 1]):
        with pytest.raises(ValueError):
            c.append(k, v, new_rows=bad)
    unchanged()
    off = torch.zeros(k.numel() + 1, dtype=k.dtype, device="cuda")[1:].view(k.shape)
    for tiles in ((off, v), (k, off), (k.transpose(0, 1), v), (k, v[:, :-1].contiguous()), (k, v.cpu())):
        with pytest.raises(ValueError):
            c.append(*tiles, new_rows=[1, 1])
    unchanged()
    c.attend(Q, lse, A, 1, new_rows=[40, 30])
    mine.check(Q, lse, A, 1, True, [40, 30])


@pytest.mark.parametrize("dtype,packed", KINDS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("rows", [127, 128])
def test_long_chunks_of_equal_lengths(dtype, packed, causal, rows):
    """Four query heads times 128 tokens are the rows from which the pages are read back; behind a
    prefix that ends inside a page."""
    c = PagedKVCache(40, 16, 2, 300, 2, 64, dtype=P.TORCH_DT[dtype], packed=packed)
    mine = Rows(c, dtype, packed)
    k, v, _, _, _ = _tiles(80, c, 37, 4, dtype)
    c.append(k, v)
    mine.append(k, v, [37, 37])
    k, v, Q, lse, A = _tiles(81, c, rows, 4, dtype)
    c.append_attend(k, v, Q, lse, A, 4, causal=causal)
    mine.append(k, v, [rows] * 2)
    mine.check(Q, lse, A, 4, causal)


def test_a_cache_on_a_stream_of_its_own():
    c, d = (PagedKVCache(24, 16, 2, 200, 2, 64) for _ in range(2))
    stream = torch.cuda.Stream()
    for i, counts in enumerate([[30, 7], [1, 30], None]):
        tiles = _tiles(90 + i, c, 30, 2, "bf16")
        other = [t.clone() for t in tiles]
        c.append_attend(*tiles, 2, new_rows=counts)
        stream.wait_stream(torch.cuda.current_stream())
        d.append_attend(*other, 2, new_rows=counts, stream=stream)
        if i == 1:
            c.release(0)
            d.release(0, stream=stream)
        k, v = d.read(stream=stream)
        torch.cuda.current_stream().wait_stream(stream)
        for a, b in zip(tiles, other):
            assert torch.equal(a, b)
        for a, b in zip(c.read(), (k, v)):
            assert torch.equal(a, b)
