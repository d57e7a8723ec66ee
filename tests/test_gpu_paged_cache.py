"""Writing into the pages of a cache and reading them back, against the definition in 64 bits."""
import numpy as np
import pytest
import torch

from nntile_amd import hip_sdpa as h
from . import paged_helpers as P

pytestmark = pytest.mark.gpu
KINDS = [("bf16", False), ("fp16", False), ("fp32", False), ("bf16", True), ("fp16", True)]


def _rows(seed, entries, rows, head, dtype, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return tuple((scale * torch.randn(entries, rows, head, generator=g)).to(P.TORCH_DT[dtype]) for _ in range(2))


def _bits(t):
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def _append_want(c, new, rows, new_rows=None):
    """Pool and scales as they are after the call (CPU)."""
    pool, scales = c.pool.clone(), c.scales.clone()
    for which, x in enumerate(new):
        x = x.reshape(c.heads, c.n_batch, rows, c.head)
        for n in range(c.n_batch):
            given = rows if new_rows is None else max(0, min(rows, new_rows[n]))
            length = max(0, min(c.lens[n], c.max_pages * c.page_rows))
            for r in range(given):
                pos = length - given + r
                page = int(c.table[n, pos // c.page_rows]) if pos >= 0 else -1
                if not 0 <= page < c.n_pages:
                    continue
                row = x[:, n, r]
                if c.packed:
                    value, byte = P.quantised(row.double().numpy())
                    code = value / np.exp2(byte.astype(np.float64) - 127)[:, None]
                    pool[page, which, :, pos % c.page_rows] = torch.from_numpy(code).float().to(torch.float8_e4m3fn)
                    scales[page, which, :, pos % c.page_rows] = torch.from_numpy(byte)
                else:
                    pool[page, which, :, pos % c.page_rows] = row
    return pool, scales


def _check_append(c, new, rows, new_rows=None):
    print("append", c.dtype, c.packed, c.n_batch, c.heads, c.head, c.page_rows, c.lens, rows, new_rows, flush=True)
    c.device()
    nr = None if new_rows is None else torch.tensor(new_rows, dtype=torch.int32).cuda()
    k, v = (x.cuda() for x in new)
    h.paged_kv_append(k, v, c.k, c.v, c.dtable, c.dlens, c.ks, c.vs, new_rows=nr)
    torch.cuda.synchronize()
    pool, scales = _append_want(c, new, rows, new_rows)
    nan = torch.isnan(pool.float())
    for which, (got, got_s) in enumerate(((c.k, c.ks), (c.v, c.vs))):
        # bit for bit, but for which NaN it is
        got = got.cpu()
        assert torch.equal(torch.isnan(got.float()), nan[:, which])
        live = ~nan[:, which]
        assert torch.equal(_bits(got)[live], _bits(pool[:, which].contiguous())[live])
        if c.packed:
            assert torch.equal(got_s.cpu(), scales[:, which])


@pytest.mark.parametrize("dtype,packed", KINDS)
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("n_batch,heads,page_rows,lens,rows,spread", [
    (1, 1, 16, [1], 1, 0), (3, 2, 16, [17, 40, 33], 5, 1), (2, 3, 64, [130, 64], 64, 0),
    (4, 1, 32, [33, 95, 32, 64], 31, 1)])
def test_append(dtype, packed, head, n_batch, heads, page_rows, lens, rows, spread):
    c = P.Case(7, dtype, packed, n_batch, heads, head, page_rows, lens, spread=spread)
    _check_append(c, _rows(8, n_batch * heads, rows, head, dtype), rows)


@pytest.mark.parametrize("dtype,packed", KINDS)
def test_append_padded_missing_pages_and_lengths_past_the_table(dtype, packed):
    # counts of all kinds; a sequence shorter than what it brings; one without a page; a length
    # past the table, which stands for the table's end; a length below 0
    c = P.Case(9, dtype, packed, 7, 2, 64, 16, [20, 3, 33, 48, 16, 40, 0], max_pages=3)
    c.table[2, 2] = -1
    c.table[3, 2] = c.n_pages
    c.table[5, 2] = 2 ** 31 - 1
    c.lens[4] = 1000
    c.table[4] = torch.tensor([int(c.table[4, 0]), c.n_pages - 1, c.n_pages - 2])
    held = {int(p) for p in c.table.reshape(-1)}
    spare = [p for p in range(c.n_pages) if p not in held]
    c.table[4, 2] = spare[0] if spare else c.table[4, 2]
    c.lens[6] = -5
    _check_append(c, _rows(10, 14, 6, 64, dtype), 6, [6, 6, 2, 7, 3, 0, -1])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_scales_at_the_borders(dtype):
    """Rows whose largest value is next to 448 times a power of two, tiny, zero, the type's
    largest; ties between two codes; infinities and NaN."""
    t = P.TORCH_DT[dtype]
    top = torch.finfo(t).max
    least = torch.finfo(t).smallest_normal * torch.finfo(t).eps
    eps = torch.finfo(t).eps
    rows = []
    for m in (448.0, 448.0 * (1 + eps), 448.0 * (1 - eps), 1.75, 1.0, top, top / 2, least, 3 * least, 0.0,
              float("inf"), float("nan"), 2.0 ** -14, 224.0, 7.0):
        x = torch.linspace(-1.0, 1.0, 64, dtype=torch.float64) * (m if np.isfinite(m) else 1.0)
        x[0] = m
        x[1], x[2], x[3] = 0.0, m * 17 / 32, -m * 17 / 256        # halfway between codes where m is one
        rows.append(x)
    x = torch.stack(rows).to(t)[None]
    n = x.shape[1]
    c = P.Case(11, dtype, True, 1, 1, 64, 16, [n])
    _check_append(c, (x, x.flip(1).contiguous()), n)


@pytest.mark.parametrize("dtype,packed", KINDS)
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("lens,page_rows,first,rows,spread", [
    ([1], 16, 0, 1, 0), ([40, 0, 33], 16, 7, 30, 1), ([130, 64], 64, 60, 70, 0), ([5, 200], 128, 300, 4, 1)])
def test_read(dtype, packed, head, lens, page_rows, first, rows, spread):
    c = P.Case(12, dtype, packed, len(lens), 2, head, page_rows, lens, spread=spread)
    if len(lens) > 2:
        c.table[2, 1] = -7
    print("read", dtype, packed, head, lens, page_rows, first, rows, flush=True)
    c.device()
    out = [torch.full((2 * len(lens), rows, head), 7.0, dtype=P.TORCH_DT[dtype], device="cuda") for _ in range(2)]
    h.paged_kv_read(c.k, c.v, c.dtable, c.dlens, *out, first=first, k_scales=c.ks, v_scales=c.vs)
    torch.cuda.synchronize()
    for which in range(2):
        want = np.zeros((2, len(lens), rows, head))
        for n in range(len(lens)):
            x, _ = c.rows(n, which)
            part = x[:, first:first + rows]
            want[:, n, :part.shape[1]] = part
        # (codes times powers of two are exact in bf16 and, of this size, in fp16)
        assert np.array_equal(out[which].double().cpu().numpy(), want.reshape(-1, rows, head))


def test_the_largest_fp16_value_reads_back_finite():
    x = torch.full((1, 1, 64), 65504.0, dtype=torch.float16)
    x[0, 0, 1] = -65504.0
    c = P.Case(13, "fp16", True, 1, 1, 64, 16, [1]).device()
    xd = x.cuda()
    h.paged_kv_append(xd, xd, c.k, c.v, c.dtable, c.dlens, c.ks, c.vs)
    out = [torch.empty_like(xd) for _ in range(2)]
    h.paged_kv_read(c.k, c.v, c.dtable, c.dlens, *out, k_scales=c.ks, v_scales=c.vs)
    # (65504 is nearest to the code of 65536, past fp16: its largest value instead)
    assert torch.equal(out[0].cpu(), x) and torch.equal(out[1].cpu(), x)


@pytest.mark.parametrize("dtype,packed", [("bf16", False), ("bf16", True)])
def test_offsets_past_32_bits(dtype, packed):
    """A pool of more than 2^32 elements: pages behind that are written and read there."""
    page_rows, head, heads = 1024, 128, 8
    per_page = page_rows * head * heads
    n_pages = 2 ** 32 // per_page + 5
    held = torch.float8_e4m3fn if packed else torch.bfloat16
    pools = [torch.empty((n_pages, heads, page_rows, head), dtype=held, device="cuda") for _ in range(2)]
    scales = [torch.zeros((n_pages, heads, page_rows), dtype=torch.uint8, device="cuda") for _ in range(2)] \
        if packed else [None, None]
    table = torch.tensor([[n_pages - 1], [n_pages // 2]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([1000, 40], dtype=torch.int32, device="cuda")
    new = [x.cuda() for x in _rows(14, 2 * heads, 40, head, dtype)]
    h.paged_kv_append(*new, *pools, table, lens, *scales)
    out = [torch.empty_like(x) for x in new]
    h.paged_kv_read(*pools, table, lens, *out, first=960, k_scales=scales[0], v_scales=scales[1])
    torch.cuda.synchronize()
    for which in range(2):
        got = out[which].reshape(heads, 2, 40, head)
        want = new[which].reshape(heads, 2, 40, head)
        assert torch.all(got[:, 1] == 0)
        x = pools[which][n_pages - 1, :, 960:1000].to(torch.bfloat16).float()
        if packed:
            x = torch.ldexp(x, scales[which][n_pages - 1, :, 960:1000].int()[..., None] - 127)
        assert torch.equal(got[:, 0].float(), x)
        # e4m3 keeps four bits: half a step of them
        assert float((got[:, 0].float() - want[:, 0].float()).abs().max()) <= (2.0 ** -4 * 8 if packed else 0)
