"""Writing into pages and reading back as many rows as take the forms with several rows a thread, with and without a
padded batch, past the caches: bit for bit against the definition on the device."""
import pytest
import torch

from nntile_amd import hip_sdpa as h

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
KINDS = [("bf16", False), ("fp16", False), ("fp32", False), ("bf16", True), ("fp16", True)]
N_BATCH, HEADS = 3, 5


def _bits(t):
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def _rows_for(dtype, head, megabytes):
    """Rows of a call whose two tiles together are just past so much, an odd number of them."""
    row = head * DT[dtype].itemsize
    return (megabytes * 2 ** 20 // (2 * row * N_BATCH * HEADS) + 1) | 1


class Pool:
    """Keys and values as halves of one pool, pages in any order, every byte a pattern."""

    def __init__(self, seed, dtype, packed, head, page_rows, lens):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.dtype, self.packed, self.head, self.page_rows, self.lens = dtype, packed, head, page_rows, lens
        self.max_pages = -(-max(lens) // page_rows)
        n_pages = N_BATCH * self.max_pages + 2
        order = torch.randperm(n_pages, generator=self.g, device="cuda")
        self.table = order[:N_BATCH * self.max_pages].view(N_BATCH, self.max_pages).to(torch.int32).contiguous()
        held = torch.float8_e4m3fn if packed else DT[dtype]
        shape = (n_pages, 2, HEADS, page_rows, head)
        if packed:
            # (every code but the two NaN)
            self.pool = torch.randint(0, 127, shape, generator=self.g, device="cuda", dtype=torch.uint8).view(held)
            self.scales = torch.randint(117, 130, shape[:4], generator=self.g, device="cuda", dtype=torch.uint8)
        else:
            self.pool = torch.randn(shape, generator=self.g, device="cuda").to(held)
            self.scales = None
        self.dlens = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def args(self):
        s = (self.scales[:, 0], self.scales[:, 1]) if self.packed else (None, None)
        return (self.pool[:, 0], self.pool[:, 1]), (self.table, self.dlens), s

    def at(self, pos):
        """page and place in it of rows `pos` [N_BATCH, rows]."""
        page = torch.gather(self.table.long(), 1, (pos // self.page_rows).clamp(0, self.max_pages - 1))
        return page, pos % self.page_rows


def _tile(pool, rows):
    """Rows of all sizes behind each other: random powers of two, zeros, infinities and NaN."""
    x = torch.randn(HEADS * N_BATCH, rows, pool.head, generator=pool.g, device="cuda")
    power = torch.randint(-14, 12, x.shape[:2], generator=pool.g, device="cuda")
    x = torch.ldexp(x, power[..., None])
    kind = torch.randint(0, 64, x.shape[:2], generator=pool.g, device="cuda")
    x[kind == 0] = 0.0
    x[..., 7] = torch.where(kind == 1, float("inf"), x[..., 7])
    x[..., 9] = torch.where(kind == 2, float("nan"), x[..., 9])
    return x.to(DT[pool.dtype])


def _power(byte):
    """2^(byte - 127) (torch.ldexp on the device is off by a rounding)."""
    return (byte.int() << 23).view(torch.float32)


def _quantised(x):
    """Codes and scale bytes of rows [.., head]; a row that is not finite is NaN."""
    f = x.float()
    a = f.abs().amax(dim=-1)
    bad = ~torch.isfinite(f).all(dim=-1)
    mantissa, exponent = torch.frexp(torch.where(bad, 1.0, a))
    k = torch.where(mantissa > 0.875, exponent - 8, exponent - 9).clamp(min=-126)
    k = torch.where(mantissa == 0, -126, k)
    codes = (f / _power(k + 127)[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
    codes = torch.where(bad[..., None], 127, codes)
    return codes.to(torch.uint8).view(torch.float8_e4m3fn), torch.where(bad, 127, k + 127).to(torch.uint8)


@pytest.mark.parametrize("dtype,packed", KINDS)
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("megabytes", [15, 17])
def test_append(dtype, packed, head, padded, megabytes):
    rows = _rows_for(dtype, head, megabytes)
    new_rows = [rows, 0, rows // 2 - 3] if padded else [rows] * N_BATCH
    lens = [rows + 21, rows, rows + 5]
    print("append", dtype, packed, head, rows, new_rows, flush=True)
    p = Pool(80, dtype, packed, head, 64, lens)
    new = _tile(p, rows), _tile(p, rows)
    want, want_s = p.pool.clone(), p.scales.clone() if packed else None
    r = torch.arange(rows, device="cuda")[None, :]
    given = torch.tensor(new_rows, device="cuda")[:, None]
    page, place = p.at(torch.tensor(lens, device="cuda")[:, None] - given + r)
    for which, x in enumerate(new):
        x = x.view(HEADS, N_BATCH, rows, head)
        for n in range(N_BATCH):
            to = page[n, :new_rows[n]], place[n, :new_rows[n]]
            for hd in range(HEADS):
                if packed:
                    codes, byte = _quantised(x[hd, n, :new_rows[n]])
                    want.view(torch.uint8)[to[0], which, hd, to[1]] = codes.view(torch.uint8)
                    want_s[to[0], which, hd, to[1]] = byte
                else:
                    want[to[0], which, hd, to[1]] = x[hd, n, :new_rows[n]]
    pages, where, scales = p.args()
    nr = torch.tensor(new_rows, dtype=torch.int32, device="cuda") if padded else None
    h.paged_kv_append(*new, *pages, *where, *scales, new_rows=nr)
    torch.cuda.synchronize()
    assert torch.equal(_bits(p.pool), _bits(want))
    if packed:
        assert torch.equal(p.scales, want_s)


@pytest.mark.parametrize("dtype,packed", KINDS)
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("megabytes", [15, 17, 127, 129])
def test_read(dtype, packed, head, megabytes):
    rows, first = _rows_for(dtype, head, megabytes), 19
    lens = [first + rows, first + rows // 3, first + rows + 40]
    print("read", dtype, packed, head, rows, lens, flush=True)
    p = Pool(81, dtype, packed, head, 32, lens)
    p.table[1, 1] = -1                      # no page: zeros
    pages, where, scales = p.args()
    out = [torch.full((HEADS * N_BATCH, rows, head), 7.0, dtype=DT[dtype], device="cuda") for _ in range(2)]
    h.paged_kv_read(*pages, *where, *out, first=first, k_scales=scales[0], v_scales=scales[1])
    torch.cuda.synchronize()
    pos = first + torch.arange(rows, device="cuda")[None, :].expand(N_BATCH, rows)
    page, place = p.at(pos)
    there = (pos < p.dlens[:, None]) & (page >= 0)
    for which in range(2):
        got = out[which].view(HEADS, N_BATCH, rows, head)
        for n in range(N_BATCH):
            for hd in range(HEADS):
                of = page[n].clamp(min=0), place[n]
                if packed:
                    x = p.pool.view(torch.uint8)[of[0], which, hd, of[1]].view(torch.float8_e4m3fn).float()
                    x = x * _power(p.scales[of[0], which, hd, of[1]])[:, None]
                else:
                    x = p.pool[of[0], which, hd, of[1]]
                # (these codes times powers of two are exact in either type)
                want = torch.where(there[n][:, None], x, 0.0).to(DT[dtype])
                assert torch.equal(_bits(got[hd, n]), _bits(want))
