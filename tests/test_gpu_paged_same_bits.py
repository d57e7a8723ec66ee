"""Attention over a paged cache gives the same bits every time, in every form and way of sharing the keys out."""
import pytest
import torch

from nntile_amd import hip_sdpa as h

pytestmark = pytest.mark.gpu
KINDS = [(torch.bfloat16, False), (torch.float16, False), (torch.float32, False), (torch.bfloat16, True),
         (torch.float16, True)]


@pytest.mark.parametrize("dtype,packed", KINDS)
@pytest.mark.parametrize("head,q_seq,group", [(128, 1, 4), (64, 4, 8), (128, 16, 4), (64, 70, 3)])
@pytest.mark.parametrize("lens", [[1001], [4096] * 8, [16000, 17, 3000, 0, 900, 64, 7777, 1, 333, 12000],
                                  [100 + 37 * i % 900 for i in range(70)]])
def test_repeated(dtype, packed, head, q_seq, group, lens):
    n, heads, page_rows = len(lens), 4, 64
    pages = -(-max(lens) // page_rows)
    print("repeat", dtype, packed, head, q_seq, group, n, flush=True)
    g = torch.Generator(device="cuda").manual_seed(97)
    shape = (n * pages, 2, heads, page_rows, head)
    if packed:
        # (every code but the two NaN)
        pool = torch.randint(0, 127, shape, generator=g, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
        scales = torch.randint(115, 121, shape[:4], generator=g, device="cuda", dtype=torch.uint8)
        ks, vs = scales[:, 0], scales[:, 1]
    else:
        pool = torch.randn(shape, generator=g, device="cuda").to(dtype)
        ks = vs = None
    table = torch.randperm(n * pages, generator=g, device="cuda").to(torch.int32).view(n, pages)
    where = torch.tensor(lens, dtype=torch.int32, device="cuda")
    Q = torch.randn(heads * group * n, q_seq, head, generator=g, device="cuda").to(dtype)
    need = h.paged_workspace_bytes(Q, n, group)
    first = None
    for fill in [0, 255] + [None] * 10:
        ws = torch.empty(need, dtype=torch.uint8, device="cuda").fill_(fill) if fill is not None else ws
        lse = torch.full(Q.shape[:2], float("nan"), device="cuda")
        A = torch.full_like(Q, float("nan"))
        h.sdpa_fwd_paged(pool[:, 0], pool[:, 1], table, where, Q, lse, A, h.MASK_CAUSAL, group, ws, k_scales=ks,
                         v_scales=vs, flags=h.OVERWRITE)
        first = (A, lse) if first is None else first
        # (no NaN: every row is written)
        assert torch.equal(A, first[0]) and torch.equal(lse, first[1])
