"""Calls of 2^32 threads and more: a launch has less in one direction, and runs the rest of a larger one without an
error only if its workgroups are numbered through two."""
import math

import pytest
import torch

from nntile_amd import hip_sdpa as h

pytestmark = pytest.mark.gpu


def _spots(total):
    """Four elements at the front, around 2^31 and 2^32, and at the end."""
    return [0, 2 ** 31 - 2, 2 ** 32 - 2, total - 4]


def test_rope_by_single_pairs():
    m, n = 3, 2 ** 32 // 3 + 1000           # (rows of no whole 16 bytes)
    print("rope", m, n, flush=True)
    src = torch.zeros(n, m, 2, dtype=torch.bfloat16, device="cuda")
    dst = torch.full_like(src, 7.0)
    sin, cos = (torch.tensor(x).to(torch.bfloat16).cuda() for x in ([0.5, 0.25, 0.0], [0.5, 1.0, -1.0]))
    pairs, out = src.view(-1, 2), dst.view(-1, 2)
    for at in _spots(m * n):
        pairs[at:at + 4] = torch.tensor([1.0, 2.0])
    h.rope(sin, cos, src, dst)
    torch.cuda.synchronize()
    for at in _spots(m * n):
        i = torch.arange(at, at + 4) % m
        s, c = sin.cpu().float()[i], cos.cpu().float()[i]
        assert torch.equal(out[at:at + 4].cpu().float(), torch.stack((c - 2 * s, s + 2 * c), dim=1))
    assert not out[2 ** 31 + 4:2 ** 32 - 4:1000003].any() and not out[2 ** 32 + 4:-4:101].any()


def test_kv_cache_append_by_single_values():
    entries, rows, head = 2, 2 ** 31 // 5 + 1000, 5
    print("append", entries, rows, head, flush=True)
    new = torch.zeros(entries, rows, head, dtype=torch.bfloat16, device="cuda")
    flat = new.view(-1)
    for at in _spots(flat.numel()):
        flat[at:at + 4] = torch.tensor([1.0, 2.0, 3.0, 4.0])
    caches = [torch.full((entries, rows + 3, head), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    h.kv_cache_append(new, new, *caches, 2)
    torch.cuda.synchronize()
    for c in caches:
        assert torch.all(c[:, :2] == 7) and torch.all(c[:, -1] == 7)
        for e in range(entries):
            for at in range(0, rows, 1 << 27):
                assert torch.equal(c[e, 2 + at:2 + min(at + (1 << 27), rows)], new[e, at:at + (1 << 27)])


def test_accumulate_by_single_rows():
    batch, seq, head = 2, 2 ** 31 + 1000, 1
    print("accumulate", batch, seq, head, flush=True)
    src, dst = (torch.zeros(batch, seq, head, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    src_lse, dst_lse = (torch.zeros(batch, seq, device="cuda") for _ in range(2))
    for at in _spots(src.numel()):
        src.view(-1)[at:at + 4] = torch.tensor([1.0, 2.0, 3.0, 4.0])
    h.accumulate_attn_output(src_lse, src, dst_lse, dst)
    torch.cuda.synchronize()
    for at in _spots(src.numel()):
        assert torch.equal(dst.view(-1)[at:at + 4].cpu().float(), torch.tensor([0.5, 1.0, 1.5, 2.0]))
    for part in dst_lse.view(-1).split(1 << 30):
        assert float((part - math.log(2.0)).abs().max()) <= 2.0 ** -22


def test_transpose_of_one_row():
    """A row of 2^30 elements and some is as many tiles of 64 x 64 as 2^32 threads take."""
    n = 2 ** 30 + 1001
    print("transpose", n, flush=True)
    src = torch.zeros(n, 1, dtype=torch.bfloat16, device="cuda")
    spots = [0, 2 ** 29 - 2, 2 ** 30 - 2, n - 4]
    for at in spots:
        src[at:at + 4, 0] = torch.tensor([1.0, 2.0, 3.0, 4.0])
    dst = torch.full((1, n), 7.0, dtype=torch.bfloat16, device="cuda")
    h.transpose(2.0, src, dst, 1, n)
    torch.cuda.synchronize()
    assert torch.equal(dst.view(-1), 2 * src.view(-1))
