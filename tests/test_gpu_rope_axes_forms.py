"""Rotary embedding with positions of several axes: the forms of large calls."""
import numpy as np
import pytest
import torch

from nntile_amd import hip_sdpa as h
from .test_gpu_rope_axes import DT, HALF_STEP, _check, _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("head,heads", [(6, 357914000), (10, 214748400)])
def test_more_pairs_than_a_launch_has_threads(head, heads):
    """2^32 pairs and some, 17 GB in place: a head size that is no multiple of 8 has a thread a pair."""
    seq, pairs_of_head = 4, 4 * (head // 2)
    assert heads * pairs_of_head > 2 ** 32
    print("rope_axes", head, heads, flush=True)
    positions = torch.tensor([[[3, 1, -7, 100]]])
    freqs, axes = h.rope_axes_freqs(head, [head // 2], device="cpu")
    x = torch.zeros(heads, seq, head, dtype=torch.bfloat16, device="cuda")
    # heads at the front, on both sides of 2^31 and 2^32 pairs, and the last ones
    g = torch.Generator().manual_seed(45)
    spots = [0, 2 ** 31 // pairs_of_head - 2, 2 ** 32 // pairs_of_head - 2, heads - 4]
    given = [torch.randn(4, seq, head, generator=g).to(torch.bfloat16) for _ in spots]
    for at, y in zip(spots, given):
        x[at:at + 4] = y.cuda()
    h.rope_axes(positions.cuda(), freqs.cuda(), axes.cuda(), x, x)
    torch.cuda.synchronize()
    for at, y in zip(spots, given):
        want, size = _want(y, positions, freqs, axes, 1, False)
        off = np.abs(x[at:at + 4].double().cpu().numpy() - want)
        assert np.all(off <= HALF_STEP["bf16"] * np.abs(want) + 2.0 ** -21 * size)
    assert not x[spots[1] + 4:spots[2]:1000003].any()


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("backward,inplace", [(False, False), (True, True), (False, True)])
@pytest.mark.parametrize("n_batch,seq,heads_q,heads_k,head,sections,shared", [
    (1, 4099, 9, 4, 128, [22, 21, 21], False),          # queries end and keys begin within eight heads
    (3, 1367, 5, 8, 128, [64], True),
    (2, 8200, 3, 2, 64, [16, 16], False),               # fewer than eight heads
    (5, 1639, 16, 0, 64, [20, 12], False),
    (1, 30000, 1, 1, 40, [12, 8], False)])
def test_eight_heads_a_thread(dtype, backward, inplace, n_batch, seq, heads_q, heads_k, head, sections, shared):
    """Calls large enough that every CU has a workgroup with eight heads a thread."""
    assert -(-n_batch * seq * (head // 8) // 256) * -(-(heads_q + heads_k) // 8) >= 256
    _check(dtype, n_batch, seq, heads_q, heads_k, head, sections, 5000, backward, shared=shared, inplace=inplace)


@pytest.mark.parametrize("backward,inplace", [(False, False), (True, True)])
@pytest.mark.parametrize("heads_q,heads_k", [(9, 4), (10, 0), (3, 11)])
def test_four_heads_a_thread_past_the_caches(backward, inplace, heads_q, heads_k):
    """fp32 tensors of 128 MB and more, read and written."""
    seq, head = 128 * 2 ** 20 // (8 * 128 * (heads_q + heads_k)) + 3, 128
    _check("fp32", 1, seq, heads_q, heads_k, head, [32, 32], 5000, backward, inplace=inplace)
