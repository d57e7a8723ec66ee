"""Rotary embedding with positions of several axes against the formula in 64 bits."""
import numpy as np
import pytest
import torch

from nntile_amd import hip_sdpa as h

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# half a step of the type, relative
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}


def _want(x, positions, freqs, axes, n_batch, backward):
    """x [heads * n_batch, seq, head] (CPU) in 64 bits."""
    pos = positions.numpy().astype(np.float64)
    pos = np.broadcast_to(pos, (pos.shape[0], n_batch, pos.shape[2]))
    ax = axes.numpy()
    angle = np.where(((ax >= 0) & (ax < len(pos)))[:, None, None], pos[np.clip(ax, 0, len(pos) - 1)], 0.0)
    angle = (angle * freqs.numpy()[:, None, None]).transpose(1, 2, 0)
    c, s = np.cos(angle), np.sin(angle) * (-1 if backward else 1)
    y = x.double().numpy().reshape(-1, n_batch, x.shape[1], x.shape[2] // 2, 2)
    out = np.stack((c * y[..., 0] - s * y[..., 1], s * y[..., 0] + c * y[..., 1]), axis=-1)
    return out.reshape(x.shape), np.broadcast_to(np.abs(y).sum(-1, keepdims=True), y.shape).reshape(x.shape)


def _check(dtype, n_batch, seq, heads_q, heads_k, head, sections, far, backward, shared=False, inplace=False, offset=0):
    print("rope_axes", dtype, n_batch, seq, heads_q, heads_k, head, sections, far, backward, flush=True)
    g = torch.Generator().manual_seed(41)
    positions = torch.randint(-far, far + 1, (len(sections), 1 if shared else n_batch, seq), generator=g)
    freqs, axes = h.rope_axes_freqs(head, sections, device="cpu")

    def tensor(heads):
        flat = torch.randn(heads * n_batch * seq * head + offset, generator=g).to(DT[dtype])
        x = flat.cuda()[offset:].view(heads * n_batch, seq, head)
        return x.cpu(), x

    q, qd = tensor(heads_q)
    k, kd = tensor(heads_k) if heads_k else (None, None)
    q_out = qd if inplace else torch.full_like(qd, float("nan"))
    k_out = None if kd is None else kd if inplace else torch.full_like(kd, float("nan"))
    h.rope_axes(positions.cuda(), freqs.cuda(), axes.cuda(), qd, q_out, kd, k_out, backward=backward)
    torch.cuda.synchronize()
    for x, got in ((q, q_out), (k, k_out)):
        if x is None:
            continue
        want, size = _want(x, positions, freqs, axes, n_batch, backward)
        # one rounding to the type; sine and cosine within 2^-22 (a quarter of it from the angle's
        # fp32 remainder of at most pi * 2^-25, the rest the functions'), two products and a sum in fp32
        bound = HALF_STEP[dtype] * np.abs(want) + 2.0 ** -21 * size + (2.0 ** -25 if dtype == "fp16" else 0)
        off = np.abs(got.double().cpu().numpy() - want)
        print("worst %.2f of the bound" % (off / np.maximum(bound, 1e-30)).max(), flush=True)
        assert np.all(off <= bound)


@pytest.mark.parametrize("dtype", sorted(DT))
@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("n_batch,seq,heads_q,heads_k,head,sections,far", [
    (1, 1, 1, 0, 2, [1], 3), (2, 1, 4, 1, 128, [64], 100000), (3, 33, 3, 2, 64, [16, 8, 8], 500),
    (1, 700, 5, 5, 128, [32, 32], 40), (2, 17, 2, 1, 6, [1, 0, 2], 9), (5, 3, 9, 9, 40, [12, 8], 2 ** 20)])
def test_against_the_formula(dtype, backward, n_batch, seq, heads_q, heads_k, head, sections, far):
    _check(dtype, n_batch, seq, heads_q, heads_k, head, sections, far, backward)


@pytest.mark.parametrize("dtype", sorted(DT))
def test_forms(dtype):
    _check(dtype, 3, 20, 2, 2, 64, [16, 16], 50, False, shared=True)
    _check(dtype, 2, 20, 4, 2, 64, [16, 16], 50, True, inplace=True)
    _check(dtype, 2, 9, 4, 2, 64, [16, 16], 50, False, offset=1)       # addresses off 16 bytes


def test_far_positions():
    _check("fp32", 1, 64, 1, 1, 128, [64], 2 ** 31, False)


def test_backward_is_the_transpose_and_undoes_the_rotation():
    g = torch.Generator().manual_seed(42)
    positions = torch.randint(0, 3000, (2, 2, 50), generator=g).cuda()
    freqs, axes = h.rope_axes_freqs(64, [20, 12])
    x, dy = (torch.randn(6, 50, 64, generator=g).cuda() for _ in range(2))
    y, dx, back = (torch.empty_like(x) for _ in range(3))
    h.rope_axes(positions, freqs, axes, x, y)
    h.rope_axes(positions, freqs, axes, dy, dx, backward=True)
    h.rope_axes(positions, freqs, axes, y, back, backward=True)
    # <dy, R x> = <R^T dy, x>, exact up to fp32
    a, b = float((dy.double() * y.double()).sum()), float((dx.double() * x.double()).sum())
    assert abs(a - b) <= 2.0 ** -20 * float((dy.double() * y.double()).abs().sum())
    assert float((back - x).abs().max()) <= 2.0 ** -20 * float(x.abs().max()) * 4
    # and against differences: the operator is linear, so a step of any size gives the derivative
    step = torch.zeros_like(x)
    step[3, 7, 21] = 0.5
    y2 = torch.empty_like(x)
    h.rope_axes(positions, freqs, axes, x + step, y2)
    slope = float(((y2.double() - y.double()) * dy.double()).sum()) / 0.5
    assert abs(slope - float(dx[3, 7, 21])) <= 1e-4 * max(1.0, abs(slope))


def test_an_axis_that_is_none_leaves_its_pairs():
    x = torch.randn(1, 4, 8).cuda()
    y = torch.empty_like(x)
    positions = torch.full((1, 1, 4), 5).cuda()
    freqs, axes = h.rope_axes_freqs(8, [4])
    axes[1], axes[3] = -1, 1
    h.rope_axes(positions, freqs, axes, x, y)
    assert torch.equal(y[..., 2:4], x[..., 2:4]) and torch.equal(y[..., 6:8], x[..., 6:8])
    assert not torch.equal(y[..., 0:2], x[..., 0:2])


def test_freqs_of_the_axes():
    f, a = h.rope_axes_freqs(16, [4, 2, 2], base=100.0, device="cpu")
    assert a.tolist() == [0, 0, 0, 0, 1, 1, 2, 2]
    assert np.allclose(f.numpy(), 100.0 ** (-np.arange(8) / 8))
    f, a = h.rope_axes_freqs(16, [4, 2, 2], base=100.0, own=True, device="cpu")
    assert np.allclose(f.numpy(), 100.0 ** -np.array([0, .25, .5, .75, 0, .5, 0, .5]))
