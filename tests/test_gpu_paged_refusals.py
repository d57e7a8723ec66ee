"""Tensors on the device that do not fit each other: refused before anything is launched."""
import pytest
import torch

from nntile_amd import hip_sdpa as h

pytestmark = pytest.mark.gpu


def _cache(packed=False):
    t = torch.float8_e4m3fn if packed else torch.bfloat16
    pool = torch.zeros(6, 2, 2, 16, 64, dtype=torch.uint8 if packed else t, device="cuda")
    pool = pool.view(t) if packed else pool
    c = dict(k_pages=pool[:, 0], v_pages=pool[:, 1], table=torch.zeros(3, 2, dtype=torch.int32, device="cuda"),
             lens=torch.ones(3, dtype=torch.int32, device="cuda"))
    if packed:
        s = torch.ones(6, 2, 2, 16, dtype=torch.uint8, device="cuda")
        c.update(k_scales=s[:, 0], v_scales=s[:, 1])
    return c


def _tile(rows=1, heads=2, dtype=torch.bfloat16):
    return torch.zeros(heads * 3, rows, 64, dtype=dtype, device="cuda")


def _calls(c, k=None, v=None, Q=None, lse=None, A=None, group=2, ws=None, new_rows=None, mode=h.MASK_CAUSAL):
    """append, read and attend with these arguments"""
    k = _tile() if k is None else k
    v = _tile() if v is None else v
    Q = _tile(heads=4) if Q is None else Q
    A = torch.zeros_like(Q) if A is None else A
    lse = torch.zeros(Q.shape[:2], device="cuda") if lse is None else lse
    if ws is None:
        ws = torch.zeros(h.paged_workspace_bytes(_tile(heads=4), 3, 2), dtype=torch.uint8, device="cuda")
    scales = {n: c[n] for n in ("k_scales", "v_scales") if n in c}
    pages = [c[n] for n in ("k_pages", "v_pages", "table", "lens")]
    return {"append": lambda: h.paged_kv_append(k, v, *pages, new_rows=new_rows, **scales),
            "read": lambda: h.paged_kv_read(*pages, k, v, **scales),
            "attend": lambda: h.sdpa_fwd_paged(*pages, Q, lse, A, mode, group, ws, new_rows=new_rows, **scales)}


ALL = ("append", "read", "attend")


def test_what_fits_runs():
    for packed in (False, True):
        for f in _calls(_cache(packed)).values():
            f()
    torch.cuda.synchronize()


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("name,make,error", [
    ("table", lambda t: t.long(), ValueError), ("table", lambda t: t[0], ValueError),
    ("table", lambda t: torch.zeros(2, 3, dtype=torch.int32, device="cuda").t(), ValueError),
    ("table", lambda t: t[:2].contiguous(), h.SdpaError), ("lens", lambda t: t.long(), ValueError),
    ("lens", lambda t: t[:2].contiguous(), h.SdpaError), ("lens", lambda t: t.cpu(), ValueError),
    ("k_pages", lambda t: t.half(), ValueError), ("k_pages", lambda t: t.contiguous(), h.SdpaError),
    ("v_pages", lambda t: t[:, :, :8], (ValueError, h.SdpaError)), ("v_pages", lambda t: t.transpose(1, 2), (ValueError, h.SdpaError)),
    ("k_pages", lambda t: t[:, 0], ValueError), ("v_pages", lambda t: t.cpu(), ValueError)])
def test_caches(packed, name, make, error):
    c = _cache(packed)
    c[name] = make(c[name])
    for f in _calls(c).values():
        with pytest.raises(error):
            f()


@pytest.mark.parametrize("name,make,error", [
    ("k_scales", lambda t: t.float(), ValueError), ("v_scales", lambda t: t[:, :, ::2], (ValueError, h.SdpaError)),
    ("k_scales", lambda t: t.contiguous(), h.SdpaError), ("v_scales", lambda t: None, h.SdpaError),
    ("k_scales", lambda t: None, (ValueError, h.SdpaError))])
def test_scales(name, make, error):
    c = _cache(True)
    c[name] = make(c[name])
    for f in _calls(c).values():
        with pytest.raises(error):
            f()


@pytest.mark.parametrize("kw,which,error", [
    (dict(k=_tile), ("append", "read"), None), (dict(k=lambda: _tile(2)), ("append", "read"), h.SdpaError),
    (dict(k=lambda: _tile(heads=3), v=lambda: _tile(heads=3)), ("append", "read"), h.SdpaError),
    (dict(v=lambda: _tile(dtype=torch.float16)), ("append", "read"), h.SdpaError),
    (dict(k=lambda: _tile(2)[:, ::2]), ("append", "read"), ValueError),
    (dict(Q=lambda: _tile(heads=3)), ("attend",), h.SdpaError),
    (dict(A=lambda: _tile(heads=4, dtype=torch.float32)), ("attend",), h.SdpaError),
    (dict(lse=lambda: torch.zeros(12, 1, dtype=torch.float64, device="cuda")), ("attend",), ValueError),
    (dict(lse=lambda: torch.zeros(12, 2, device="cuda")), ("attend",), h.SdpaError),
    (dict(ws=lambda: torch.zeros(1024, dtype=torch.uint8, device="cuda")), ("attend",), h.SdpaError),
    (dict(group=lambda: 0), ("attend",), h.SdpaError), (dict(group=lambda: 4), ("attend",), h.SdpaError),
    (dict(mode=lambda: h.MASK_ADDITIVE), ("attend",), h.SdpaError),
    (dict(new_rows=lambda: torch.ones(2, dtype=torch.int32, device="cuda")), ("append", "attend"), h.SdpaError),
    (dict(new_rows=lambda: torch.ones(3, device="cuda")), ("append", "attend"), ValueError)])
def test_tiles(kw, which, error):
    calls = _calls(_cache(), **{n: f() for n, f in kw.items()})
    for name in which:
        if error is None:
            calls[name]()
        else:
            with pytest.raises(error):
                calls[name]()


def test_fp32_tiles_have_no_8_bit_pages():
    c = _cache(True)
    calls = _calls(c, k=_tile(dtype=torch.float32), v=_tile(dtype=torch.float32),
                   Q=_tile(heads=4, dtype=torch.float32))
    for f in calls.values():
        with pytest.raises(h.SdpaError):
            f()


@pytest.mark.parametrize("change,error", [
    (dict(positions=lambda t: t.int()), ValueError), (dict(positions=lambda t: t[:, :, :4].contiguous()), h.SdpaError),
    (dict(positions=lambda t: torch.zeros(3, 5, 5, dtype=torch.int64, device="cuda")), h.SdpaError),
    (dict(freqs=lambda t: t.float()), ValueError), (dict(freqs=lambda t: t[:7].contiguous()), h.SdpaError),
    (dict(axes=lambda t: t.long()), ValueError), (dict(axes=lambda t: t[:7].contiguous()), h.SdpaError),
    (dict(q_out=lambda t: t[:4].contiguous()), h.SdpaError), (dict(q_out=lambda t: t.float()), h.SdpaError),
    (dict(k=lambda t: t.half()), h.SdpaError), (dict(k=lambda t: None), h.SdpaError),
    (dict(q=lambda t: t.transpose(1, 2)), ValueError), (dict(axes=lambda t: t.cpu()), ValueError)])
def test_rotations(change, error):
    freqs, axes = h.rope_axes_freqs(16, [2, 3, 3])
    a = dict(positions=torch.zeros(3, 2, 5, dtype=torch.int64, device="cuda"), freqs=freqs, axes=axes)
    for n, heads in (("q", 4), ("q_out", 4), ("k", 2), ("k_out", 2)):
        a[n] = torch.zeros(heads * 2, 5, 16, dtype=torch.bfloat16, device="cuda")
    h.rope_axes(**a)
    for n, f in change.items():
        a[n] = f(a[n])
    with pytest.raises(error):
        h.rope_axes(**a)
