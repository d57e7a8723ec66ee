"""Tensors on the device that do not fit each other, for the calls on 4-bit pages, the weights of cached rows and their
eviction: refused before anything is launched."""
import pytest
import torch

from nntile_amd import hip_sdpa as h

pytestmark = pytest.mark.gpu

BITS = [4, 8, 16]


def _cache(bits=4):
    """6 pages of 16 rows, 2 heads of 64, 3 sequences."""
    if bits == 16:
        pool = torch.zeros(6, 2, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    else:
        pool = torch.zeros(6, 2, 2, 16, 8 * bits, dtype=torch.uint8, device="cuda")
        pool = pool.view(torch.float4_e2m1fn_x2 if bits == 4 else torch.float8_e4m3fn)
    c = dict(k_pages=pool[:, 0], v_pages=pool[:, 1], table=torch.zeros(3, 2, dtype=torch.int32, device="cuda"),
             lens=torch.ones(3, dtype=torch.int32, device="cuda"))
    if bits != 16:
        s = torch.full((6, 2, 2, 16) + ((2,) if bits == 4 else ()), 127, dtype=torch.uint8, device="cuda")
        c.update(k_scales=s[:, 0], v_scales=s[:, 1])
    return c


def _tile(rows=1, heads=2, dtype=torch.bfloat16):
    return torch.zeros(heads * 3, rows, 64, dtype=dtype, device="cuda")


def _calls(c, dtype=torch.bfloat16, **given):
    k, Q = _tile(dtype=dtype), _tile(heads=4, dtype=dtype)
    a = dict(k=k, v=k.clone(), Q=Q, A=torch.zeros_like(Q), lse=torch.zeros(Q.shape[:2], device="cuda"), group=2,
             ws=torch.zeros(h.paged_workspace_bytes(_tile(heads=4), 3, 2), dtype=torch.uint8, device="cuda"),
             weights=torch.zeros(6, 32, device="cuda"), out=torch.zeros(6, 32, device="cuda"),
             kept=torch.zeros(6, 5, dtype=torch.int32, device="cuda"), recent=2, decay=1.0, new_rows=None, mode=h.MASK_CAUSAL)
    a.update(given)
    scales = {n: c[n] for n in ("k_scales", "v_scales") if n in c}
    k_scales = {n: c[n] for n in ("k_scales",) if n in c}
    pages = [c[n] for n in ("k_pages", "v_pages", "table", "lens")]
    return {"append": lambda: h.paged_kv_append(a["k"], a["v"], *pages, new_rows=a["new_rows"], **scales),
            "read": lambda: h.paged_kv_read(*pages, a["k"], a["v"], **scales),
            "attend": lambda: h.sdpa_fwd_paged(*pages, a["Q"], a["lse"], a["A"], a["mode"], a["group"], a["ws"],
                                               new_rows=a["new_rows"], **scales),
            "weights": lambda: h.paged_attn_weights(pages[0], *pages[2:], a["Q"], a["lse"], a["weights"], a["mode"],
                                                    a["group"], new_rows=a["new_rows"], decay=a["decay"], **k_scales),
            "evict": lambda: h.paged_kv_evict(*pages, a["weights"], a["out"], a["kept"], a["recent"], **scales)}


@pytest.mark.parametrize("bits", BITS)
def test_what_fits_runs(bits):
    for f in _calls(_cache(bits)).values():
        f()
    torch.cuda.synchronize()


KEYS_ONLY = ("weights",)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("name,make,error", [
    ("table", lambda t: t.long(), ValueError), ("table", lambda t: t[0], ValueError),
    ("table", lambda t: t[:2].contiguous(), h.SdpaError), ("lens", lambda t: t.long(), ValueError),
    ("lens", lambda t: t[:2].contiguous(), h.SdpaError), ("lens", lambda t: t.cpu(), ValueError),
    ("k_pages", lambda t: t.view(torch.uint8), (ValueError, h.SdpaError)), ("k_pages", lambda t: t.contiguous(), h.SdpaError),
    ("k_pages", lambda t: t[:, 0], ValueError), ("v_pages", lambda t: t.cpu(), ValueError),
    ("v_pages", lambda t: t.transpose(1, 2), (ValueError, h.SdpaError))])
def test_caches(bits, name, make, error):
    c = _cache(bits)
    c[name] = make(c[name])
    for call, f in _calls(c).items():
        if call == "weights" and (name == "v_pages" or c["k_pages"].dtype != torch.uint8 and c["k_pages"].is_contiguous()):
            continue        # (the values are not looked at)
        with pytest.raises(error):
            f()


@pytest.mark.parametrize("name,make,error", [
    ("k_scales", lambda t: t.float(), ValueError), ("k_scales", lambda t: t[..., 0], ValueError),
    ("v_scales", lambda t: t[..., :1], (ValueError, h.SdpaError)), ("k_scales", lambda t: t.contiguous(), h.SdpaError),
    ("v_scales", lambda t: None, h.SdpaError), ("k_scales", lambda t: None, (ValueError, h.SdpaError)),
    ("k_scales", lambda t: t[:5], h.SdpaError), ("k_scales", lambda t: t.cpu(), ValueError)])
def test_scales_of_four_bits(name, make, error):
    c = _cache(4)
    c[name] = make(c[name])
    for call, f in _calls(c).items():
        if call == "weights" and (name == "v_scales" or c[name] is not None and c[name].is_contiguous() and c[name].shape[0] == 6
                                  and c[name].dtype == torch.uint8 and c[name].is_cuda and c[name].dim() == 4):
            continue
        with pytest.raises(error):
            f()


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("given,which,error", [
    (dict(Q=lambda: _tile(heads=3)), ("attend", "weights"), h.SdpaError),
    (dict(Q=lambda: _tile(heads=4).transpose(0, 1)), ("attend", "weights"), (ValueError, h.SdpaError)),
    (dict(lse=lambda: torch.zeros(12, 1, dtype=torch.float64, device="cuda")), ("attend", "weights"), ValueError),
    (dict(lse=lambda: torch.zeros(12, 2, device="cuda")), ("attend", "weights"), h.SdpaError),
    (dict(lse=lambda: torch.zeros(12, 1)), ("attend", "weights"), ValueError),
    (dict(group=lambda: 0), ("attend", "weights"), h.SdpaError), (dict(group=lambda: 4), ("attend", "weights"), h.SdpaError),
    (dict(mode=lambda: h.MASK_ADDITIVE), ("attend", "weights"), h.SdpaError),
    (dict(new_rows=lambda: torch.ones(2, dtype=torch.int32, device="cuda")), ("append", "attend", "weights"), h.SdpaError),
    (dict(ws=lambda: torch.zeros(1024, dtype=torch.uint8, device="cuda")), ("attend",), h.SdpaError),
    (dict(weights=lambda: torch.zeros(6, 31, device="cuda"), out=lambda: torch.zeros(6, 31, device="cuda")),
     ("weights", "evict"), h.SdpaError),
    (dict(weights=lambda: torch.zeros(5, 32, device="cuda"), out=lambda: torch.zeros(5, 32, device="cuda")),
     ("weights", "evict"), h.SdpaError),
    (dict(weights=lambda: torch.zeros(6, 32, dtype=torch.float64, device="cuda")), ("weights", "evict"), ValueError),
    (dict(weights=lambda: torch.zeros(6, 64, device="cuda")[:, ::2]), ("weights", "evict"), ValueError),
    (dict(weights=lambda: torch.zeros(6, 32)), ("weights", "evict"), ValueError),
    (dict(out=lambda: torch.zeros(6, 33, device="cuda")), ("evict",), h.SdpaError),
    (dict(decay=lambda: -0.1), ("weights",), h.SdpaError), (dict(decay=lambda: 1.5), ("weights",), h.SdpaError),
    (dict(decay=lambda: float("nan")), ("weights",), h.SdpaError), (dict(decay=lambda: "1"), ("weights",), TypeError),
    (dict(kept=lambda: torch.zeros(6, 5, device="cuda")), ("evict",), ValueError),
    (dict(kept=lambda: torch.zeros(5, 5, dtype=torch.int32, device="cuda")), ("evict",), h.SdpaError),
    (dict(kept=lambda: torch.zeros(6, 0, dtype=torch.int32, device="cuda")), ("evict",), h.SdpaError),
    (dict(recent=lambda: -1), ("evict",), h.SdpaError), (dict(recent=lambda: 6), ("evict",), h.SdpaError)])
def test_arguments(bits, given, which, error):
    calls = _calls(_cache(bits), **{n: f() for n, f in given.items()})
    for name in which:
        with pytest.raises(error):
            calls[name]()


def test_fp32_tiles_have_no_4_bit_pages():
    for call, f in _calls(_cache(4), dtype=torch.float32).items():
        if call != "evict":
            with pytest.raises(h.SdpaError):
                f()
