"""What the calls on 4-bit pages, on received weights and of eviction refuse, at the C ABI and in Python (no GPU: nothing is
launched)."""
import ctypes

import pytest
import torch

from nntile_amd import hip_sdpa as h
from nntile_amd.kv_cache import PagedKVCache

KINDS = [("paged", "bf16"), ("paged", "fp16"), ("paged", "fp32"), ("paged4", "bf16"), ("paged4", "fp16")]


def test_struct_layouts_match_header():
    assert ctypes.sizeof(h.PagedWeightsArgs) == 15 * 8 + 3 * 8 + 8 + 3 * 8
    assert h.PagedWeightsArgs.decay.offset == 15 * 8 + 3 * 8 + 4
    assert ctypes.sizeof(h.PagedEvictArgs) == 15 * 8 + 3 * 8 + 3 * 8


def _cache(kind="paged4", **kw):
    c = h.PagedCacheArgs()
    c.k_pages = c.v_pages = c.table = c.lens = 4096         # never dereferenced on these paths
    c.head, c.page_rows, c.n_head_kv, c.n_pages, c.max_pages, c.n_batch = 64, 16, 2, 5, 3, 2
    c.page_stride = 64 * 16 * 2
    if kind == "paged4":
        c.k_scales = c.v_scales = 4096
        c.scale_stride = 64
    for name, v in kw.items():
        setattr(c, name, v)
    return c


def _attend(c):
    a = h.PagedArgs()
    a.cache = c
    a.q_seq, a.kv_group, a.mask_mode, a.flags = 1, 2, h.MASK_CAUSAL, h.OVERWRITE
    a.Q = a.lse = a.A = 4096
    return a


def _weights(kind, **kw):
    a = h.PagedWeightsArgs()
    a.cache = _cache(kind)
    a.q_seq, a.kv_group, a.columns, a.mask_mode, a.decay = 1, 2, 48, h.MASK_CAUSAL, 1.0
    a.Q = a.lse = a.weights = 4096
    for name, v in kw.items():
        setattr(a, name, v)
    return a


def _evict(kind, **kw):
    a = h.PagedEvictArgs()
    a.cache = _cache(kind)
    a.keep, a.recent, a.columns = 10, 3, 48
    a.weights = a.weights_out = a.kept = 4096
    for name, v in kw.items():
        setattr(a, name, v)
    return a


BAD_CACHES = [
    (dict(k_pages=None), h.EINVAL), (dict(v_pages=None), h.EINVAL), (dict(table=None), h.EINVAL), (dict(lens=None), h.EINVAL),
    (dict(k_scales=None), h.EINVAL), (dict(v_scales=None), h.EINVAL), (dict(k_scales=None, v_scales=None), h.EINVAL),
    (dict(k_pages=4104), h.EINVAL), (dict(v_pages=4104), h.EINVAL), (dict(k_scales=4104), h.EINVAL), (dict(v_scales=4100), h.EINVAL),
    (dict(lens=4098), h.EINVAL), (dict(table=4097), h.EINVAL), (dict(new_rows=4097), h.EINVAL),
    (dict(page_stride=64 * 16 * 2 - 32), h.EINVAL), (dict(page_stride=64 * 16 * 2 + 16), h.EINVAL), (dict(page_stride=1 << 60), h.EINVAL),
    (dict(scale_stride=48), h.EINVAL), (dict(scale_stride=72), h.EINVAL), (dict(scale_stride=1 << 60), h.EINVAL),
    (dict(n_pages=1 << 31), h.EINVAL), (dict(max_pages=1 << 28), h.EINVAL), (dict(n_batch=1 << 31), h.EINVAL), (dict(n_head_kv=0), h.EINVAL),
    (dict(head=32), h.EUNSUPPORTED), (dict(head=96), h.EUNSUPPORTED), (dict(page_rows=8), h.EUNSUPPORTED), (dict(page_rows=48), h.EUNSUPPORTED)]


@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("change,code", BAD_CACHES)
def test_bad_caches_of_four_bits(t, change, code):
    L = h.lib()
    c = _cache(**change)
    assert getattr(L, "nntile_hip_paged4_kv_append_" + t)(None, ctypes.byref(c), 1, 4096, 4096) == code
    assert getattr(L, "nntile_hip_paged4_kv_read_" + t)(None, ctypes.byref(c), 0, 1, 4096, 4096) == code
    assert getattr(L, "nntile_hip_sdpa_fwd_paged4_" + t)(None, ctypes.byref(_attend(c)), 4096, 1 << 40) == code
    a = _evict("paged4")
    a.cache = c
    assert getattr(L, "nntile_hip_paged4_kv_evict_" + t)(None, ctypes.byref(a)) == code
    w = _weights("paged4", cache=c)
    if set(change) <= {"v_pages", "v_scales"}:
        w.decay = 2.0           # (the values are not looked at: it is this that is refused)
        code = h.EINVAL
    assert getattr(L, "nntile_hip_paged4_attn_weights_" + t)(None, ctypes.byref(w)) == code


@pytest.mark.parametrize("t", ["bf16", "fp16"])
def test_bad_moves_and_attention_of_four_bits(t):
    L = h.lib()
    append, read = (getattr(L, "nntile_hip_paged4_kv_%s_%s" % (w, t)) for w in ("append", "read"))
    c = ctypes.byref(_cache())
    assert append(None, None, 1, 4096, 4096) == h.EINVAL
    assert append(None, c, -1, 4096, 4096) == h.EINVAL and append(None, c, 1 << 30, 4096, 4096) == h.EINVAL
    assert append(None, c, 1, None, 4096) == h.EINVAL and append(None, c, 1, 4096, 4104) == h.EINVAL
    assert append(None, c, 0, None, None) == h.OK and read(None, c, 5, 0, None, None) == h.OK
    assert read(None, c, -1, 1, 4096, 4096) == h.EINVAL and read(None, c, (1 << 31) - 1, 1, 4096, 4096) == h.EINVAL
    assert read(None, c, 0, 1, 4104, 4096) == h.EINVAL and read(None, c, 0, 1, 4096, None) == h.EINVAL
    attend = getattr(L, "nntile_hip_sdpa_fwd_paged4_" + t)
    assert attend(None, None, 4096, 1 << 40) == h.EINVAL
    for change, code in ((dict(q_seq=0), h.EINVAL), (dict(kv_group=0), h.EINVAL), (dict(Q=4104), h.EINVAL), (dict(lse=None), h.EINVAL),
                         (dict(flags=64), h.EINVAL), (dict(mask_mode=h.MASK_BOOL), h.EUNSUPPORTED), (dict(mask_mode=17), h.EINVAL)):
        a = _attend(_cache())
        for name, v in change.items():
            setattr(a, name, v)
        assert attend(None, ctypes.byref(a), 4096, 1 << 40) == code
    need = L.nntile_hip_sdpa_fwd_paged_workspace_bytes(ctypes.byref(_attend(_cache())))
    assert need > 0
    for ws, size in ((None, need), (4104, need), (4096, need - 1)):
        assert attend(None, ctypes.byref(_attend(_cache())), ws, size) == h.EWORKSPACE


@pytest.mark.parametrize("kind,t", KINDS)
@pytest.mark.parametrize("change,code", [
    (dict(q_seq=0), h.EINVAL), (dict(kv_group=-1), h.EINVAL), (dict(q_seq=1 << 31), h.EINVAL), (dict(Q=None), h.EINVAL),
    (dict(Q=4104), h.EINVAL), (dict(lse=None), h.EINVAL), (dict(lse=4098), h.EINVAL), (dict(weights=None), h.EINVAL),
    (dict(weights=4097), h.EINVAL), (dict(columns=47), h.EINVAL), (dict(columns=1 << 31), h.EINVAL), (dict(decay=-0.01), h.EINVAL),
    (dict(decay=1.01), h.EINVAL), (dict(decay=float("nan")), h.EINVAL), (dict(mask_mode=h.MASK_ADDITIVE), h.EUNSUPPORTED),
    (dict(mask_mode=9), h.EINVAL)])
def test_bad_weights(kind, t, change, code):
    f = getattr(h.lib(), "nntile_hip_%s_attn_weights_%s" % (kind, t))
    assert f(None, None) == h.EINVAL
    assert f(None, ctypes.byref(_weights(kind, **change))) == code


@pytest.mark.parametrize("kind,t", KINDS)
@pytest.mark.parametrize("change", [dict(keep=0), dict(keep=-5), dict(keep=1 << 31), dict(recent=-1), dict(recent=11), dict(columns=47),
                                    dict(columns=1 << 31), dict(weights=None), dict(weights_out=None), dict(kept=None),
                                    dict(weights=4098), dict(weights_out=4099), dict(kept=4097)])
def test_bad_evictions(kind, t, change):
    f = getattr(h.lib(), "nntile_hip_%s_kv_evict_%s" % (kind, t))
    assert f(None, None) == h.EINVAL
    assert f(None, ctypes.byref(_evict(kind, **change))) == h.EINVAL


def test_more_work_than_a_launch_has():
    """Blocks of rows past 2^31, entries past it."""
    c = _cache("paged", n_batch=1 << 20, n_head_kv=1 << 8, max_pages=1 << 5, page_stride=1 << 30)
    w = _weights("paged", cache=c, columns=512)
    assert h.lib().nntile_hip_paged_attn_weights_bf16(None, ctypes.byref(w)) == h.EINVAL         # 2^28 pairs, 8 blocks of 64 rows each
    e = _evict("paged", cache=_cache("paged", n_batch=1 << 20, n_head_kv=1 << 10, page_stride=1 << 30))
    assert h.lib().nntile_hip_paged_kv_evict_fp32(None, ctypes.byref(e)) == h.EINVAL


def test_sequences_longer_than_the_walks_count():
    """2^31 - 2^16 rows: their number and a step more are no 32-bit integers."""
    big = dict(page_rows=65536, n_head_kv=1, n_batch=1, max_pages=32767, page_stride=64 * 65536)
    for kind in ("paged", "paged4"):
        c = _cache(kind, **dict(big, **({} if kind == "paged" else dict(scale_stride=2 * 65536))))
        w, e = _weights(kind, cache=c, columns=(1 << 31) - 1), _evict(kind, cache=c, columns=(1 << 31) - 1)
        assert getattr(h.lib(), "nntile_hip_%s_attn_weights_bf16" % kind)(None, ctypes.byref(w)) == h.EINVAL
        assert getattr(h.lib(), "nntile_hip_%s_kv_evict_bf16" % kind)(None, ctypes.byref(e)) == h.EINVAL
    a = _attend(c)
    a.q_seq = a.kv_group = 1
    assert h.lib().nntile_hip_sdpa_fwd_paged4_bf16(None, ctypes.byref(a), 4096, 1 << 40) == h.EINVAL
    e = _evict("paged", keep=(1 << 30) + 1)
    assert h.lib().nntile_hip_paged_kv_evict_bf16(None, ctypes.byref(e)) == h.EINVAL


@pytest.mark.parametrize("t,head", [("bf16", 128), ("bf16", 64), ("fp16", 128), ("fp16", 64)])
def test_tiles_of_128_gib(t, head):
    """2^30 rows of 128 bytes and more take 2^32 threads and more in one direction of a launch."""
    c = _cache("paged4", head=head, page_rows=1024, n_head_kv=2, n_pages=5, max_pages=1 << 20, n_batch=2,
               page_stride=head * 2048, scale_stride=head // 32 * 2048)
    rows = 1 << 28
    assert getattr(h.lib(), "nntile_hip_paged4_kv_append_" + t)(None, ctypes.byref(c), rows, 4096, 4096) == h.EINVAL
    if head == 128:         # (four rows a thread: 2^30 rows of 64 values are 2^31 threads)
        assert getattr(h.lib(), "nntile_hip_paged4_kv_read_" + t)(None, ctypes.byref(c), 0, rows, 4096, 4096) == h.EINVAL


def test_caches_that_are_not_made():
    make = lambda **kw: PagedKVCache(4, 16, 1, 64, 1, 64, device="cpu", **kw)
    for bits in (0, 1, 2, 3, 16, 32, "4"):
        with pytest.raises(ValueError):
            make(bits=bits)
    with pytest.raises(ValueError):
        make(packed=True, bits=4)
    for bits in (4, 8):
        with pytest.raises(TypeError):
            make(bits=bits, dtype=torch.float32)
    c = make(bits=4)
    assert c.k_pages.dtype == torch.float4_e2m1fn_x2 and c.k_pages.shape == (4, 1, 16, 32) and c.k_scales.shape == (4, 1, 16, 2)
    assert make(bits=8).k_pages.dtype == make(packed=True).k_pages.dtype == torch.float8_e4m3fn
    assert c.weights is None and make(weighted=True).weights.shape == (1, 64)


def test_tensors_of_the_host_are_refused():
    c = PagedKVCache(4, 16, 1, 64, 1, 64, device="cpu", bits=4, weighted=True)
    if not torch.cuda.is_available():
        for call in (lambda: c.observe(torch.zeros(1, 1, 64, dtype=torch.bfloat16), torch.zeros(1, 1), 1), lambda: c.evict(4)):
            with pytest.raises((ValueError, RuntimeError)):
                call()
