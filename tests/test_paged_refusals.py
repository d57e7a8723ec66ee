"""What the paged cache and the rotary embedding of several axes refuse, at the C ABI and in Python
(no GPU: nothing is launched)."""
import ctypes

import pytest
import torch

from nntile_amd import hip_sdpa as h
from nntile_amd.kv_cache import PagedKVCache

TYPES = ("bf16", "fp16", "fp32")


def test_struct_layouts_match_header():
    assert ctypes.sizeof(h.PagedCacheArgs) == 15 * 8
    assert ctypes.sizeof(h.PagedArgs) == 15 * 8 + 2 * 8 + 8 + 3 * 8
    assert ctypes.sizeof(h.RopeAxesArgs) == 7 * 8 + 8 + 7 * 8


def _cache(**kw):
    c = h.PagedCacheArgs()
    c.k_pages = c.v_pages = c.table = c.lens = 4096         # never dereferenced on these paths
    c.head, c.page_rows, c.n_head_kv, c.n_pages, c.max_pages, c.n_batch = 64, 16, 2, 5, 3, 2
    c.page_stride = 64 * 16 * 2
    for k, v in kw.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [
    (dict(k_pages=None), h.EINVAL), (dict(v_pages=None), h.EINVAL), (dict(table=None), h.EINVAL),
    (dict(lens=None), h.EINVAL), (dict(k_pages=4104), h.EINVAL), (dict(lens=4098), h.EINVAL),
    (dict(table=4097), h.EINVAL), (dict(new_rows=4097), h.EINVAL),
    (dict(head=0), h.EINVAL), (dict(page_rows=0), h.EINVAL), (dict(n_head_kv=-1), h.EINVAL),
    (dict(n_pages=0), h.EINVAL), (dict(max_pages=0), h.EINVAL), (dict(n_batch=0), h.EINVAL),
    (dict(n_pages=1 << 31), h.EINVAL), (dict(max_pages=1 << 28), h.EINVAL), (dict(n_batch=1 << 31), h.EINVAL),
    (dict(page_stride=64 * 16 * 2 - 8), h.EINVAL), (dict(page_stride=64 * 16 * 2 + 2), h.EINVAL),
    (dict(page_stride=1 << 60), h.EINVAL), (dict(k_scales=4096), h.EINVAL),
    (dict(head=32), h.EUNSUPPORTED), (dict(head=96), h.EUNSUPPORTED), (dict(page_rows=8), h.EUNSUPPORTED),
    (dict(page_rows=48), h.EUNSUPPORTED), (dict(page_rows=1 << 17), h.EUNSUPPORTED)]
PACKED = dict(k_scales=4096, v_scales=4096, scale_stride=32)
BAD_PACKED = [(dict(PACKED, scale_stride=16), h.EINVAL), (dict(PACKED, scale_stride=40), h.EINVAL),
              (dict(PACKED, k_scales=4104), h.EINVAL), (dict(PACKED, scale_stride=1 << 60), h.EINVAL)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("change,code", BAD_CACHES + BAD_PACKED)
def test_bad_caches(t, change, code):
    if t == "fp32" and "scale_stride" in change:
        code = h.EUNSUPPORTED
    L = h.lib()
    c = _cache(**change)
    assert getattr(L, "nntile_hip_paged_kv_append_" + t)(None, ctypes.byref(c), 1, 4096, 4096) == code
    assert getattr(L, "nntile_hip_paged_kv_read_" + t)(None, ctypes.byref(c), 0, 1, 4096, 4096) == code
    a = _attend()
    a.cache = c
    assert getattr(L, "nntile_hip_sdpa_fwd_paged_" + t)(None, ctypes.byref(a), 4096, 1 << 40) == code


@pytest.mark.parametrize("t", TYPES)
def test_bad_moves(t):
    L = h.lib()
    append, read = (getattr(L, "nntile_hip_paged_kv_%s_%s" % (w, t)) for w in ("append", "read"))
    c = ctypes.byref(_cache())
    assert append(None, None, 1, 4096, 4096) == h.EINVAL
    assert append(None, c, -1, 4096, 4096) == h.EINVAL
    assert append(None, c, 1 << 30, 4096, 4096) == h.EINVAL         # 2 * 2 * 2^30 rows
    assert append(None, c, 1, None, 4096) == h.EINVAL
    assert append(None, c, 1, 4096, 4104) == h.EINVAL
    assert append(None, c, 0, None, None) == h.OK
    assert read(None, None, 0, 1, 4096, 4096) == h.EINVAL
    assert read(None, c, -1, 1, 4096, 4096) == h.EINVAL
    assert read(None, c, (1 << 31) - 1, 1, 4096, 4096) == h.EINVAL
    assert read(None, c, 0, -1, 4096, 4096) == h.EINVAL
    assert read(None, c, 0, 1, 4104, 4096) == h.EINVAL
    assert read(None, c, 0, 1, 4096, None) == h.EINVAL
    assert read(None, c, 5, 0, None, None) == h.OK


def _attend(**kw):
    a = h.PagedArgs()
    a.cache = _cache()
    a.q_seq, a.kv_group, a.mask_mode = 1, 2, h.MASK_CAUSAL
    a.Q = a.lse = a.A = 4096
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("t", TYPES)
def test_bad_attention(t):
    L = h.lib()
    f = getattr(L, "nntile_hip_sdpa_fwd_paged_" + t)
    need = L.nntile_hip_sdpa_fwd_paged_workspace_bytes(ctypes.byref(_attend()))
    assert need > 0 and need % 4 == 0
    assert f(None, None, 4096, need) == h.EINVAL
    for change in (dict(q_seq=0), dict(kv_group=0), dict(q_seq=1 << 31), dict(kv_group=1 << 31), dict(q_seq=1 << 29),
                   dict(Q=None), dict(lse=None), dict(A=None), dict(Q=4104), dict(A=4100), dict(lse=4098),
                   dict(mask_mode=7), dict(mask_mode=-1), dict(flags=2), dict(flags=h.FORM_SPLIT)):
        assert f(None, ctypes.byref(_attend(**change)), 4096, 1 << 40) == h.EINVAL, change
    for mode in (h.MASK_ADDITIVE, h.MASK_BOOL):
        assert f(None, ctypes.byref(_attend(mask_mode=mode)), 4096, need) == h.EUNSUPPORTED
    assert f(None, ctypes.byref(_attend()), None, need) == h.EWORKSPACE
    assert f(None, ctypes.byref(_attend()), 4104, need) == h.EWORKSPACE
    assert f(None, ctypes.byref(_attend()), 4096, need - 1) == h.EWORKSPACE
    assert L.nntile_hip_sdpa_fwd_paged_workspace_bytes(None) == 0
    assert L.nntile_hip_sdpa_fwd_paged_workspace_bytes(ctypes.byref(_attend(q_seq=0))) == 0


def _rope(**kw):
    a = h.RopeAxesArgs()
    a.head, a.seq, a.n_batch, a.heads_q, a.heads_k, a.n_axes, a.pos_batch_stride = 64, 5, 2, 4, 2, 3, 5
    a.positions = a.freqs = a.axes = a.q = a.k = a.q_out = a.k_out = 4096
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("t", TYPES)
def test_bad_rotations(t):
    f = getattr(h.lib(), "nntile_hip_rope_axes_" + t)
    assert f(None, None) == h.EINVAL
    for change in (dict(head=63), dict(head=-2), dict(seq=-1), dict(n_batch=-1), dict(heads_q=-1), dict(heads_k=-1),
                   dict(n_axes=0), dict(n_axes=1 << 31), dict(pos_batch_stride=4), dict(pos_batch_stride=-5),
                   dict(positions=None), dict(freqs=None), dict(axes=None), dict(q=None), dict(q_out=None),
                   dict(k=None), dict(k_out=None), dict(positions=4100), dict(freqs=4100), dict(axes=4098),
                   dict(q=4097), dict(k_out=4097), dict(seq=1 << 40, pos_batch_stride=1 << 40, n_batch=1 << 20)):
        assert f(None, ctypes.byref(_rope(**change))) == h.EINVAL, change
    for change in (dict(head=0), dict(seq=0, pos_batch_stride=0), dict(n_batch=0), dict(heads_q=0, heads_k=0)):
        assert f(None, ctypes.byref(_rope(**change))) == h.OK, change


T = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
I = torch.zeros(2, 3, dtype=torch.int32)
PAGES = torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16)


@pytest.mark.parametrize("call", [
    lambda: h.paged_kv_append(T, T, PAGES, PAGES, I, I[:, 0].contiguous()),
    lambda: h.paged_kv_read(PAGES, PAGES, I, I[:, 0].contiguous(), T, T),
    lambda: h.sdpa_fwd_paged(PAGES, PAGES, I, I[:, 0].contiguous(), T, torch.zeros(4, 2), T, h.MASK_CAUSAL, 1, T),
    lambda: h.rope_axes(torch.zeros(1, 2, 2, dtype=torch.int64), torch.zeros(32, dtype=torch.float64),
                        torch.zeros(32, dtype=torch.int32), T, T)])
def test_tensors_off_the_device_are_refused(call):
    with pytest.raises(ValueError, match="contiguous device tensors"):
        call()


def test_objects_that_are_no_tensors_are_refused():
    with pytest.raises(TypeError, match="torch tensor"):
        h.rope_axes([1], T, T, T, T)
    with pytest.raises(TypeError, match="torch tensor"):
        h.paged_kv_append(T.tolist(), T, PAGES, PAGES, I, I)


def test_frequencies_are_refused():
    for head, sections in ((64, [16, 17]), (64, []), (63, [31]), (64, [33, -1]), (0, [0])):
        with pytest.raises(ValueError):
            h.rope_axes_freqs(head, sections, device="cpu")


def test_caches_that_cannot_be():
    for bad in (dict(page_rows=8), dict(page_rows=40), dict(n_pages=0), dict(n_batch=0), dict(max_rows=0),
                dict(head=32), dict(n_head_kv=0)):
        with pytest.raises(ValueError):
            PagedKVCache(**dict(dict(n_pages=4, page_rows=16, n_batch=2, max_rows=64, n_head_kv=2, head=64,
                                     device="cpu"), **bad))
    with pytest.raises(TypeError):
        PagedKVCache(4, 16, 2, 64, 2, 64, dtype=torch.float32, packed=True, device="cpu")
    with pytest.raises(TypeError):
        PagedKVCache(4, 16, 2, 64, 2, 64, dtype=torch.int8, device="cpu")
    c = PagedKVCache(4, 16, 2, 64, 2, 64, device="cpu")
    one = torch.zeros(4, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="contiguous device tensors"):
        c.append(one, one)
    with pytest.raises(ValueError):
        c.append(one, one.float())
    with pytest.raises(ValueError):
        c.append(one[:2], one[:2])
    assert c.lengths == [0, 0] and c.free_pages == 4


def test_workspace_sizes():
    q = torch.zeros(32, 3, 128)
    small = h.paged_workspace_bytes(q, 2, 4)
    assert small > 0 and h.paged_workspace_bytes(torch.zeros(32, 30, 128), 2, 4) > small
    for n_batch, group in ((3, 4), (0, 1), (1, 0)):
        with pytest.raises(h.SdpaError):
            h.paged_workspace_bytes(q, n_batch, group)
