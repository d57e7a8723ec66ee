"""What PagedKVCache does on the host around the weights of its rows and their eviction (no GPU: the calls are taken by
doubles that note what they get)."""
import contextlib

import pytest
import torch

from nntile_amd import hip_sdpa as h
from nntile_amd.kv_cache import PagedKVCache


def _place(t):
    return t.untyped_storage().data_ptr()


class Doubles:
    """Stand in for the calls of hip_sdpa and for the streams."""

    def __init__(self, monkeypatch, fail=False):
        self.calls, self.recorded = [], []
        for name in ("paged_attn_weights", "paged_kv_evict"):
            monkeypatch.setattr(h, name, lambda *a, _name=name, **kw: self._call(_name, a, kw))
        monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
        monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: self.recorded.append((_place(t), s)))
        monkeypatch.setattr(torch.Tensor, "pin_memory", lambda t, *a: t)
        self.fail = fail

    def _call(self, name, a, kw):
        if self.fail:
            raise h.SdpaError(h.EINVAL, "refused")
        self.calls.append((name, a, kw))

    def told(self, stream):
        return {place for place, s in self.recorded if s == stream}

    def tensors(self):
        return {_place(t) for _, a, kw in self.calls for t in list(a) + list(kw.values()) if isinstance(t, torch.Tensor)}


def _cache(lengths, **kw):
    c = PagedKVCache(**dict(dict(n_pages=40, page_rows=16, n_batch=len(lengths), max_rows=160, n_head_kv=2, head=64,
                                 bits=4, weighted=True, device="cpu"), **kw))
    c._reserve(lengths, None)
    c._upload(c.lens, lengths, None)
    c.lengths = list(lengths)
    return c


@pytest.mark.parametrize("bits", [None, 4, 8])
def test_the_calls_tell_of_their_tensors(monkeypatch, bits):
    d = Doubles(monkeypatch)
    c = _cache([70, 30], bits=bits)
    Q = torch.zeros(8, 3, 64, dtype=c.dtype)
    lse = torch.zeros(8, 3)
    c.observe(Q, lse, 2, stream="side")
    c.evict(40, 8, stream="side")
    assert [name for name, _, _ in d.calls] == ["paged_attn_weights", "paged_kv_evict"]
    for t in (Q, lse, c.pool, c.table, c.lens, c.weights) + (() if bits is None else (c.scales,)):
        assert _place(t) in d.tensors() and _place(t) in d.told("side")


def test_an_eviction_frees_pages_and_lowers_lengths(monkeypatch):
    Doubles(monkeypatch)
    c = _cache([70, 30, 16, 160])
    before, free = [list(p) for p in c._pages], c.free_pages
    c.evict(32, 32)
    assert c.lengths == [32, 30, 16, 32] and c.lens.tolist() == [32, 30, 16, 32]
    assert [len(p) for p in c._pages] == [2, 2, 1, 2] and c.free_pages == free + 3 + 8
    for n, pages in enumerate(c._pages):
        assert pages == before[n][:len(pages)]
        assert c.table[n].tolist() == pages + [-1] * (c.max_pages - len(pages))
    c.evict(100)            # nothing to do
    assert c.lengths == [32, 30, 16, 32] and c.free_pages == free + 11


def test_a_refused_eviction_leaves_the_cache(monkeypatch):
    d = Doubles(monkeypatch)
    c = _cache([70, 30])
    d.fail = True
    pages, lens, table = [list(p) for p in c._pages], c.lens.clone(), c.table.clone()
    with pytest.raises(h.SdpaError):
        c.evict(10)
    assert c.lengths == [70, 30] and c._pages == pages and torch.equal(c.lens, lens) and torch.equal(c.table, table)


def test_a_new_sequence_begins_without_weights(monkeypatch):
    Doubles(monkeypatch)
    c = _cache([70, 30])
    c.weights.fill_(3.0)
    c.release(1)
    of = c.weights.view(2, 2, -1)
    assert float(of[:, 1].abs().max()) == 0 and float(of[:, 0].min()) == 3


@pytest.mark.parametrize("kw", [dict(bits=4, weighted=False), dict(bits=8), dict(bits=None), dict(bits=4)])
@pytest.mark.parametrize("max_rows,page_rows", [((1 << 30) + 1, 65536), ((1 << 30) + 1, 16), ((1 << 31) - 65536, 65536)])
def test_more_rows_than_attention_weights_or_eviction_take(kw, max_rows, page_rows):
    """Refused where the cache is made, not when it is filled."""
    with pytest.raises(ValueError, match="2\\^30 rows"):
        _cache([0], **dict(dict(n_pages=1, n_head_kv=1, max_rows=max_rows, page_rows=page_rows), **kw))


@pytest.mark.parametrize("n_batch,n_head_kv,max_rows,page_rows,head,bits,dtype", [
    (1 << 16, 1 << 10, 33 * 64, 16, 64, 4, torch.bfloat16),        # 2^26 entries of 33 blocks
    (1 << 20, 1 << 10, 16, 16, 64, 4, torch.bfloat16),             # 2^30 entries, K and V
    (1 << 20, 1 << 8, 16, 16, 128, None, torch.float32)])          # 2^28 entries, K and V, 8 times 64 bytes
def test_more_entries_than_weights_or_eviction_take(n_batch, n_head_kv, max_rows, page_rows, head, bits, dtype):
    with pytest.raises(ValueError, match="2\\^31"):
        PagedKVCache(1, page_rows, n_batch, max_rows, n_head_kv, head, dtype=dtype, bits=bits, weighted=True, device="cpu")


def test_as_many_rows_as_they_take():
    c = PagedKVCache(1, 65536, 1, 1 << 30, 1, 64, bits=4, device="cpu")
    assert c.max_pages * c.page_rows == 1 << 30
    # (rows as they are, without weights: up to 2^31)
    c = PagedKVCache(1, 65536, 1, (1 << 31) - 65536, 1, 64, device="cpu")
    assert c.max_pages * c.page_rows == (1 << 31) - 65536
