"""What PagedKVCache does on the host around its calls: which tensors it tells the allocator of, which memory it keeps
(no GPU: the calls are taken by doubles that note what they get)."""
import contextlib
import weakref

import pytest
import torch

from nntile_amd import hip_sdpa as h
from nntile_amd.kv_cache import PagedKVCache


def _place(t):
    return t.untyped_storage().data_ptr()


class Doubles:
    """Stand in for the calls of hip_sdpa and for the streams."""

    def __init__(self, monkeypatch):
        self.calls, self.recorded = [], []
        for name in ("paged_kv_read", "sdpa_fwd_tile_cache", "sdpa_fwd_paged"):
            monkeypatch.setattr(h, name, lambda *a, _name=name, **kw: self.calls.append((_name, a, kw)))
        monkeypatch.setattr(h, "tile_cache_workspace_bytes", lambda *a, **kw: 4096)
        monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
        monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: self.recorded.append((_place(t), s)))

    def told(self, stream):
        return {place for place, s in self.recorded if s == stream}

    def names(self):
        return [name for name, _, _ in self.calls]

    def tensors(self):
        return {_place(t) for _, a, kw in self.calls for t in list(a) + list(kw.values()) if isinstance(t, torch.Tensor)}


def _cache(lengths, packed=True, **kw):
    c = PagedKVCache(**dict(dict(n_pages=64, page_rows=64, n_batch=len(lengths), max_rows=1024, n_head_kv=2, head=64,
                                 packed=packed, device="cpu"), **kw))
    c.lengths = list(lengths)
    return c


def _queries(c, q_seq, group):
    Q = torch.zeros(c.n_head_kv * group * c.n_batch, q_seq, c.head, dtype=c.dtype)
    return Q, torch.zeros(Q.shape[:2]), torch.zeros_like(Q)


def test_a_chunk_that_is_read_back_tells_of_its_tensors(monkeypatch):
    """As many queries as go through the tile kernels, on a stream that is given: queries, results and the
    cache's tensors are in use there."""
    d = Doubles(monkeypatch)
    c = _cache([600, 600])
    tiles = _queries(c, 512, 1)
    c.attend(*tiles, 1, stream="side")
    assert d.names() == ["paged_kv_read", "sdpa_fwd_tile_cache"]
    for t in tiles + (c.pool, c.scales, c.lens, c.table):
        assert _place(t) in d.tensors() and _place(t) in d.told("side")


def test_reading_back_tells_of_the_cache(monkeypatch):
    d = Doubles(monkeypatch)
    c = _cache([600, 30])
    c.read(stream="side")
    for t in (c.pool, c.scales, c.lens, c.table):
        assert _place(t) in d.tensors() and _place(t) in d.told("side")


def test_attention_over_the_pages_tells_of_its_tensors(monkeypatch):
    d = Doubles(monkeypatch)
    c = _cache([600, 30])
    tiles = _queries(c, 5, 4)
    c.attend(*tiles, 4, stream="side")
    assert d.names() == ["sdpa_fwd_paged"]
    assert d.tensors() <= d.told("side")


def test_nothing_is_told_of_the_current_stream(monkeypatch):
    d = Doubles(monkeypatch)
    c = _cache([600, 600])
    c.attend(*_queries(c, 512, 1), 1)
    c.attend(*_queries(c, 3, 1), 1)
    c.read()
    assert d.recorded == []


def test_a_workspace_is_not_let_go(monkeypatch):
    """Calls of more and more query rows, down to a generation step again: what an earlier call on whatever stream may
    still use stays with the cache."""
    d = Doubles(monkeypatch)
    c = _cache([600, 30])
    given = []
    for q_seq, group in ((1, 1), (1, 4), (5, 4), (9, 4), (40, 4), (300, 1), (1, 1)):
        c.attend(*_queries(c, q_seq, group), group)
        name, a, kw = d.calls.pop()
        assert name == "sdpa_fwd_paged" and a[9].numel() >= h.paged_workspace_bytes(a[4], 2, group)
        given.append(weakref.ref(a[9]))
        del a, kw
    # (some sizes only: those of 16, 32 and 64 rows)
    assert all(ref() is not None for ref in given) and len({_place(ref()) for ref in given}) == 3


@pytest.mark.parametrize("which", ["tiles", "workspace"])
def test_a_chunk_without_memory_for_the_copy_takes_the_pages(monkeypatch, which):
    """The pool may fill the device: a chunk whose copy has no place is answered all the same."""
    d = Doubles(monkeypatch)
    c = _cache([600, 600])
    tiles = _queries(c, 512, 1)
    empty = torch.empty

    def full(*a, **kw):
        if (which == "tiles") == (kw.get("dtype") == c.dtype):
            raise torch.OutOfMemoryError("no memory")
        return empty(*a, **kw)

    def paged_only(*a, **kw):
        monkeypatch.setattr(torch, "empty", empty)
        return bytes_of(*a, **kw)

    bytes_of = h.paged_workspace_bytes
    monkeypatch.setattr(h, "paged_workspace_bytes", paged_only)
    monkeypatch.setattr(torch, "empty", full)
    c.attend(*tiles, 1)
    assert d.names()[-1] == "sdpa_fwd_paged" and "sdpa_fwd_tile_cache" not in d.names()


@pytest.mark.parametrize("sizes", [dict(max_rows=1 << 31, page_rows=65536), dict(max_rows=(1 << 31) - 15, page_rows=16),
                                   dict(max_rows=1 << 40, page_rows=4096)])
def test_more_rows_than_the_calls_take(sizes):
    """max_pages * page_rows is below 2^31 for every call: refused where the cache is made, not by an append that has
    counted its rows already."""
    with pytest.raises(ValueError, match="below 2\\^31"):
        _cache([0], n_pages=1, n_head_kv=1, packed=False, **sizes)
