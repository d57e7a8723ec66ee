"""PagedKVCache on streams that are not the current one."""
import pytest
import torch

from nntile_amd.kv_cache import PagedKVCache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("causal", [True, False])
def test_a_chunk_that_is_read_back_on_another_stream(packed, causal):
    """512 queries of a head: read back and given to the tile kernels.  Queries that the caller lets go right behind the
    call keep their memory until the stream is past it."""
    g = torch.Generator().manual_seed(70)
    c, d = (PagedKVCache(40, 64, 2, 600, 2, 64, packed=packed) for _ in range(2))
    k, v = (torch.randn(4, 512, 64, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    q = torch.randn(4, 512, 64, generator=g).to(torch.bfloat16).cuda()
    results = []
    side = torch.cuda.Stream()
    for cache, stream in ((c, None), (d, side)):
        Q, lse, A = q.clone(), torch.empty(4, 512, device="cuda"), torch.empty_like(q)
        side.wait_stream(torch.cuda.current_stream())
        cache.append_attend(k, v, Q, lse, A, 1, causal=causal, stream=stream)
        place = Q.data_ptr()
        del Q
        if stream is not None:
            # the allocator may not give it to the current stream while `side` is under way
            with torch.cuda.stream(side):
                busy = torch.cuda.Event()
                busy.record()
            again = torch.full_like(q, float("nan"))
            assert again.data_ptr() != place or busy.query()
            torch.cuda.current_stream().wait_stream(side)
        results.append((A, lse) + cache.read(stream=stream))
        torch.cuda.synchronize()
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("packed", [False, True])
def test_a_chunk_that_is_kept_to_the_pages(packed):
    """NaN among the newest values: with DENSE_ROWS out of reach the tokens before do not notice."""
    g = torch.Generator().manual_seed(71)
    c = PagedKVCache(20, 64, 1, 600, 1, 64, packed=packed)
    c.DENSE_ROWS = 1 << 62
    q_seq, group = 200, 4
    k, v = (torch.randn(1, q_seq, 64, generator=g).to(torch.bfloat16) for _ in range(2))
    v[0, q_seq - 3, 5] = float("nan")
    Q = torch.randn(group, q_seq, 64, generator=g).to(torch.bfloat16).cuda()
    lse, A = torch.empty(group, q_seq, device="cuda"), torch.empty_like(Q)
    c.append_attend(k.cuda(), v.cuda(), Q, lse, A, group)
    odd = A.isnan().any(-1)
    assert not odd[:, :-3].any() and odd[:, -3:].all() and not lse.isnan().any()
