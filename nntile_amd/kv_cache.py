"""Key/value cache of the decode path, on the HIP entry points.

Mirror of `KVCache` (wrappers/python/nntile/layer/cache_utils.py:117-225) and
of the way `LlamaAttention.forward_dynamic` uses it
(wrappers/python/nntile/model/llama_attention.py:518-531, 643-731): tensors
preallocated with `max_cache_size` rows on the sequence axis, `append` writes
the new rows behind the filled ones, `len()` is the number of filled rows.

What differs, on purpose: the reference copies the filled part of both caches
into fresh dense tensors before every attention call (`k_partial`,
`v_partial`) and materialises a bool mask slice for the new queries; here
`attend` hands the caches to the decode kernel with their capacity and the
visibility rule `key <= query + (len - q_seq)`, so a decode step reads the
filled rows once and writes only the new ones; `append_attend` does the
append and the attention of a decode step in one launch.

Tensors are C-ordered torch device tensors: K, V `[entries, seq, head]`
(entries = n_batch * n_head_kv, NNTile's `[head, seq, n_batch, n_head_kv]`),
Q, A `[entries * kv_group, q_seq, head]`.
"""
import torch

from . import hip_sdpa


class KVCache:
    def __init__(self, max_cache_size, seq_size_dim=1):
        if seq_size_dim != 1:
            # [head, seq, ...] is the only layout the attention path uses
            raise ValueError("the sequence axis of an attention tile is axis 1")
        self.max_cache_size = int(max_cache_size)
        self.seq_size_dim = seq_size_dim
        self.k = None
        self.v = None
        self.k_cache_size = 0
        self.v_cache_size = 0
        self._workspace = None

    def __len__(self):
        return self.k_cache_size

    def _init_from_tensor(self, t):
        entries, _, head = t.shape
        return torch.zeros((entries, self.max_cache_size, head), dtype=t.dtype, device=t.device)

    def append(self, k_partial, v_partial, stream=None):
        """Write the new rows behind the filled ones.  More rows than the cache
        has left raise (the reference raises in
        LlamaAttention._append_to_kv_cache); nothing is written then."""
        if k_partial.shape[1] != v_partial.shape[1]:
            raise ValueError("k and v must bring the same number of tokens")
        if self.k is None:
            self.k = self._init_from_tensor(k_partial)
            self.v = self._init_from_tensor(v_partial)
        rows = k_partial.shape[1]
        if rows + self.k_cache_size > self.max_cache_size:
            raise hip_sdpa.SdpaError(
                hip_sdpa.EINVAL,
                "kv_cache_append: overload internal state: try add %d to %d, max: %d"
                % (rows, self.k_cache_size, self.max_cache_size))
        hip_sdpa.kv_cache_append(k_partial, v_partial, self.k, self.v, self.k_cache_size,
                                 stream=stream)
        self.k_cache_size += rows
        self.v_cache_size += rows

    def append_attend(self, k_partial, v_partial, Q, lse, A, n_batch, kv_group, causal=True,
                      mask=None, stream=None):
        """`append` followed by `attend`, same results bit for bit; on the
        decode kernels' shapes the two are ONE launch (the
        attention reads the new rows from k_partial / v_partial while other
        workgroups of the launch write them into the caches)."""
        if mask is None and stream is None:
            mode = hip_sdpa.MASK_CAUSAL if causal else hip_sdpa.MASK_NONE
            step = hip_sdpa._native().cache_step
            rc = step(self.k, self.v, k_partial, v_partial, Q, lse, A, self.k_cache_size,
                      self.max_cache_size, n_batch, kv_group, mode, hip_sdpa.OVERWRITE,
                      self._workspace, None)
            if rc == hip_sdpa.OK:
                self._mask_in_use = None
                rows = k_partial.shape[1]
                self.k_cache_size += rows
                self.v_cache_size += rows
                return
            # (what is left - a first call, a larger workspace, other shapes,
            # a call to be refused - takes the long way below)
        rows, q_seq = k_partial.shape[1], Q.shape[1]
        one_launch = (self.k is not None and v_partial.shape[1] == rows
                      and kv_group * q_seq <= 64 and Q.shape[2] in (64, 128)
                      and rows + self.k_cache_size <= self.max_cache_size
                      and k_partial.is_contiguous() and v_partial.is_contiguous())
        if not one_launch:
            self.append(k_partial, v_partial, stream=stream)
            self.attend(Q, lse, A, n_batch, kv_group, causal=causal, mask=mask, stream=stream)
            return
        k_seq = self.k_cache_size + rows
        mode = hip_sdpa.MASK_CAUSAL if causal else hip_sdpa.MASK_NONE
        sliced = None
        if mask is not None:
            # (the slice that goes with the cache as it will be after the append)
            sliced, mode = self._mask_slice_for(mask, q_seq, k_seq), hip_sdpa.MASK_BOOL
        if stream is not None:
            for t in (sliced, k_partial, v_partial):
                if t is not None:
                    t.record_stream(stream)
        self._mask_in_use = sliced
        workspace = self._decode_workspace(k_seq, Q, n_batch, kv_group, stream)
        hip_sdpa.sdpa_fwd_decode_append_cache(
            k_partial, v_partial, self.k, self.v, k_seq, Q, sliced, lse, A, mode, n_batch, kv_group,
            workspace, causal_offset=k_seq - q_seq, flags=hip_sdpa.OVERWRITE, stream=stream)
        # (only now: a refused call leaves the cache as it was)
        self.k_cache_size += rows
        self.v_cache_size += rows

    def _decode_workspace(self, k_seq, Q, n_batch, kv_group, stream):
        need = hip_sdpa.decode_cache_workspace_bytes(k_seq, Q, n_batch, kv_group)
        if self._workspace is None or self._workspace.numel() < need:
            # (a launch of an earlier call may still read the old workspace:
            # it is kept until the one after next replaces it)
            self._retired_workspace = self._workspace
            self._workspace = torch.empty(need, dtype=torch.uint8, device=Q.device)
        if stream is not None:
            self._workspace.record_stream(stream)
        return self._workspace

    @property
    def k_partial(self):
        """The filled rows, as a view (the reference returns a copy)."""
        return self.k[:, :self.k_cache_size]

    @property
    def v_partial(self):
        return self.v[:, :self.v_cache_size]

    def clear(self):
        self.k = None
        self.v = None
        self.k_cache_size = 0
        self.v_cache_size = 0
        self._workspace = None

    def mask_slice(self, mask, q_seq):
        """The mask rows that go with the last q_seq tokens of the cache
        (Sdpa._prepare_mask_for_kv_cache, wrappers/python/nntile/layer/sdpa.py:
        489-531).  mask: bool device tensor [queries, keys] in C order (the
        reference's [keys, queries]), True = visible.  A mask that already is
        [q_seq, len] is used as it is; otherwise everything is visible except
        where the mask, read at query position len - q_seq + j, says
        otherwise."""
        return self._mask_slice_for(mask, q_seq, len(self))

    @staticmethod
    def _mask_slice_for(mask, q_seq, k_seq):
        if tuple(mask.shape) == (q_seq, k_seq):
            return mask.contiguous()
        out = torch.ones((q_seq, k_seq), dtype=torch.bool, device=mask.device)
        first = k_seq - q_seq
        rows = max(0, min(q_seq, mask.shape[0] - first))
        cols = min(k_seq, mask.shape[1])
        if rows > 0 and cols > 0 and first >= 0:
            out[:rows, :cols] = mask[first:first + rows, :cols]
        return out

    def attend(self, Q, lse, A, n_batch, kv_group, causal=True, mask=None, stream=None):
        """A = attention of Q over the filled rows; the q_seq queries are the
        last q_seq tokens of the cache (append first).  lse and A are
        overwritten.  mask: None (the causal rule when `causal`, else nothing
        hidden) or a bool mask as for `mask_slice`, whose slice is then passed
        as values.  Few rows (kv_group * q_seq <= 64, head 64 or 128) take the
        split-key decode kernel of the tile type, everything else - longer
        chunks, head 32 - the tile kernel, which shares its key axis out over
        workgroups where the chunk's rows do not fill the chip; both read the
        caches in place."""
        k_seq = len(self)
        q_seq = Q.shape[1]
        mode = hip_sdpa.MASK_CAUSAL if causal else hip_sdpa.MASK_NONE
        sliced = None
        if mask is not None:
            sliced, mode = self.mask_slice(mask, q_seq), hip_sdpa.MASK_BOOL

        def keep(t):
            # The kernels are enqueued behind torch's back; its allocator does
            # not know they read t.  On a stream other than the current one the
            # allocator is told; in every case the tensor stays referenced
            # here until the next call.
            if stream is not None and t is not None:
                t.record_stream(stream)
            return t

        self._mask_in_use = keep(sliced)
        decode = kv_group * q_seq <= 64 and Q.shape[2] in (64, 128)
        if not decode:
            need = hip_sdpa.tile_cache_workspace_bytes(k_seq, Q, mode)
            workspace = None
            if need:
                # (its own for each call, in the memory of the call's stream:
                # calls on several streams may overlap)
                with torch.cuda.stream(stream):
                    workspace = torch.empty(need, dtype=torch.uint8, device=Q.device)
            hip_sdpa.sdpa_fwd_tile_cache(
                self.k, self.v, k_seq, Q, sliced, lse, A, mode, n_batch, kv_group,
                causal_offset=k_seq - q_seq, flags=hip_sdpa.OVERWRITE, stream=stream,
                workspace=workspace)
            return
        workspace = self._decode_workspace(k_seq, Q, n_batch, kv_group, stream)
        hip_sdpa.sdpa_fwd_decode_cache(
            self.k, self.v, k_seq, Q, sliced, lse, A, mode, n_batch, kv_group, workspace,
            causal_offset=k_seq - q_seq, flags=hip_sdpa.OVERWRITE, stream=stream)


class PagedKVCache:
    """Key/value cache whose sequences have lengths of their own: rows lie in
    pages of a pool that all sequences share, as they are or in 8 bits (e4m3 with
    one power of two per row).  What `KVCache` does for a batch of equal lengths,
    for a batch that is served: sequences end (`release`) and their pages go to others.

    Tensors as for `KVCache`: K, V `[n_head_kv * n_batch, rows, head]`, Q, A
    `[n_head_kv * kv_group * n_batch, q_seq, head]`, entry = sequence + n_batch *
    head index.  The lengths are known to the host, which hands out the pages;
    the kernels read lengths and page table on the device.  A caller that
    captures its steps calls hip_sdpa.paged_kv_append / sdpa_fwd_paged with
    `table` and a `lens` of its own instead: this class's bookkeeping would run once,
    at the capture.  Calls of one cache share its workspace: they belong on one stream,
    or are ordered by the caller.
    """

    def __init__(self, n_pages, page_rows, n_batch, max_rows, n_head_kv, head, dtype=torch.bfloat16,
                 packed=False, device="cuda"):
        if page_rows < 16 or page_rows > 65536 or page_rows & (page_rows - 1):
            raise ValueError("page_rows is a power of two from 16 to 65536")
        if min(n_pages, n_batch, max_rows, n_head_kv) < 1 or head not in (64, 128):
            raise ValueError("a cache needs pages, sequences, rows and heads of size 64 or 128")
        if -(-max_rows // page_rows) * page_rows > 0x7fffffff or n_batch * n_head_kv > 0x7fffffff:
            raise ValueError("the rows of a sequence's pages, and sequences times heads, are below 2^31")
        hip_sdpa.dtype_name(torch.empty(0, dtype=dtype))
        if packed and dtype == torch.float32:
            raise TypeError("8-bit pages hold bf16 and fp16 tiles")
        self.dtype, self.packed = dtype, bool(packed)
        self.n_batch, self.n_head_kv, self.head = n_batch, n_head_kv, head
        self.page_rows, self.max_pages = page_rows, -(-max_rows // page_rows)
        # (a page's keys and values behind each other)
        shape = (n_pages, 2, n_head_kv, page_rows, head)
        pool = torch.zeros(shape, dtype=torch.uint8 if packed else dtype, device=device)
        self.pool = pool.view(torch.float8_e4m3fn) if packed else pool
        self.k_pages, self.v_pages = self.pool[:, 0], self.pool[:, 1]
        self.scales = torch.ones(shape[:4], dtype=torch.uint8, device=device) if packed else None
        self.k_scales, self.v_scales = (self.scales[:, 0], self.scales[:, 1]) if packed else (None, None)
        self.table = torch.full((n_batch, self.max_pages), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(n_batch, dtype=torch.int32, device=device)
        self.lengths = [0] * n_batch
        self._pages = [[] for _ in range(n_batch)]
        self._free = list(range(n_pages - 1, -1, -1))
        self._workspace, self._old_workspaces = None, []

    @property
    def free_pages(self):
        return len(self._free)

    def _counts(self, rows, new_rows):
        if new_rows is None:
            return [rows] * self.n_batch
        counts = [int(c) for c in new_rows]
        if len(counts) != self.n_batch or min(counts) < 0 or max(counts) > rows:
            raise ValueError("new_rows are the new tokens of every sequence, at most the tile's rows")
        return counts

    def _upload(self, target, values, stream):
        """Host values into a device tensor, ordered on `stream`."""
        host = torch.tensor(values, dtype=torch.int32).pin_memory()
        with torch.cuda.stream(stream):
            target.copy_(host, non_blocking=True)
        if stream is not None:
            target.record_stream(stream)

    def _in_use(self, stream, *tensors):
        """The cache's tensors and these are in use on a stream that is given: memory of
        theirs that is freed waits for it."""
        if stream is not None:
            for t in (self.pool, self.scales, self.table, self.lens) + tensors:
                if t is not None:
                    t.record_stream(stream)

    def _reserve(self, counts, stream):
        wanted = []
        for n, count in enumerate(counts):
            rows = self.lengths[n] + count
            if rows > self.max_pages * self.page_rows:
                raise hip_sdpa.SdpaError(hip_sdpa.EINVAL, "paged_kv_append: sequence %d: %d rows, max: %d"
                                         % (n, rows, self.max_pages * self.page_rows))
            wanted.append(max(0, -(-rows // self.page_rows) - len(self._pages[n])))
        if sum(wanted) > len(self._free):
            raise hip_sdpa.SdpaError(hip_sdpa.EINVAL, "paged_kv_append: %d pages wanted, %d free"
                                     % (sum(wanted), len(self._free)))
        if any(wanted):
            for n, count in enumerate(wanted):
                self._pages[n] += [self._free.pop() for _ in range(count)]
            self._upload(self.table, [p + [-1] * (self.max_pages - len(p)) for p in self._pages], stream)

    def append(self, k, v, new_rows=None, stream=None):
        """Write k, v ([n_head_kv * n_batch, rows, head]) behind the rows of the
        sequences; new_rows: how many of `rows` each brings (a list; None: all).
        More rows than a sequence may have, or than there are pages, raise;
        nothing is changed then."""
        if (k.dim() != 3 or k.shape != v.shape or k.dtype != self.dtype or v.dtype != self.dtype
                or k.shape[0] != self.n_head_kv * self.n_batch or k.shape[2] != self.head):
            raise ValueError("k and v are tiles [n_head_kv * n_batch, rows, head] of the cache's type")
        for t in (k, v):
            if not (t.is_cuda and t.is_contiguous() and t.device == self.lens.device
                    and t.device.index == torch.cuda.current_device()):
                raise ValueError("tiles must be contiguous device tensors of the cache's device, "
                                 "which is the current one")
            if t.data_ptr() % 16:
                raise ValueError("tiles start at multiples of 16 bytes")
        rows = k.shape[1]
        counts = self._counts(rows, new_rows)
        self._reserve(counts, stream)
        lengths = [length + count for length, count in zip(self.lengths, counts)]
        uniform = new_rows is None
        if uniform:
            with torch.cuda.stream(stream):
                self.lens.add_(rows)
            given = None
        else:
            self._upload(self.lens, lengths, stream)
            given = self._on_device(counts, stream)
        self._in_use(stream, k, v)
        hip_sdpa.paged_kv_append(k, v, self.k_pages, self.v_pages, self.table, self.lens, self.k_scales,
                                 self.v_scales, new_rows=given, stream=stream)
        self.lengths = lengths

    def _on_device(self, counts, stream):
        with torch.cuda.stream(stream):
            t = torch.empty(self.n_batch, dtype=torch.int32, device=self.lens.device)
        self._upload(t, counts, stream)
        return t

    def read(self, first=0, rows=None, stream=None):
        """Rows [first, first + rows) of every sequence as dense tiles (K, V) of the
        cache's type; rows behind a sequence's last are zeros.  rows None: up to
        the longest sequence's end."""
        rows = max(0, max(self.lengths) - first) if rows is None else rows
        with torch.cuda.stream(stream):
            k = torch.empty((self.n_head_kv * self.n_batch, rows, self.head), dtype=self.dtype,
                            device=self.lens.device)
            v = torch.empty_like(k)
        self._in_use(stream)
        hip_sdpa.paged_kv_read(self.k_pages, self.v_pages, self.table, self.lens, k, v, first=first,
                               k_scales=self.k_scales, v_scales=self.v_scales, stream=stream)
        return k, v

    @property
    def k_partial(self):
        """The filled rows of the keys (a copy, as the reference's)."""
        return self.read()[0]

    @property
    def v_partial(self):
        return self.read()[1]

    # Queries of a key/value head from which a chunk of a batch of equal lengths is worth the copy
    # that the tile kernels' denser products need: one number for all types and sizes, on either side of
    # where they meet (us over the pages, read back).  bf16, 8 heads of 128, 4 x 2048 rows: 256 queries
    # 36.3, 47.9, 512 50.1, 46.9, 1024 95.1, 54.0; one sequence of 4096: 512 34.0, 37.8, 1024 50.9, 41.1.
    # fp32, 12 heads of 64, 2 x 2048: 128 31.1, 33.8, 256 56.2, 45.2, 512 93.4, 53.5.
    DENSE_ROWS = 512

    def _read_back(self, length, Q, mode, stream):
        """Dense keys and values for the tile kernels, and their workspace; None where the pool
        leaves no memory for them."""
        try:
            k, v = self.read(rows=length, stream=stream)
            need = hip_sdpa.tile_cache_workspace_bytes(length, Q, mode)
            if not need:
                return k, v, None
            with torch.cuda.stream(stream):
                return k, v, torch.empty(need, dtype=torch.uint8, device=Q.device)
        except torch.OutOfMemoryError:
            return None

    def attend(self, Q, lse, A, kv_group, causal=True, new_rows=None, stream=None):
        """A = attention of Q over the sequences' rows; the queries of a sequence are
        its newest tokens (append first), the first new_rows of q_seq (a list; None:
        all).  lse and A are overwritten; queries without a visible row get
        lse = -inf, A = 0.  What lies in rows that a query does not see does not reach it,
        but for chunks of DENSE_ROWS queries and more, which go through the tile kernels:
        there a NaN or an infinity among the values of a newer token may make tokens just
        before it NaN.  A larger DENSE_ROWS keeps a cache to its pages."""
        q_seq = Q.shape[1]
        counts = self._counts(q_seq, new_rows)
        mode = hip_sdpa.MASK_CAUSAL if causal else hip_sdpa.MASK_NONE
        length = self.lengths[0]
        self._in_use(stream, Q, lse, A)
        if (kv_group * q_seq >= self.DENSE_ROWS and new_rows is None and length >= q_seq
                and min(self.lengths) == max(self.lengths)):
            dense = self._read_back(length, Q, mode, stream)
            if dense is not None:
                k, v, workspace = dense
                hip_sdpa.sdpa_fwd_tile_cache(k, v, length, Q, None, lse, A, mode, n_batch=self.n_batch,
                                             kv_group=kv_group, causal_offset=length - q_seq,
                                             flags=hip_sdpa.OVERWRITE, stream=stream, workspace=workspace)
                return
        given = None if new_rows is None else self._on_device(counts, stream)
        need = hip_sdpa.paged_workspace_bytes(Q, self.n_batch, kv_group)
        if self._workspace is None or self._workspace.numel() < need:
            # (a launch of an earlier call, on whatever stream, may still use the old one; there are three sizes)
            self._old_workspaces.append(self._workspace)
            with torch.cuda.stream(stream):
                self._workspace = torch.empty(need, dtype=torch.uint8, device=Q.device)
        if stream is not None:
            self._workspace.record_stream(stream)
        hip_sdpa.sdpa_fwd_paged(self.k_pages, self.v_pages, self.table, self.lens, Q, lse, A, mode,
                                kv_group, self._workspace, k_scales=self.k_scales, v_scales=self.v_scales,
                                new_rows=given, flags=hip_sdpa.OVERWRITE, stream=stream)

    def append_attend(self, k, v, Q, lse, A, kv_group, causal=True, new_rows=None, stream=None):
        """`append` followed by `attend`: a generation step."""
        self.append(k, v, new_rows=new_rows, stream=stream)
        self.attend(Q, lse, A, kv_group, causal=causal, new_rows=new_rows, stream=stream)

    def release(self, n, stream=None):
        """Sequence n is over: its pages are free for others."""
        self._free += reversed(self._pages[n])
        self._pages[n] = []
        self.lengths[n] = 0
        self._upload(self.lens, self.lengths, stream)
        self._upload(self.table, [p + [-1] * (self.max_pages - len(p)) for p in self._pages], stream)
