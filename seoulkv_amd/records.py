"""A cache of FP8 ``[V || K]`` records for several sequences, and a decoder's
operators around it.

The reference serves one immutable sequence (``README.md:66-69``).  A
``RecordCache`` holds the records of ``dense_decode_static`` for ``batch``
sequences, contiguous or in the pages of a :class:`~seoulkv_amd.paged.KVPagePool`
(those of a paged ``SeoulKV4`` among them), with what changes from step to
step in device memory, so that every call can be captured in a HIP graph:

``lengths``    int32 [batch]: committed tokens of each sequence.  Tokens that
               ``write`` stores lie behind them until the caller raises it
               (``cache.lengths += accepted``).
``positions``  int32 [batch, 4, capacity]: the position of each slot's token.
``weights``    float32 [batch, 4, capacity]: attention weight accumulated by
               ``key_weights``, by which ``evict`` chooses.

One round of speculative decoding::

    q = cache.write(k, v, q=q, table=table, positions=pos)   # drafts, rotated
    out, lse = cache.tree_decode(q, tree)                     # verify them
    cache.key_weights(q, lse, tree)                           # on the steps that count
    ...                                                       # accept some
    cache.write(k_accepted, v_accepted, table=table, positions=pos_accepted)
    cache.lengths += accepted

and, when a cache has grown to its budget, ``cache.evict(smaller, keep)``.
``lengths`` counts slots: after an eviction it is no position any more.

All calls enqueue on PyTorch's current stream and never synchronise; tensors
used on another stream are the caller's to order, as with any torch operator.
Calls may overlap (other streams) unless one writes what another reads.
"""

from __future__ import annotations

import torch

from seoulkv_amd import _hip
from seoulkv_amd.paged import KVPagePool, N_KV_HEADS, RECORD_BYTES
from seoulkv_amd.rope import RotaryTable, _no_grad, _written

N_HEADS, HEAD_DIM = 16, 256
MAX_DRAFTS = 64
MAX_BATCH = 1024
MAX_CAPACITY = 1 << 20


class RecordCache:
    """The records of ``batch`` sequences and what goes with them.

    ``records``: uint8 [batch, 4, capacity, 512] (or [4, capacity, 512], one
    sequence), or with ``page_table`` a :class:`KVPagePool` or its pages
    [n_pages, 4, page_tokens, 512].  ``page_table``: physical page of each
    logical page, [batch, pages per sequence] (nested lists or an int32
    tensor; -1: none; capacity = pages x page_tokens).  Sequences may share
    pages that are only read (``write`` and ``evict`` into such a cache
    raise).  ``lengths``: int32 device tensor [batch], kept, or ints.
    ``positions`` and ``weights``: tensors to keep, or ``None`` to have none.
    The kernels read the kept tensors where they lie: change their values in
    place.  (An int32 ``page_table`` on the device is kept too; the check for
    shared pages is the constructor's.)"""

    _KEPT = ("records", "lengths", "positions", "weights", "page_table", "status")
    _desc = None

    def __setattr__(self, name, value):
        if name in self._KEPT and self._desc is not None and value is not getattr(self, name):
            raise AttributeError(f"change {name} in place: the kernels read this tensor")
        object.__setattr__(self, name, value)

    def __enter__(self):
        self._open()
        return self

    def __exit__(self, exc_type, exc_value, traceback):
        self.close()

    def __init__(self, records, lengths, *, page_table=None, positions=None, weights=None):
        pool = records if isinstance(records, KVPagePool) else None
        if pool is not None:
            records = pool.pages
            if page_table is None:
                raise ValueError("a page pool needs a page_table")
        if not isinstance(records, torch.Tensor) or records.dtype != torch.uint8 or records.device.type != "cuda":
            raise ValueError("expected uint8 records on a GPU")
        if page_table is None and records.dim() == 3:
            records = records.unsqueeze(0)
        if records.dim() != 4 or records.shape[1] != N_KV_HEADS or records.shape[3] != RECORD_BYTES \
                or not records.is_contiguous():
            raise ValueError("expected contiguous records [batch, 4, capacity, 512] or pages "
                             "[n_pages, 4, page_tokens, 512]")
        self._pool, self.records, self.device = pool, records, records.device
        self._index = records.device.index
        self._owned: list[int] = []
        self.shared = False
        if page_table is None:
            self.page_table = None
            self.batch, self.capacity = records.shape[0], records.shape[2]
            self._pages: set[int] | None = None
        else:
            self.page_table = self._checked_table(page_table)
            self.batch = self.page_table.shape[0]
            self.capacity = self.page_table.shape[1] * records.shape[2]
        if not 1 <= self.batch <= MAX_BATCH or not 1 <= self.capacity <= MAX_CAPACITY:
            raise ValueError(f"batch {self.batch} outside [1, {MAX_BATCH}] or capacity {self.capacity} "
                             f"outside [1, 2^20]")
        if not isinstance(lengths, torch.Tensor):
            lengths = torch.tensor([int(n) for n in lengths], dtype=torch.int32, device=self.device)
        self.lengths = self._kept("lengths", lengths, torch.int32, (self.batch,))
        slots = (self.batch, N_KV_HEADS, self.capacity)
        self.positions = self._kept("positions", positions, torch.int32, slots)
        self.weights = self._kept("weights", weights, torch.float32, slots)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._desc = _hip.RecordCacheDesc(
            records=records.data_ptr(), batch=self.batch, capacity=self.capacity,
            n_pages=0 if page_table is None else records.shape[0],
            page_tokens=0 if page_table is None else records.shape[2],
            table_len=0 if page_table is None else self.page_table.shape[1],
            page_table=None if page_table is None else self.page_table.data_ptr(),
            lengths=self.lengths.data_ptr(),
            positions=None if positions is None else self.positions.data_ptr(),
            weights=None if weights is None else self.weights.data_ptr(),
            status=self.status.data_ptr())
        # what this constructor enqueued is done before any stream uses it
        torch.cuda.current_stream(self.device).synchronize()

    @classmethod
    def allocate(cls, batch: int, capacity: int, *, device="cuda", pool: KVPagePool | None = None) -> "RecordCache":
        """An empty cache with positions and weights.  With ``pool`` its
        records live in pages taken from the pool (capacity rounded up to
        whole pages), which go back on :meth:`close`."""
        if type(batch) is not int or type(capacity) is not int or not 1 <= batch <= MAX_BATCH \
                or not 1 <= capacity <= MAX_CAPACITY:
            raise ValueError(f"batch must be an int in [1, {MAX_BATCH}], capacity one in [1, 2^20]")
        table, owned = None, []
        if pool is None:
            records = torch.zeros((batch, N_KV_HEADS, capacity, RECORD_BYTES), dtype=torch.uint8,
                                  device=torch.device(device))
            device = records.device
        else:
            per = pool.pages_for(capacity)
            capacity, device, records = per * pool.page_tokens, pool.device, pool
            owned = pool.allocate(batch * per)
            table = [owned[b * per:(b + 1) * per] for b in range(batch)]
        try:
            slots = (batch, N_KV_HEADS, capacity)
            cache = cls(records, torch.zeros(batch, dtype=torch.int32, device=device), page_table=table,
                        positions=torch.zeros(slots, dtype=torch.int32, device=device),
                        weights=torch.zeros(slots, device=device))
        except Exception:
            if owned:
                pool.release(owned)
            raise
        cache._owned = owned
        return cache

    def close(self) -> None:
        """End the use of this cache: pages that :meth:`allocate` took go back
        to their pool, after the work that uses them; idempotent."""
        self._desc = None
        if self._owned:
            torch.cuda.synchronize(self.device)
            self._pool.release(self._owned)
            self._owned = []

    # --------------------------------------------------------------- checks
    def _checked_table(self, table) -> torch.Tensor:
        host = torch.as_tensor(table).cpu()
        if host.dim() != 2 or host.numel() == 0 or host.dtype not in (torch.int32, torch.int64):
            raise ValueError("expected an integer page_table [batch, pages per sequence]")
        pages = host[host >= 0].tolist()
        if int(host.min()) < -1 or int(host.max()) >= self.records.shape[0]:
            raise ValueError(f"page_table entries must lie in [-1, {self.records.shape[0]})")
        tokens = self.records.shape[2]
        if not 16 <= tokens <= 65536 or tokens & (tokens - 1):
            raise ValueError("page_tokens must be a power of two in [16, 65536]")
        self._pages = set(pages)
        self.shared = len(self._pages) != len(pages)
        if isinstance(table, torch.Tensor) and table.device == self.device and table.dtype == torch.int32 \
                and table.is_contiguous():
            return table  # kept: a later change of its entries is followed
        return host.to(torch.int32).contiguous().to(self.device)

    def _kept(self, name, t, dtype, shape):
        if t is None:
            return None
        if t.dtype != dtype or tuple(t.shape) != shape or t.device != self.device or not t.is_contiguous():
            raise ValueError(f"expected contiguous {dtype} {name} {list(shape)} on {self.device}")
        return t

    def _open(self):
        if self._desc is None:
            raise RuntimeError("RecordCache is closed")
        return self._desc

    def _writable(self):
        if self.shared:
            raise ValueError("sequences of this cache share pages: it can only be read")

    def _rows(self, name, t, heads):
        """A BF16 tensor [batch, n, heads, 256] on this device, its last
        dimension contiguous."""
        shape = t.shape if isinstance(t, torch.Tensor) else ()
        if len(shape) != 4 or shape[0] != self.batch or shape[2] != heads or shape[3] != HEAD_DIM \
                or t.dtype != torch.bfloat16 or t.device != self.device:
            raise ValueError(f"expected BF16 {name} [{self.batch}, n, {heads}, {HEAD_DIM}] on {self.device}")
        return t if t.stride(3) == 1 else t.contiguous()

    def _optional(self, name, t, dtypes, shape):
        if t is None:
            return None
        if not isinstance(t, torch.Tensor) or t.dtype not in dtypes or t.shape != shape or t.device != self.device:
            raise ValueError(f"expected {name} {list(shape)} of {' or '.join(map(str, dtypes))} on {self.device}")
        return t.contiguous()

    def _queries(self, q):
        q = self._rows("q", q, N_HEADS)
        if q.shape[1] > MAX_DRAFTS:
            raise ValueError(f"{q.shape[1]} drafts above {MAX_DRAFTS}")
        b, n, h, _ = q.stride()
        if q.data_ptr() % 16 or (b | n | h) % 8:
            q = q.clone(memory_format=torch.contiguous_format)  # 16-byte rows
        return q

    # ------------------------------------------------------------ operators
    def write(self, k: torch.Tensor, v: torch.Tensor, *, q: torch.Tensor | None = None,
              table: RotaryTable | None = None, positions: torch.Tensor | None = None,
              counts: torch.Tensor | None = None, q_out: torch.Tensor | None = None) -> torch.Tensor | None:
        """Store n tokens of every sequence in slots ``lengths[b] ..``: V, and
        K turned by ``table`` (``None``: as given) to ``positions`` (int32 or
        int64 [batch, n]; default ``lengths[b] + i``, which is right as long as
        slots are positions: not after an eviction), each rounded once to FP8; the slots' positions are set and their weights zeroed.  ``k``,
        ``v``: BF16 [batch, n, 4, 256], any strides with a contiguous last
        dimension.  ``q`` (BF16 [batch, n, 16, 256]) is turned likewise and
        returned (in ``q_out`` if given, which may be ``q``; not over ``k`` or ``v``).  ``counts``
        (int32 [batch]): only the first ``counts[b]`` tokens are stored.
        Tokens past the capacity are dropped and reported by
        :meth:`synchronize`.  ``lengths`` does not change."""
        desc = self._open()
        self._writable()
        k, v = self._rows("k", k, N_KV_HEADS), self._rows("v", v, N_KV_HEADS)
        n = k.shape[1]
        if v.shape[1] != n:
            raise ValueError("k and v hold different numbers of tokens")
        if n > self.capacity:
            raise ValueError(f"{n} tokens for a capacity of {self.capacity}")
        if q is not None:
            q = self._rows("q", q, N_HEADS)
            if q.shape[1] != n:
                raise ValueError("q and k hold different numbers of tokens")
            if q_out is None:
                q_out = q.new_empty(q.shape)
            elif q_out.stride(-1) != 1 or self._rows("q_out", q_out, N_HEADS).shape != q.shape:
                raise ValueError("q_out must be like q, its last dimension contiguous")
        elif q_out is not None:
            raise ValueError("q_out without q")
        if table is not None and (not isinstance(table, RotaryTable) or table.device != self.device
                                  or table.rotary_dim > HEAD_DIM):
            raise ValueError(f"expected a RotaryTable of at most {HEAD_DIM} elements on {self.device}")
        positions = self._optional("positions", positions, (torch.int32, torch.int64), (self.batch, n))
        if positions is not None and self.positions is not None and \
                positions.untyped_storage().data_ptr() == self.positions.untyped_storage().data_ptr():
            positions = positions.clone()  # slots' own positions change while they are read
        counts = self._optional("counts", counts, (torch.int32,), (self.batch,))
        _no_grad("write", k, v, q, q_out, self.weights)
        if n == 0:
            return q_out
        _hip.call_on(self._index, "skv_cache_write", desc, None if table is None else table._desc,
                     _hip.rows_desc(k), _hip.rows_desc(v), None if q is None else _hip.rows_desc(q),
                     None if q is None else _hip.rows_desc(q_out), n, _hip.pointer(positions),
                     positions is not None and positions.dtype == torch.int64, _hip.pointer(counts))
        _written(self.records, self.positions, self.weights, q_out)
        return q_out

    def tree_decode(self, q: torch.Tensor, tree: torch.Tensor | None = None, *,
                    counts: torch.Tensor | None = None, cap: float = 0.0,
                    out: torch.Tensor | None = None, lse: torch.Tensor | None = None):
        """Attention of n <= 64 drafted tokens of every sequence (``q``: BF16
        [batch, n, 16, 256]) over its committed slots and over the drafts
        stored behind them: row i sees draft j where bit j of ``tree[b][i]``
        (int64 [batch, n]) is set; default: a chain, j <= i.  ``counts`` (int32
        [batch]): drafts of each sequence; the rows behind them are padding.
        ``cap`` > 0: scores ``q.k / 16`` become ``cap * tanh(score / cap)``.
        Returns ``(out, lse)``: BF16 [batch, n, 16, 256] and float32 [batch,
        n, 16], the log of the sum of exp(score); 0 and -inf for a row that
        sees nothing."""
        desc = self._open()
        q = self._queries(q)
        n = q.shape[1]
        tree = self._optional("tree", tree, (torch.int64,), (self.batch, n))
        counts = self._optional("counts", counts, (torch.int32,), (self.batch,))
        _no_grad("tree_decode", q, out, lse)
        given = out, lse
        if out is None:
            out = q.new_empty((self.batch, n, N_HEADS, HEAD_DIM))
        elif not out.is_contiguous() or self._rows("out", out, N_HEADS).shape[1] != n:
            raise ValueError("out must be contiguous and like q")
        if lse is None:
            lse = q.new_empty((self.batch, n, N_HEADS), dtype=torch.float32)
        else:
            self._kept("lse", lse, torch.float32, (self.batch, n, N_HEADS))
        if n == 0:
            return out, lse
        size = _hip.load_library().skv_tree_workspace(self.batch, n)
        work = q.new_empty(size, dtype=torch.uint8)
        _hip.call_on(self._index, "skv_tree_decode", desc, _hip.rows_desc(q), n, _hip.pointer(tree),
                     _hip.pointer(counts), cap, out.data_ptr(), lse.data_ptr(), work.data_ptr(), size)
        _written(*given)
        return out, lse

    def key_weights(self, q: torch.Tensor, lse: torch.Tensor, tree: torch.Tensor | None = None, *,
                    counts: torch.Tensor | None = None, cap: float = 0.0, accumulate: bool = True) -> None:
        """Add to ``weights[b][g][t]`` the attention weight exp(score - lse)
        that the rows of :meth:`tree_decode` (same arguments; ``lse``: its
        result) and the 4 query heads of KV head g give slot t; with
        ``accumulate=False`` replace it (slots past the drafts stay).  The
        cache has to be as it was then: ``lse`` belongs to those lengths and
        records."""
        desc = self._open()
        if self.weights is None:
            raise ValueError("the cache has no weights")
        q = self._queries(q)
        n = q.shape[1]
        tree = self._optional("tree", tree, (torch.int64,), (self.batch, n))
        counts = self._optional("counts", counts, (torch.int32,), (self.batch,))
        lse = self._optional("lse", lse, (torch.float32,), (self.batch, n, N_HEADS))
        if lse is None:
            raise ValueError("key_weights needs tree_decode's lse")
        _no_grad("key_weights", q, lse, self.weights)
        if n == 0:
            raise ValueError("key_weights needs at least one row")
        _hip.call_on(self._index, "skv_key_weights", desc, _hip.rows_desc(q), n, lse.data_ptr(),
                     _hip.pointer(tree), _hip.pointer(counts), cap, bool(accumulate))
        _written(self.weights)

    def evict(self, to: "RecordCache", keep: int, *, sink: int = 128, local: int = 256) -> None:
        """Copy what stays of every sequence and KV head into ``to`` (same
        batch, other memory), in slot order: at most ``keep`` slots, the first
        ``sink``, the last ``local`` committed ones and of the rest the
        heaviest by ``weights`` (ties: the lowest slot; NaN counts least).
        Slots whose page is none hold no key: they are passed over and count
        nowhere.  Records, positions and weights go along and ``to.lengths``
        is set; this cache does not change.  What falls on a slot of ``to``
        without a page is dropped and reported by ``to.synchronize()``.  Heads
        keep different tokens: ``to.positions`` says which (needs positions in
        both caches); the position after the last is not ``to.lengths``."""
        if not isinstance(to, RecordCache):
            raise TypeError("expected a RecordCache to evict into")
        desc, to_desc = self._open(), to._open()
        if self.weights is None:
            raise ValueError("the cache has no weights")
        if to.device != self.device or to.batch != self.batch:
            raise ValueError("both caches must hold as many sequences on one device")
        if any(type(x) is not int for x in (keep, sink, local)) or min(sink, local) < 0 or keep < 1 \
                or sink + local > keep or keep > to.capacity:
            raise ValueError(f"keep {keep} must hold sink {sink} + local {local} and fit the capacity "
                             f"{to.capacity}")
        to._writable()
        _no_grad("evict", self.weights, to.weights)
        if self._pages is not None and to._pages is not None and \
                self.records.data_ptr() == to.records.data_ptr() and not self._pages.isdisjoint(to._pages):
            raise ValueError("the two caches share pages")
        size = _hip.load_library().skv_evict_workspace(self.batch, self.capacity, keep)
        work = torch.empty(size, dtype=torch.uint8, device=self.device)
        _hip.call_on(self._index, "skv_evict", desc, to_desc, keep, sink, local, work.data_ptr(), size)
        _written(to.records, to.positions if self.positions is not None else None, to.weights, to.lengths)

    def synchronize(self) -> None:
        """Wait for the device; raise if a write or an eviction into this cache
        since the last call dropped tokens (past the capacity, or without a
        page)."""
        torch.cuda.synchronize(self.device)
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            what = [t for b, t in ((1, "past the capacity"), (2, "without a page")) if bits & b]
            raise RuntimeError(f"RecordCache dropped tokens {' and '.join(what)}")
