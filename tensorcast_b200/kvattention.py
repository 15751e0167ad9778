"""Attention over the paged KV pool, and eviction from it by accumulated attention weight.

Both work on the pool and the tables of ``kvcache.KvWorkload`` (a token row of a page is
``kv_heads`` rows of ``head_dim`` 16-bit values; plane ``2 * layer`` holds a layer's keys,
``2 * layer + 1`` its values), beside ``kvcache.KvGatherHash``:

* ``KvAttention.run`` lets the newest tokens of every sequence attend over the sequence's pages
  (tcx_kv_attention): one query token per sequence (decode) or several (a prompt, a chunk of one,
  speculated tokens), with a sliding window and first tokens that stay visible, behind a prefix
  that all sequences share, and with every token's softmax weight added to accumulators;
* ``KvEvict.run`` keeps each sequence's first, newest and heaviest tokens by those accumulators
  and copies them to new pages (tcx_kv_evict).

An object holds the tables of one batch on the device. ``seq_tokens`` (and ``prefix_tokens``) are
read on the device by every call, so a program lets a sequence grow by writing them in place, up
to the pages' capacity, also between the replays of a captured call; page tables may be written in
place likewise. Every object has its own copy of the lengths, made from ``w.seq_tokens``: where one
object's sequences have grown, another one (the eviction behind some steps of decode, say) is given
them by ``other.seq_tokens.copy_(grown.seq_tokens)``. The object must live as long as a graph that captured its calls. Everything is
inference: no gradients.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

from . import _native
from .kvcache import KvWorkload

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_STATUS = {1: "page slot outside the pool", 2: "more tokens than the sequence's pages hold",
           3: "budget past the destination pages", 4: "a copy into shared memory did not arrive"}


_raw_stream = torch._C._cuda_getCurrentRawStream  # by device index, without building a Stream
_capturing = torch._C._cuda_isCurrentStreamCapturing


def _refuse(message: str):
    raise _native.TcxInvalidArgument(_native.INVALID_ARGUMENT, message)


def _cuda_device(device) -> torch.device:
    d = torch.device(device)
    if d.type != "cuda":
        _refuse(f"device must be a CUDA device, got {d}")
    return d if d.index is not None else torch.device("cuda", torch.cuda.current_device())


def _slots(table, what: str) -> np.ndarray:
    """Page slots in 32 bits; -1, a usual mark of an unused entry, becomes one outside of every pool."""
    t = np.asarray(table)
    for slot in (int(t.min()), int(t.max())) if t.size else ():
        if not -(1 << 31) <= slot < 1 << 32:
            _refuse(f"{what}: page slot {slot} does not fit 32 bits")
    return t.astype(np.uint32)


def _check_tables(w: KvWorkload, what: str) -> None:
    offs = np.asarray(w.page_offsets).astype(np.int64)
    if offs.size != w.n_seq + 1 or offs[0] != 0 or (np.diff(offs) < 0).any():
        _refuse(f"{what}: page_offsets must start at 0 and not decrease")
    if int(offs[-1]) != np.asarray(w.page_table).size:
        _refuse(f"{what}: page_offsets end at {int(offs[-1])}, the page table has {np.asarray(w.page_table).size}")
    _slots(w.page_table, what)
    tokens = np.asarray(w.seq_tokens).astype(np.int64)
    if (tokens < 0).any():
        _refuse(f"{what}: seq_tokens must not be negative")
    if (tokens > np.diff(offs) * w.page_tokens).any():
        _refuse(f"{what}: a sequence has more tokens than its pages hold")


class _Tables:
    """Device tables of one object, in one allocation."""

    def __init__(self, device, arrays: dict):
        sizes = {k: -(-v.nbytes // 16) * 16 for k, v in arrays.items()}
        host = np.zeros(max(sum(sizes.values()), 16), np.uint8)
        at = 0
        for k, v in arrays.items():
            host[at:at + v.nbytes] = np.ascontiguousarray(v).view(np.uint8).reshape(-1)
            at += sizes[k]
        self.buffer = torch.from_numpy(host).to(device)
        at = 0
        for k, v in arrays.items():
            setattr(self, k, self.buffer[at:at + v.nbytes].view(torch.int64 if v.itemsize == 8 else torch.int32))
            at += sizes[k]


class _OnDevice:
    """Stream, device and status handling of a call."""

    def _bind(self, w: KvWorkload, tables: dict) -> _Tables:
        t = self._tables = _Tables(self.device, tables)
        self._pool_bytes = w.planes * w.pool_pages * w.page_tokens * w.token_bytes
        self._stream = _raw_stream(self.device.index)  # the stream whose order the tables' memory follows
        self.status = t.status
        return t

    def _on(self, stream, call):
        """`call` with this object's device current and, where one is given, on `stream`."""
        handle = getattr(stream, "cuda_stream", stream)
        with torch.cuda.device(self.device):
            if handle is None:
                return call()
            s = torch.cuda.ExternalStream(handle, self.device) if handle else torch.cuda.default_stream(self.device)
            with torch.cuda.stream(s):
                return call()

    def _current(self) -> int:
        """The current stream. The tables outlive what runs on it now, also where it is not their own."""
        raw = _raw_stream(self.device.index)
        if raw != self._stream and not _capturing():
            self._tables.buffer.record_stream(torch.cuda.current_stream(self.device))
        return raw

    def check_status(self) -> None:
        """Waits for the device, all its streams, and raises what a call has recorded since the last check."""
        torch.cuda.synchronize(self.device)
        code = int(self.status.item())
        if code:
            self.status.zero_()
            torch.cuda.synchronize(self.device)  # calls on other streams that follow record anew
            raise _native.TcxError(_native.DATA_LOSS, _STATUS.get(code, f"kv attention status {code}"))

    def _pool(self, pool: torch.Tensor) -> int:
        if not pool.is_cuda or pool.get_device() != self.device.index or not pool.is_contiguous():
            _refuse(f"pool must be a contiguous tensor on {self.device}")
        if pool.nbytes < self._pool_bytes:
            _refuse(f"pool has {pool.nbytes} bytes, its planes need {self._pool_bytes}")
        return pool.data_ptr()


class KvAttention(_OnDevice):
    """Attention of each sequence's newest ``query_tokens`` (1 each by default) over its pages.

    Query i of a sequence of n tokens with m query tokens stands at position n - m + i (behind the
    prefix, where there is one); its own key and value are in the pages already. It sees the tokens
    up to its own position; with ``window`` > 0 only the last ``window`` of them, its own among
    them, and the first ``sinks`` of all. A query that sees nothing gets 0, and -inf for ``lse``.
    ``prefix_pages`` lists the pool slots of a prefix of ``prefix_tokens`` tokens that stands
    before every sequence's own tokens and is read once for all of them.
    """

    def __init__(self, w: KvWorkload, q_heads: int, kv_heads: int, dtype: torch.dtype = torch.bfloat16, *,
                 query_tokens=None, window: int = 0, sinks: int = 0, scale: float | None = None, prefix_pages=None,
                 prefix_tokens: int = 0, device="cuda"):
        if dtype not in _DTYPES:
            _refuse(f"dtype must be torch.bfloat16 or torch.float16, got {dtype}")
        if kv_heads < 1 or q_heads < 1 or q_heads % kv_heads:
            _refuse(f"q_heads ({q_heads}) must be a multiple of kv_heads ({kv_heads})")
        if w.token_bytes not in (kv_heads * 128, kv_heads * 256):
            _refuse(f"token_bytes {w.token_bytes}: {kv_heads} heads of 64 or 128 16-bit values are needed")
        if w.page_tokens < 8 or w.page_tokens % 8:
            _refuse(f"page_tokens must be a multiple of 8, got {w.page_tokens}")
        if w.planes < 2 or w.planes % 2:
            _refuse(f"planes must be layers x {{K, V}}, got {w.planes}")
        if window < 0 or sinks < 0:
            _refuse("window and sinks must not be negative")
        if max(window, sinks) >= 1 << 30:
            _refuse("window and sinks must be below 2^30")
        head_dim = w.token_bytes // (2 * kv_heads)
        scale = head_dim ** -0.5 if scale is None else float(scale)
        if not scale > 0 or not math.isfinite(scale):
            _refuse(f"scale must be > 0 and finite, got {scale}")
        _check_tables(w, "sequences")
        counts = np.ones(w.n_seq, np.int64) if query_tokens is None else np.asarray(query_tokens, np.int64)
        if counts.shape != (w.n_seq,) or (counts < 0).any():
            _refuse(f"query_tokens must be {w.n_seq} counts, none negative")
        if prefix_pages is None and prefix_tokens:
            _refuse("prefix_tokens without prefix_pages")
        pages = np.zeros(0, np.uint32) if prefix_pages is None else _slots(prefix_pages, "prefix")
        if prefix_tokens < 0 or prefix_tokens > pages.size * w.page_tokens:
            _refuse(f"prefix_tokens {prefix_tokens}: the prefix pages hold {pages.size * w.page_tokens}")
        self.w, self.q_heads, self.kv_heads, self.head_dim, self.dtype = w, q_heads, kv_heads, head_dim, dtype
        self.q_offsets = np.concatenate([[0], np.cumsum(counts)])
        self.device = _cuda_device(device)
        offs = np.asarray(w.page_offsets).astype(np.uint64)
        t = self._bind(w, {
            "page_offsets": offs, "page_table": _slots(w.page_table, "sequences"),
            "seq_tokens": np.asarray(w.seq_tokens).astype(np.uint32), "q_offsets": self.q_offsets.astype(np.uint32),
            "prefix_table": pages, "prefix_tokens": np.array([prefix_tokens], np.uint32),
            "status": np.zeros(1, np.uint32)})
        self.page_table, self.seq_tokens = t.page_table, t.seq_tokens
        self.prefix_tokens = None if prefix_pages is None else t.prefix_tokens
        self._args = _native.KvAttentionArgs(
            planes=w.planes, pool_pages=w.pool_pages, page_tokens=w.page_tokens, kv_heads=kv_heads, q_heads=q_heads,
            head_dim=head_dim, dtype=_DTYPES[dtype], d_page_table=t.page_table.data_ptr() if offs[-1] else None,
            d_page_offsets=t.page_offsets.data_ptr(), d_seq_tokens=t.seq_tokens.data_ptr(), n_seq=w.n_seq,
            d_q_offsets=t.q_offsets.data_ptr(), q_tokens=int(self.q_offsets[-1]),
            max_q=int(counts.max(initial=0)), total_pages=int(offs[-1]),
            max_pages=int(np.diff(offs).max(initial=0)),
            d_prefix_table=None if prefix_pages is None else t.buffer.data_ptr() if not pages.size
            else t.prefix_table.data_ptr(), prefix_pages=pages.size, d_prefix_tokens=t.prefix_tokens.data_ptr(),
            window=window, sinks=sinks, scale=scale, d_status=t.status.data_ptr())
        self._shape = (q_heads, head_dim)
        # what new outputs are like (no memory of their own: cheaper to allocate by than by a shape)
        self._out_like = torch.empty(1, dtype=dtype, device=self.device).expand(self._args.q_tokens, *self._shape)
        self._lse_like = torch.empty(1, device=self.device).expand(self._args.q_tokens, q_heads)
        self._scratch_bytes = {}  # with and without weights
        self._workspaces = {}     # scratch and counters, by stream

    @property
    def weight_columns(self) -> int:
        """Columns of ``weights``: token j of sequence s is column page_offsets[s] * page_tokens + j."""
        return int(self.w.page_offsets[-1]) * self.w.page_tokens

    def _rows(self, x: torch.Tensor, what: str):
        """(address, token stride, head stride) of queries or outputs."""
        if x.dtype is not self.dtype or not x.is_cuda or x.get_device() != self.device.index:
            _refuse(f"{what} must be {self.dtype} on {self.device}, got {x.dtype} on {x.device}")
        if x.dim() != 3 or x.shape[0] < self._args.q_tokens or x.shape[1:] != self._shape:
            _refuse(f"{what} must be [>= {self._args.q_tokens} tokens, {self.q_heads}, {self.head_dim}], "
                    f"got {list(x.shape)}")
        tokens, heads, values = x.stride()
        at = x.data_ptr()
        if tokens % 8 or heads % 8:  # the stride of an axis of one entry is never used
            tokens, heads = tokens if x.shape[0] > 1 else 0, heads if self.q_heads > 1 else 0
        if values != 1 or tokens % 8 or heads % 8 or at % 16:
            _refuse(f"{what} must have dense heads, strides that are multiples of 8 and 16-byte alignment")
        return at, tokens, heads

    def _check_apart(self, tokens: int, heads: int) -> None:
        """Rows of an output with these strides must lie apart, whichever axis is the outer one."""
        n, m, dim = self._args.q_tokens, self.q_heads, self.head_dim
        outer = lambda n, tokens, m, heads: ((m < 2 or heads >= dim) and  # noqa: E731
                                             (n < 2 or tokens >= (m - 1) * heads + dim))
        if not outer(n, tokens, m, heads) and not outer(m, heads, n, tokens):
            _refuse(f"out's rows overlap: strides of {tokens} (tokens) and {heads} (heads)")

    def _workspace(self, a, stream: int):
        """Scratch and counters: a stream's calls share them, a captured graph has its own."""
        weighed = a.d_weights is not None
        need = self._scratch_bytes.get(weighed)
        if need is None:
            need = self._scratch_bytes[weighed] = _native.lib().tcx_kv_attention_scratch_bytes(ctypes.byref(a))
        capturing = _capturing()
        found = None if capturing else self._workspaces.get(stream)
        if found is None or found[0].numel() < need:
            found = (torch.empty(need, dtype=torch.uint8, device=self.device),
                     torch.zeros(_native.KV_COUNTERS, dtype=torch.int32, device=self.device))
            if not capturing:
                self._workspaces[stream] = found
        a.d_counters = found[1].data_ptr()
        return found[0].data_ptr(), need

    def run(self, pool: torch.Tensor, layer: int, q: torch.Tensor, *, weights: torch.Tensor | None = None,
            out: torch.Tensor | None = None, lse: torch.Tensor | None = None, stream=None):
        """(out, lse) of the batch's query tokens, in q's order, for one layer of ``pool``.

        ``q`` is [tokens, q_heads, head_dim] (a part of a wider projection's rows, for instance),
        the sequences' query tokens one after the other; rows behind the last sequence's are padding,
        which is not touched in a given ``out`` or ``lse`` and 0 in a new one. ``lse`` is float32
        [tokens, q_heads], the natural logarithm of each row's sum of exponentials. ``weights``,
        float32 [kv_heads, weight_columns], gains each token's softmax weights. ``stream`` is a
        stream or its handle; the current one by default. Calls of one object may run on several
        streams at once, those of one stream from one thread at a time."""
        if stream is not None or self.device.index != torch.cuda.current_device():
            return self._on(stream, lambda: self.run(pool, layer, q, weights=weights, out=out, lse=lse))
        a = _native.KvAttentionArgs.from_buffer_copy(self._args)
        a.d_pool = self._pool(pool)
        if not 0 <= layer < self.w.planes // 2:
            _refuse(f"layer {layer}: the pool has {self.w.planes // 2}")
        a.k_plane, a.v_plane = 2 * layer, 2 * layer + 1
        a.d_q, a.q_token_stride, a.q_head_stride = self._rows(q, "q")
        if q.requires_grad and torch.is_grad_enabled():
            _refuse("KvAttention has no gradient: call it under torch.no_grad()")
        rows = q.shape[0]
        padded = rows > a.q_tokens
        if out is None:
            out = torch.empty_like(self._out_like) if not padded else torch.zeros(
                (rows, *self._shape), dtype=self.dtype, device=self.device)
            a.d_out, a.out_token_stride, a.out_head_stride = out.data_ptr(), *out.stride()[:2]
        else:
            a.d_out, a.out_token_stride, a.out_head_stride = self._rows(out, "out")
            if out.untyped_storage().data_ptr() in (q.untyped_storage().data_ptr(),
                                                    pool.untyped_storage().data_ptr()):
                _refuse("out must not share memory with q or the pool")
            self._check_apart(a.out_token_stride, a.out_head_stride)
        if lse is None:
            lse = torch.empty_like(self._lse_like) if not padded else torch.zeros((rows, self.q_heads),
                                                                                  device=self.device)
        elif (lse.dtype != torch.float32 or lse.device != self.device or not lse.is_contiguous() or lse.dim() != 2
              or lse.shape[0] < a.q_tokens or lse.shape[1] != self.q_heads):
            _refuse(f"lse must be contiguous float32 [>= {a.q_tokens}, {self.q_heads}] on {self.device}")
        a.d_lse = lse.data_ptr()
        if weights is not None:
            if self.prefix_tokens is not None:
                _refuse("weights are not accumulated with a shared prefix")
            columns = self.weight_columns
            if (weights.dtype != torch.float32 or weights.get_device() != self.device.index
                    or weights.shape != (self.kv_heads, columns)
                    or (columns and weights.stride(1) != 1)
                    or (self.kv_heads > 1 and weights.stride(0) < columns)):
                _refuse(f"weights must be float32 [{self.kv_heads}, {columns}] on {self.device}, "
                        "dense in its columns")
            a.d_weights, a.weights_head_stride = weights.data_ptr(), weights.stride(0)
        if a.q_tokens:
            current = self._current()
            scratch, need = self._workspace(a, current)
            rc = _native.lib().tcx_kv_attention(ctypes.byref(a), scratch, need, current)
            if rc:
                _native._raise(rc)
        return out, lse

    def check_status(self) -> None:
        try:
            super().check_status()
        except _native.TcxError:
            self._workspaces.clear()  # a call that gave up leaves its counters as they were
            raise


class KvEvict(_OnDevice):
    """Keeps min(n, budget) tokens of each sequence for every layer and kv head: the first ``sinks``,
    the newest ``recent`` and, of the rest, the heaviest (equal weights by lower index, NaN lowest).

    ``dst`` holds the pages that the kept rows are copied to, in their old order, and the budgets as
    its ``seq_tokens``; its pages must be distinct and none of ``w``'s. A budget must hold ``sinks +
    recent`` tokens, or the whole sequence where that is shorter. Where a sequence outgrows such a
    budget in place (``seq_tokens``), its first ``sinks`` tokens stay and as many of the newest as the
    budget holds behind them. The source pages are only read: other sequences may share them. Rows are copied whole, so the element type does not matter.
    """

    def __init__(self, w: KvWorkload, dst: KvWorkload, kv_heads: int, *, sinks: int = 0, recent: int = 0,
                 device="cuda"):
        if (w.planes, w.pool_pages, w.page_tokens, w.token_bytes) != (dst.planes, dst.pool_pages, dst.page_tokens,
                                                                     dst.token_bytes) or w.n_seq != dst.n_seq:
            _refuse("w and dst must describe the same pool and as many sequences")
        if w.planes < 2 or w.planes % 2:
            _refuse(f"planes must be layers x {{K, V}}, got {w.planes}")
        if kv_heads < 1 or w.token_bytes % (16 * kv_heads):
            _refuse(f"token_bytes {w.token_bytes} must be kv_heads ({kv_heads}) rows of a multiple of 16 bytes")
        if sinks < 0 or recent < 0:
            _refuse("sinks and recent must not be negative")
        _check_tables(w, "sequences")
        _check_tables(dst, "destination")
        # a sequence that its budget holds whole keeps everything
        stays = np.minimum(np.asarray(w.seq_tokens).astype(np.int64), min(sinks + recent, 1 << 32))
        if (np.asarray(dst.seq_tokens).astype(np.int64) < stays).any():
            _refuse(f"a budget is below sinks + recent ({sinks + recent}) and below its sequence")
        table, to = _slots(w.page_table, "sequences"), _slots(dst.page_table, "destination")
        if np.unique(to).size != to.size:
            _refuse("a destination page is listed twice")
        if np.isin(to, table).any():
            _refuse("a destination page is a source page")
        self.w, self.dst, self.kv_heads, self.device = w, dst, kv_heads, _cuda_device(device)
        u32 = lambda x: np.asarray(x).astype(np.uint32)  # noqa: E731
        u64 = lambda x: np.asarray(x).astype(np.uint64)  # noqa: E731
        t = self._bind(w, {
            "page_offsets": u64(w.page_offsets), "dst_page_offsets": u64(dst.page_offsets),
            "page_table": table, "dst_page_table": to, "seq_tokens": u32(w.seq_tokens),
            "budgets": u32(dst.seq_tokens), "status": np.zeros(1, np.uint32)})
        self.page_table, self.seq_tokens = t.page_table, t.seq_tokens
        self._args = _native.KvEvictArgs(
            planes=w.planes, pool_pages=w.pool_pages, page_tokens=w.page_tokens, kv_heads=kv_heads,
            head_bytes=w.token_bytes // kv_heads, d_page_table=t.page_table.data_ptr() or t.buffer.data_ptr(),
            d_page_offsets=t.page_offsets.data_ptr(), d_seq_tokens=t.seq_tokens.data_ptr(),
            d_dst_page_table=t.dst_page_table.data_ptr() or t.buffer.data_ptr(),
            d_dst_page_offsets=t.dst_page_offsets.data_ptr(), d_budgets=t.budgets.data_ptr(), n_seq=w.n_seq,
            dst_total_pages=int(dst.page_offsets[-1]), sinks=min(sinks, 1 << 32), recent=min(recent, 1 << 32),
            d_status=t.status.data_ptr())
        layers = w.planes // 2
        self._weights_shape = (layers, kv_heads, int(w.page_offsets[-1]) * w.page_tokens)
        shape = (layers, kv_heads, int(dst.page_offsets[-1]) * dst.page_tokens)
        one = torch.zeros(1, dtype=torch.int32, device=self.device)
        # what the outputs are like (no memory of their own)
        self._like = one.expand(shape), one.float().expand(shape), one.expand(w.n_seq)

    def run(self, pool: torch.Tensor, weights: torch.Tensor, stream=None):
        """(keep, weights, tokens) after the eviction; the destination pages of ``pool`` are written.

        ``weights`` is float32 [layers, kv_heads, columns], token j of sequence s in column
        page_offsets[s] * page_tokens + j. ``keep`` (int32) and the new weights are [layers, kv_heads,
        dst columns] in the same form for ``dst``: the kept tokens' old indices (-1 behind them) and
        their weights (0 behind them). ``tokens`` (int32) holds every sequence's new length."""
        if stream is not None or self.device.index != torch.cuda.current_device():
            return self._on(stream, lambda: self.run(pool, weights))
        a = _native.KvEvictArgs.from_buffer_copy(self._args)
        a.d_pool = self._pool(pool)
        if (weights.dtype != torch.float32 or weights.get_device() != self.device.index
                or weights.shape != self._weights_shape or (self._weights_shape[2] and weights.stride(2) != 1)):
            _refuse(f"weights must be float32 {list(self._weights_shape)} on {self.device}, dense in its columns")
        a.d_weights = weights.data_ptr() or self._tables.buffer.data_ptr()
        a.weights_layer_stride, a.weights_head_stride = weights.stride()[:2]
        keep, left, tokens = (torch.empty_like(x) for x in self._like)
        a.d_keep, a.d_dst_weights, a.d_dst_tokens = keep.data_ptr(), left.data_ptr(), tokens.data_ptr()
        _native.call("tcx_kv_evict", ctypes.byref(a), self._current())
        return keep, left, tokens
