"""Paged key-value cache of a decoder: attention of one new token per sequence, and the cache's pages.

A layer's keys and values live in pages of ``page_size`` tokens, ``[num_pages, kv_heads, page_size, head_dim]``.  Each
sequence is a row of a block table: int32 page indexes, -1 where it has none.  Tables, lengths and the number of rows
that hold each page stay on the device, so a decode step never waits for the host and can be captured in a CUDA
graph.  Pages are taken lowest index first; every result is a function of the state alone.

The functions work on plain tensors; ``PagedKVCache`` keeps them together.  As with the other operators there is no
CPU path: CPU tensors are rejected.  A call that the device has to refuse (too few free pages, a row named twice)
leaves the state as it was and is recorded in the device status word: ``check()``.
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from .ops import _cuda_index, _ptr, _raw_stream

_DTYPES = {torch.bfloat16: _lib.CQ_DT_BF16, torch.float16: _lib.CQ_DT_F16, torch.float8_e4m3fn: _lib.CQ_DT_FP8_E4M3}
_SITES = {101: "free", 102: "fork", 103: "reserve"}


def _i32(t: torch.Tensor, dim: int, name: str) -> torch.Tensor:
    if t.dtype is not torch.int32 or t.dim() != dim or (not t.is_contiguous() and t.numel() and t.stride(-1) != 1):
        raise ValueError(f"{name} must be int32 with {dim} dimension(s), its last one contiguous")
    return t


def _cache_pair(k: torch.Tensor, v: torch.Tensor, dim: int) -> tuple:
    """Checks a pair of caches and gives their strides."""
    if k.dim() != dim or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in _DTYPES:
        raise ValueError("key and value cache must be bf16, f16 or float8_e4m3fn tensors of one shape and type: "
                         f"{dim} dimensions ending in [num_pages, kv_heads, page_size, head_dim]")
    strides = k.stride()
    if strides != v.stride() or strides[-1] != 1:
        raise ValueError("key and value cache must have the same strides, the last one 1")
    return strides


def _head_scale(s: torch.Tensor | None, heads: int, dtype: torch.dtype, name: str):
    if s is None:
        return None
    if dtype != torch.float8_e4m3fn:
        raise ValueError(f"{name} goes with a float8_e4m3fn cache")
    if s.dtype != torch.float32 or s.shape != (heads,) or not s.is_contiguous():
        raise ValueError(f"{name} must be contiguous f32 [{heads}]")
    return s.data_ptr()


@functools.lru_cache(maxsize=1024)
def _attention_workspace(batch: int, q_heads: int, kv_heads: int, head_dim: int, span: int, window: int, sinks: int) -> int:
    return _lib.load().cq_paged_attention_workspace_bytes(batch, q_heads, kv_heads, head_dim, span, window, sinks)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    seq_lens: torch.Tensor, *, rows: torch.Tensor | None = None, scale: float | None = None,
                    window: int = 0, sinks: int = 0, k_scale: torch.Tensor | None = None,
                    v_scale: torch.Tensor | None = None, out: torch.Tensor | None = None, return_lse: bool = False):
    """Attention of one new token per sequence: q [B, q_heads, D] (bf16 or f16, strided rows and heads allowed) over
    the cached tokens of table row ``rows[b]`` (default: row b), seq_lens [table rows] of them, the new one among them.

    caches [num_pages, kv_heads, page_size, D] of q's type or float8_e4m3fn (with ``k_scale`` / ``v_scale`` f32
    [kv_heads]); q_heads a multiple of kv_heads, D 64, 128 or 256.  ``window`` > 0: only the last ``window`` tokens
    and the first ``sinks`` ones are visible.  A row that sees nothing gives zeros (lse -inf).  ``scale`` defaults to
    D ** -0.5.  Returns out [B, q_heads, D], with ``return_lse`` also f32 [B, q_heads]."""
    dt, ct = q.dtype, k_cache.dtype
    if q.dim() != 3 or (dt is not torch.bfloat16 and dt is not torch.float16):
        raise ValueError("q must be bf16 or f16 [B, q_heads, D]")
    b, hq, d = q.shape
    sp, sh, st, _ = _cache_pair(k_cache, v_cache, 4)
    pages, hk, page, dc = k_cache.shape
    if dc != d or d not in (64, 128, 256):
        raise ValueError(f"head_dim must be 64, 128 or 256 in q and the caches, got {d} and {dc}")
    if hk < 1 or hq < 1 or hq % hk:
        raise ValueError(f"q_heads ({hq}) must be a multiple of kv_heads ({hk})")
    if ct is not dt and ct is not torch.float8_e4m3fn:
        raise ValueError(f"the caches must hold {dt} or float8_e4m3fn, got {k_cache.dtype}")
    if window < 0 or sinks < 0:
        raise ValueError("window and sinks must not be negative")
    _i32(block_table, 2, "block_table")
    _i32(seq_lens, 1, "seq_lens")
    table_rows, width = block_table.shape
    if seq_lens.shape[0] != table_rows:
        raise ValueError(f"seq_lens must have one entry per table row ({table_rows})")
    if rows is None:
        if b > table_rows:
            raise ValueError(f"{b} queries for {table_rows} table rows")
    elif _i32(rows, 1, "rows").shape[0] != b:
        raise ValueError(f"rows must have {b} entries")
    idx = _cuda_index(q, k_cache, v_cache, block_table, seq_lens, rows, k_scale, v_scale, out)
    if idx != torch.cuda.current_device():
        with torch.cuda.device(idx):
            return paged_attention(q, k_cache, v_cache, block_table, seq_lens, rows=rows, scale=scale, window=window,
                                   sinks=sinks, k_scale=k_scale, v_scale=v_scale, out=out, return_lse=return_lse)
    ks, vs = _head_scale(k_scale, hk, ct, "k_scale"), _head_scale(v_scale, hk, ct, "v_scale")
    qb, qh, qd = q.stride()
    qp = q.data_ptr()
    if qd != 1 or qb % 8 or qh % 8 or qp % 16:
        q = q.clone(memory_format=torch.contiguous_format)
        qb, qh, qp = hq * d, d, q.data_ptr()
    if out is None:
        out = q.new_empty((b, hq, d))
    elif out.shape != (b, hq, d) or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError(f"out must be contiguous {q.dtype} [{b}, {hq}, {d}]")
    lse = q.new_empty((b, hq), dtype=torch.float32) if return_lse else None
    nbytes = _attention_workspace(b, hq, hk, d, width * page, window, sinks)
    ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes > 0 else None
    status = _lib.load().cq_paged_attention(
        qp, qb, qh, _DTYPES[dt], b, hq, hk, d, k_cache.data_ptr(), v_cache.data_ptr(), _DTYPES[ct], pages, page, sp, sh, st,
        block_table.data_ptr(), table_rows, width, max(block_table.stride(0), width), _ptr(rows), seq_lens.data_ptr(),
        d ** -0.5 if scale is None else scale, window, sinks, ks, vs, out.data_ptr(), _ptr(lse), _ptr(ws), nbytes,
        _raw_stream(idx))
    if status:
        _lib.check("cq_paged_attention", status)
    return (out, lse) if return_lse else out


def append_kv(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              block_table: torch.Tensor, rows: torch.Tensor, positions: torch.Tensor, *,
              k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None) -> None:
    """New keys and values into the cache: token t of k, v [T, kv_heads, D] (bf16 or f16) goes to position
    ``positions[t]`` of table row ``rows[t]`` (int32).  With k, v [layers, T, kv_heads, D] and caches [layers,
    num_pages, kv_heads, page_size, D], every layer in one call.  A token without a place (position -1 of a refused
    reservation, a missing page) is skipped.  A float8_e4m3fn cache receives x / scale of the head, rounded to
    nearest and kept inside the format's finite range."""
    if k.dim() not in (3, 4) or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("k and v must be bf16 or f16 of one shape, [T, kv_heads, D] or [layers, T, kv_heads, D]")
    cs, shape = _cache_pair(k_cache, v_cache, k.dim() + 1), k_cache.shape
    layers, t, hk, d = k.shape if k.dim() == 4 else (1, *k.shape)
    if (k.dim() == 4 and shape[0] != layers) or shape[-3] != hk or shape[-1] != d:
        raise ValueError(f"caches {tuple(shape)} do not fit k {tuple(k.shape)}")
    if k_cache.dtype != k.dtype and k_cache.dtype != torch.float8_e4m3fn:
        raise ValueError(f"the caches must hold {k.dtype} or float8_e4m3fn, got {k_cache.dtype}")
    _i32(block_table, 2, "block_table")
    if _i32(rows, 1, "rows").shape[0] != t or _i32(positions, 1, "positions").shape[0] != t:
        raise ValueError(f"rows and positions must have one entry per token ({t})")
    idx = _cuda_index(k, v, k_cache, v_cache, block_table, rows, positions, k_scale, v_scale)
    if idx != torch.cuda.current_device():
        with torch.cuda.device(idx):
            return append_kv(k, v, k_cache, v_cache, block_table, rows, positions, k_scale=k_scale, v_scale=v_scale)
    ks, vs = _head_scale(k_scale, hk, k_cache.dtype, "k_scale"), _head_scale(v_scale, hk, k_cache.dtype, "v_scale")
    (kp, ksl, kst, ksh), (vp, vsl, vst, vsh) = _new_rows(k, k.dim()), _new_rows(v, k.dim())
    table_rows, width = block_table.shape
    status = _lib.load().cq_kv_append(
        kp.data_ptr(), ksl, kst, ksh, vp.data_ptr(), vsl, vst, vsh, _DTYPES[k.dtype], layers, t, hk, d,
        k_cache.data_ptr(), v_cache.data_ptr(), _DTYPES[k_cache.dtype], shape[-4], shape[-2],
        cs[0] if len(cs) == 5 else 0, cs[-4], cs[-3], cs[-2], block_table.data_ptr(), table_rows, width,
        max(block_table.stride(0), width), rows.data_ptr(), positions.data_ptr(), ks, vs, _raw_stream(idx))
    if status:
        _lib.check("cq_kv_append", status)


def _new_rows(x: torch.Tensor, dim: int):
    """x itself, or a contiguous copy where its rows are not 16-byte aligned, and its layer, token and head strides."""
    s = x.stride()
    if s[-1] != 1 or s[-2] % 8 or s[-3] % 8 or (dim == 4 and s[0] % 8) or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        s = x.stride()
    return x, s[0] if dim == 4 else 0, s[-3], s[-2]


def _state(block_table, seq_lens, ref_counts):
    _i32(block_table, 2, "block_table")
    _i32(seq_lens, 1, "seq_lens")
    _i32(ref_counts, 1, "ref_counts")
    if seq_lens.shape[0] != block_table.shape[0]:
        raise ValueError(f"seq_lens must have one entry per table row ({block_table.shape[0]})")


def _page_layout(k_cache: torch.Tensor, v_cache: torch.Tensor, num_pages: int):
    """(layers, bytes between layers, bytes of a page) of caches [layers, num_pages, kv_heads, page_size, D]."""
    strides = _cache_pair(k_cache, v_cache, 5)
    layers, pages, hk, page, d = k_cache.shape
    if pages != num_pages:
        raise ValueError(f"the caches have {pages} pages, ref_counts {num_pages}")
    if not k_cache.is_contiguous() and strides[1:] != (hk * page * d, page * d, d, 1):
        raise ValueError("a layer of the caches must be contiguous, so that a page is one block")
    size = k_cache.element_size()
    return layers, strides[0] * size, hk * page * d * size


def _update(block_table, seq_lens, ref_counts, page_size, free=None, src=None, dst=None, reserve=None, count=0,
            k_cache=None, v_cache=None):
    _state(block_table, seq_lens, ref_counts)
    for name, t in (("rows", free), ("src", src), ("dst", dst), ("rows", reserve)):
        if t is not None:
            _i32(t, 1, name)
    if src is not None and src.shape != dst.shape:
        raise ValueError("src and dst must have the same number of rows")
    counts = None
    if isinstance(count, torch.Tensor):
        counts, count = _i32(count, 1, "count"), 0
        if counts.shape != reserve.shape:
            raise ValueError("count must have one entry per row")
    elif count < 0:
        raise ValueError("count must not be negative")
    idx = _cuda_index(block_table, seq_lens, ref_counts, free, src, dst, reserve, counts, k_cache, v_cache)
    if idx != torch.cuda.current_device():
        with torch.cuda.device(idx):
            return _update(block_table, seq_lens, ref_counts, page_size, free, src, dst, reserve,
                           count if counts is None else counts, k_cache, v_cache)
    pages = ref_counts.shape[0]
    layers = layer_bytes = page_bytes = n = nbytes = 0
    start = copies = ws = None
    if reserve is not None:
        layers, layer_bytes, page_bytes = _page_layout(k_cache, v_cache, pages)
        n = reserve.shape[0]
        start = seq_lens.new_empty(n)
        copies = seq_lens.new_empty((n, 2))
        nbytes = 4 * (2 * n + pages)
        ws = seq_lens.new_empty(2 * n + pages)
    rows, width = block_table.shape
    status = _lib.load().cq_pages_update(
        block_table.data_ptr(), rows, width, max(block_table.stride(0), width), seq_lens.data_ptr(),
        ref_counts.data_ptr(), pages, page_size, _ptr(free), 0 if free is None else free.shape[0], _ptr(src), _ptr(dst),
        0 if dst is None else dst.shape[0], _ptr(reserve), n, _ptr(counts), count, _ptr(start), _ptr(copies),
        _ptr(k_cache), _ptr(v_cache), layers, layer_bytes, page_bytes, _ptr(ws), nbytes, _raw_stream(idx))
    if status:
        _lib.check("cq_pages_update", status)
    return start, copies


def free_rows(block_table, seq_lens, ref_counts, rows, page_size: int) -> None:
    """The rows (int32, distinct) give up their pages and become empty; a page that no row holds any more is free."""
    _update(block_table, seq_lens, ref_counts, page_size, free=rows)


def fork_rows(block_table, seq_lens, ref_counts, src, dst, page_size: int) -> None:
    """The empty rows ``dst`` become copies of ``src`` (a source may repeat): pages are shared, nothing is moved."""
    _update(block_table, seq_lens, ref_counts, page_size, src=src, dst=dst)


def reserve_tokens(block_table, seq_lens, ref_counts, rows, count, k_cache, v_cache):
    """Room for ``count`` more tokens (an int, or int32 [n]) in each of the rows (int32 [n], distinct).

    A row whose last page is partly filled and shared gets its own copy of it, in all layers of the caches [layers,
    num_pages, kv_heads, page_size, D].  Returns (start, copies): int32 [n], the position of each row's first new
    token, and int32 [n, 2], the (source, destination) pages copied, -1 where none.  All or nothing: with too few
    free pages (or too narrow a table) the state stays as it was, start is -1 and the device status word says so."""
    return _update(block_table, seq_lens, ref_counts, k_cache.shape[3], reserve=rows, count=count, k_cache=k_cache,
                   v_cache=v_cache)


def branch_rows(block_table, seq_lens, ref_counts, src, dst, count, k_cache, v_cache):
    """One resampling step: the rows ``dst`` are freed, become copies of ``src`` and get room for ``count`` new tokens
    - ``free_rows(dst)``, ``fork_rows(src, dst)`` and ``reserve_tokens(dst, count)`` in one call."""
    return _update(block_table, seq_lens, ref_counts, k_cache.shape[3], free=dst, src=src, dst=dst, reserve=dst,
                   count=count, k_cache=k_cache, v_cache=v_cache)


def compact_pages(block_table, ref_counts, k_cache, v_cache, *, out_table: torch.Tensor | None = None,
                  out_refs: torch.Tensor | None = None):
    """All held pages to the lowest indexes, so that the rest of the pool can be given back: with L held pages, those
    at L and above move, in order, to the free pages below L.  Moves the data in every layer of the caches [layers,
    num_pages, kv_heads, page_size, D] and returns (block_table, ref_counts, moves) after it: new tensors, or
    ``out_table`` and ``out_refs`` (which may be the inputs); moves int32 [num_pages // 2, 2] as (from, to), then -1."""
    _i32(block_table, 2, "block_table")
    _i32(ref_counts, 1, "ref_counts")
    idx = _cuda_index(block_table, ref_counts, k_cache, v_cache, out_table, out_refs)
    if idx != torch.cuda.current_device():
        with torch.cuda.device(idx):
            return compact_pages(block_table, ref_counts, k_cache, v_cache, out_table=out_table, out_refs=out_refs)
    pages = ref_counts.shape[0]
    layers, layer_bytes, page_bytes = _page_layout(k_cache, v_cache, pages)
    rows, width = block_table.shape
    if out_table is None:
        out_table = ref_counts.new_empty((rows, width))
    elif _i32(out_table, 2, "out_table").shape != block_table.shape:
        raise ValueError("out_table must have the shape of block_table")
    if out_refs is None:
        out_refs = ref_counts.new_empty(pages)
    elif _i32(out_refs, 1, "out_refs").shape[0] != pages:
        raise ValueError("out_refs must have the shape of ref_counts")
    moves = ref_counts.new_empty((pages // 2, 2))
    ws = ref_counts.new_empty(pages)
    status = _lib.load().cq_pages_compact(
        block_table.data_ptr(), rows, width, max(block_table.stride(0), width), out_table.data_ptr(),
        max(out_table.stride(0), width), ref_counts.data_ptr(), out_refs.data_ptr(), pages, moves.data_ptr(),
        k_cache.data_ptr(), v_cache.data_ptr(), layers, layer_bytes, page_bytes, ws.data_ptr(), 4 * pages,
        _raw_stream(idx))
    if status:
        _lib.check("cq_pages_compact", status)
    return out_table, out_refs, moves


def check() -> None:
    """Raise if the device refused a call since the last check (synchronizes the current stream)."""
    status, site = _lib.take_device_status(torch.cuda.current_stream().cuda_stream)
    if status:
        raise _lib.CQError(f"cache {_SITES.get(site, f'site {site}')}", status, _lib.status_string(status))


class PagedKVCache:
    """Keys and values of ``layers`` layers in one pool of pages, with room for ``rows`` sequences of up to
    ``max_tokens`` tokens.  ``rows`` arguments are int32 device tensors of distinct row numbers."""

    def __init__(self, layers: int, num_pages: int, kv_heads: int, head_dim: int, rows: int, max_tokens: int,
                 page_size: int = 16, dtype: torch.dtype = torch.bfloat16, device="cuda",
                 k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None):
        if dtype not in _DTYPES:
            raise ValueError(f"cache type must be bf16, f16 or float8_e4m3fn, got {dtype}")
        if page_size < 8 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 8 to 1024, got {page_size}")
        self.page_size = page_size
        shape = (layers, num_pages, kv_heads, page_size, head_dim)
        self.k, self.v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        self.block_table = torch.full((rows, -(-max_tokens // page_size)), -1, dtype=torch.int32, device=device)
        self.seq_lens = torch.zeros(rows, dtype=torch.int32, device=device)
        self.ref_counts = torch.zeros(num_pages, dtype=torch.int32, device=device)
        self.k_scale, self.v_scale = k_scale, v_scale

    def _books(self):
        return self.block_table, self.seq_lens, self.ref_counts

    def free(self, rows: torch.Tensor) -> None:
        free_rows(*self._books(), rows, self.page_size)

    def fork(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        fork_rows(*self._books(), src, dst, self.page_size)

    def reserve(self, rows: torch.Tensor, count) -> torch.Tensor:
        """Positions of the rows' first new tokens (-1 where the pool had no room: see ``check``)."""
        return reserve_tokens(*self._books(), rows, count, self.k, self.v)[0]

    def branch(self, src: torch.Tensor, dst: torch.Tensor, count) -> torch.Tensor:
        return branch_rows(*self._books(), src, dst, count, self.k, self.v)[0]

    def compact(self) -> None:
        compact_pages(self.block_table, self.ref_counts, self.k, self.v, out_table=self.block_table,
                      out_refs=self.ref_counts)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, rows: torch.Tensor, positions: torch.Tensor) -> None:
        append_kv(k, v, self.k[layer], self.v[layer], self.block_table, rows, positions, k_scale=self.k_scale,
                  v_scale=self.v_scale)

    def attend(self, layer: int, q: torch.Tensor, rows: torch.Tensor | None = None, **kw) -> torch.Tensor:
        return paged_attention(q, self.k[layer], self.v[layer], self.block_table, self.seq_lens, rows=rows,
                               k_scale=self.k_scale, v_scale=self.v_scale, **kw)

    def check(self) -> None:
        check()
