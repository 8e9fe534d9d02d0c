"""Paged key-value cache of a decoder: attention of one new token per sequence, and the cache's pages.

A layer's keys and values live in pages of ``page_size`` tokens, ``[num_pages, kv_heads, page_size, head_dim]``.  Each
sequence is a row of a block table: int32 page indexes, -1 where it has none.  Tables, lengths and the number of rows
that hold each page stay on the device, so a decode step never waits for the host and can be captured in a CUDA
graph.  Pages are taken lowest index first; every result is a function of the state alone.

The functions work on plain tensors; ``PagedKVCache`` keeps them together.  As with the other operators there is no
CPU path: CPU tensors are rejected.  What the device has to refuse is recorded in its status word (``check()``): a
call with a wrong list of rows (out of range, named twice) changes nothing; a reservation without room (too few free
pages, too narrow a table) reserves nothing - ``branch_rows`` has freed and forked its rows by then.
"""
from __future__ import annotations

import torch

from . import _lib

_DTYPES = (torch.bfloat16, torch.float16, torch.float8_e4m3fn)
_SITES = {101: "free", 102: "fork", 103: "reserve"}


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    seq_lens: torch.Tensor, *, rows: torch.Tensor | None = None, scale: float | None = None,
                    window: int = 0, sinks: int = 0, k_scale: torch.Tensor | None = None,
                    v_scale: torch.Tensor | None = None, out: torch.Tensor | None = None, return_lse: bool = False):
    """Attention of one new token per sequence: q [B, q_heads, D] (bf16 or f16, strided rows and heads allowed) over
    the cached tokens of table row ``rows[b]`` (default: row b), seq_lens [table rows] of them, the new one among them.

    caches [num_pages, kv_heads, page_size, D] of q's type or float8_e4m3fn (with ``k_scale`` / ``v_scale`` f32
    [kv_heads]); q_heads a multiple of kv_heads, D 64, 128 or 256.  ``window`` > 0: only the last ``window`` tokens
    and the first ``sinks`` ones are visible.  A row that sees nothing gives zeros (lse -inf).  ``scale`` defaults to
    D ** -0.5.  Returns out [B, q_heads, D], with ``return_lse`` also f32 [B, q_heads].

    Scores, exponentials and sums are fp32.  A softmax weight enters the product with the values as two 16-bit parts: to
    2^-16 of itself with a bf16 cache, to 2^-22 of itself and 2^-40 of the largest with the others.  An infinite value in
    sight makes its element of the output not finite, but NaN also where the definition gives an infinity.  A table
    whose rows share memory (one row expanded to several queries) is copied first."""
    return _lib.decode().paged_attention(q, k_cache, v_cache, block_table, seq_lens, rows, scale, window, sinks, k_scale,
                                         v_scale, out, return_lse)


def append_kv(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              block_table: torch.Tensor, rows: torch.Tensor, positions: torch.Tensor, *,
              k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None) -> None:
    """New keys and values into the cache: token t of k, v [T, kv_heads, D] (bf16 or f16) goes to position
    ``positions[t]`` of table row ``rows[t]`` (int32).  With k, v [layers, T, kv_heads, D] and caches [layers,
    num_pages, kv_heads, page_size, D], every layer in one call.  A token without a place (position -1 of a refused
    reservation, a missing page) is skipped.  A float8_e4m3fn cache receives x / scale of the head, rounded to
    nearest and kept inside the format's finite range."""
    _lib.decode().append_kv(k, v, k_cache, v_cache, block_table, rows, positions, k_scale, v_scale)


def free_rows(block_table, seq_lens, ref_counts, rows, page_size: int) -> None:
    """The rows (int32, distinct) give up their pages and become empty; a page that no row holds any more is free."""
    _lib.decode().pages_update(block_table, seq_lens, ref_counts, page_size, rows, None, None, None, None, 0, None, None)


def fork_rows(block_table, seq_lens, ref_counts, src, dst, page_size: int) -> None:
    """The empty rows ``dst`` become copies of ``src`` (a source may repeat): pages are shared, nothing is moved."""
    _lib.decode().pages_update(block_table, seq_lens, ref_counts, page_size, None, src, dst, None, None, 0, None, None)


def reserve_tokens(block_table, seq_lens, ref_counts, rows, count, k_cache, v_cache):
    """Room for ``count`` more tokens (an int, or int32 [n]) in each of the rows (int32 [n], distinct).

    A row whose last page is partly filled and shared gets its own copy of it, in all layers of the caches [layers,
    num_pages, kv_heads, page_size, D].  Returns (start, copies): int32 [n], the position of each row's first new
    token, and int32 [n, 2], the (source, destination) pages copied, -1 where none.  All or nothing: with too few
    free pages (or too narrow a table) the state stays as it was, start is -1 and the device status word says so."""
    counts, count = (count, 0) if isinstance(count, torch.Tensor) else (None, count)
    return _lib.decode().pages_update(block_table, seq_lens, ref_counts, k_cache.shape[3], None, None, None, rows, counts,
                                      count, k_cache, v_cache)


def branch_rows(block_table, seq_lens, ref_counts, src, dst, count, k_cache, v_cache):
    """One resampling step: the rows ``dst`` are freed, become copies of ``src`` and get room for ``count`` new tokens
    - ``free_rows(dst)``, ``fork_rows(src, dst)`` and ``reserve_tokens(dst, count)`` in one call.  A wrong list (a source
    among the destinations, a row out of range or named twice) changes nothing.  With too few free pages the
    reservation alone is refused: what ``dst`` held is gone, the rows are copies of ``src`` without the new room, and
    ``reserve_tokens(dst, count)`` gives it to them once other rows are freed."""
    counts, count = (count, 0) if isinstance(count, torch.Tensor) else (None, count)
    return _lib.decode().pages_update(block_table, seq_lens, ref_counts, k_cache.shape[3], dst, src, dst, dst, counts, count,
                                      k_cache, v_cache)


def compact_pages(block_table, ref_counts, k_cache, v_cache, *, out_table: torch.Tensor | None = None,
                  out_refs: torch.Tensor | None = None):
    """All held pages to the lowest indexes, so that the rest of the pool can be given back: with L held pages, those
    at L and above move, in order, to the free pages below L.  Moves the data in every layer of the caches [layers,
    num_pages, kv_heads, page_size, D] and returns (block_table, ref_counts, moves) after it: new tensors, or
    ``out_table`` and ``out_refs`` (which may be the inputs); moves int32 [num_pages // 2, 2] as (from, to), then -1."""
    return _lib.decode().compact_pages(block_table, ref_counts, k_cache, v_cache, out_table, out_refs)


def check(device=None) -> None:
    """Raise if the device (default: the current one) refused a call since the last check.  Synchronizes its current
    stream."""
    with torch.cuda.device(device):                      # each device has a status word of its own
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
        check(self.k.device)
