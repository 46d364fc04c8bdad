"""An 8-bit KV cache in pages, the attention that reads it, and the pages' bookkeeping.

``mimir_amd.cache`` keeps keys and values in bf16, a row of positions for each sequence
(src/mimir/model/layers.py:107-115).  Here they are 8-bit floats (e4m3) in pages of 64 tokens
that any row may hold: half the bytes that a decode step reads, prompts shared between
rows, and no memory for positions that are not filled.

* :class:`PagedCache`: the pool.  A page holds 64 tokens of every layer and kv head, keys as
  [token][head_dim], values as [head_dim][token], and one power-of-two scale for its keys and one
  for its values of each layer and head.
* :class:`PageTable`: which pages each row holds, and how many rows hold each page.
* :func:`attention_with_pages`: append the new tokens, then attend (decode and prefill).
* :func:`reserve_pages`, :func:`release_rows`, :func:`fork_rows`, :func:`compact_pages`,
  :func:`copy_pages`.

Every call only enqueues work on the current stream: lengths, tables and free pages stay on
the device, so a decode step with its bookkeeping can be captured in a HIP graph.  Free
pages are handed out lowest first and counts are integers, so results do not depend on timing.
bf16 queries, head_dim 64 or 128; there is no CPU fallback.
"""

from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Optional

import torch
from torch import Tensor

from . import _capi
from . import prefixlm as P

PAGE_TOKENS = _capi.PAGE_TOKENS
_INTS = (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8)


class PagedCache(NamedTuple):
    """A pool of pages: token t's key is ``keys[page, layer, head, t % 64] * 2**key_exponents[page, layer, head]``,
    its value ``values[page, layer, head, :, t % 64] * 2**value_exponents[page, layer, head]``."""
    keys: Tensor              # float8_e4m3fn [pages, layers, heads, 64, head_dim]
    values: Tensor            # float8_e4m3fn [pages, layers, heads, head_dim, 64]
    key_exponents: Tensor     # int8 [pages, layers, heads]
    value_exponents: Tensor   # int8 [pages, layers, heads]

    @classmethod
    def create(cls, num_pages: int, num_layers: int, num_heads: int, head_dim: int, device=None) -> "PagedCache":
        zeros = lambda *tail: torch.zeros((num_pages, num_layers, num_heads, *tail), dtype=torch.uint8,  # noqa: E731
                                          device=device)
        return cls(zeros(PAGE_TOKENS, head_dim).view(torch.float8_e4m3fn), zeros(head_dim, PAGE_TOKENS).view(torch.float8_e4m3fn),
                   zeros().view(torch.int8), zeros().view(torch.int8))


class PageTable(NamedTuple):
    """``pages[row, i]``: the page of the row's tokens [64 i, 64 i + 64), -1 where none; ``lengths[row]``:
    tokens held; ``counts[page]``: table entries that name the page (0: free); ``missing``: pages
    asked for that the pool did not have, added up."""
    pages: Tensor    # int32 [rows, max_pages]
    lengths: Tensor  # int32 [rows]
    counts: Tensor   # int32 [num_pages]
    missing: Tensor  # int32 [1]

    @classmethod
    def create(cls, num_rows: int, max_pages: int, num_pages: int, device=None) -> "PageTable":
        zeros = lambda n: torch.zeros(n, dtype=torch.int32, device=device)  # noqa: E731
        return cls(torch.full((num_rows, max_pages), -1, dtype=torch.int32, device=device), zeros(num_rows), zeros(num_pages), zeros(1))


# ---------------------------------------------------------------- checks

def _check_cache(cache: PagedCache, device=None):
    keys, values, ke, ve = cache
    if keys.dim() != 5 or keys.shape[3] != PAGE_TOKENS:
        raise ValueError(f"keys must be [pages, layers, heads, {PAGE_TOKENS}, head_dim], got shape {tuple(keys.shape)}")
    pages, layers, heads, _, d = keys.shape
    if values.shape != (pages, layers, heads, d, PAGE_TOKENS) or ke.shape != (pages, layers, heads) or ve.shape != ke.shape:
        raise ValueError(f"values and exponents do not fit keys {tuple(keys.shape)}: {tuple(values.shape)}, {tuple(ke.shape)}, "
                         f"{tuple(ve.shape)}")
    if keys.dtype != torch.float8_e4m3fn or values.dtype != keys.dtype:
        raise TypeError(f"a paged cache holds float8_e4m3fn keys and values, got {keys.dtype} and {values.dtype}")
    if ke.dtype != torch.int8 or ve.dtype != torch.int8:
        raise TypeError(f"exponents must be int8, got {ke.dtype} and {ve.dtype}")
    P._check_device_tensor("keys", keys)
    for name, t in zip(PagedCache._fields, cache):
        if t.device != (device or keys.device):
            raise ValueError(f"{name} is on {t.device}, not {device or keys.device}")
        # the layers and heads of a page lie side by side
        if not t[0:1].is_contiguous() or (pages > 1 and t.stride(0) < t[0].numel()):
            raise ValueError(f"the pages of {name} must be contiguous")


def _check_table(table: PageTable):
    P._check_device_tensor("pages", table.pages)
    for name, t, dims in zip(PageTable._fields, table, (2, 1, 1, 1)):
        if t.dtype != torch.int32 or t.dim() != dims or t.device != table.pages.device:
            raise ValueError(f"{name} must be int32 with {dims} dimension(s) on {table.pages.device}, got {tuple(t.shape)} {t.dtype} "
                             f"on {t.device}")
        if (t.stride(-1) != 1 and t.shape[-1] > 1) or (dims == 2 and t.shape[0] > 1 and t.stride(0) < t.shape[1]):
            raise ValueError(f"{name} must be laid out row by row")
    if table.lengths.shape[0] != table.pages.shape[0] or table.missing.shape[0] != 1:
        raise ValueError(f"table of {table.pages.shape[0]} rows with {table.lengths.shape[0]} lengths and {table.missing.shape[0]} counters")


def _row_list(name: str, t: Tensor, device) -> Tensor:
    if t.dim() != 1 or t.dtype not in _INTS:
        raise ValueError(f"{name} must be a vector of whole numbers, got {tuple(t.shape)} {t.dtype}")
    if t.dtype == torch.int64:  # what 32 bits do not hold stays outside, rather than wrap to a row or page
        t = t.clamp(-(1 << 31), (1 << 31) - 1)
    return t.to(device=device, dtype=torch.int32).contiguous()


def _params(table: Optional[PageTable], cache: Optional[PagedCache] = None) -> _capi.PagesParams:
    p = _capi.PagesParams()
    if table is not None:
        _check_table(table)
        p.pages, p.lengths, p.counts, p.missing = (t.data_ptr() for t in table)
        p.pages_stride = max(table.pages.stride(0), table.pages.shape[1])
        p.rows, p.width, p.num_pages = *table.pages.shape, table.counts.shape[0]
    if cache is not None:
        _check_cache(cache, None if table is None else table.pages.device)
        if table is not None and cache.keys.shape[0] != table.counts.shape[0]:
            raise ValueError(f"a cache of {cache.keys.shape[0]} pages for a table of {table.counts.shape[0]}")
        p.num_pages = cache.keys.shape[0]
        for i, t in enumerate(cache):
            p.data[i] = t.data_ptr()
            p.data_bytes[i] = math.prod(t.shape[1:])
            p.data_stride[i] = t.stride(0)
    return p


def _workspace(p: _capi.PagesParams, items: int, device) -> Tensor:
    nbytes = int(_capi.load().mimir_prefixlm_pages_workspace_bytes(ctypes.byref(p), items))
    ws = torch.empty(nbytes // 4, dtype=torch.int32, device=device)
    p.workspace, p.workspace_bytes = ws.data_ptr(), nbytes
    return ws


def _served(call: str, table: PageTable, cache: Optional[PagedCache], first=None, second=None):
    """The call's result from the native host calls, None if it takes the general path."""
    if not table.pages.is_cuda:
        return None
    return _capi.host().pages(call, table, cache, first, second, P._stream(table.pages.device))


def _call(entry: str, device, p, *args) -> None:
    lib = _capi.load()
    with torch.cuda.device(device):
        _capi.raise_for_status(lib, getattr(lib, entry)(ctypes.byref(p), *args, P._stream(device)))


# ---------------------------------------------------------------- pages of rows

def copy_pages(cache: PagedCache, source: Tensor, destination: Tensor) -> None:
    """Page ``destination[i]`` becomes a copy of page ``source[i]``, all layers.  Numbers outside the pool
    are skipped; a destination must not come twice nor be a source (``ValueError`` with
    ``mimir_amd.set_validate_metadata(True)``, else such a page holds either's data)."""
    p = _params(None, cache)
    device = cache.keys.device
    src, dst = _row_list("source", source, device), _row_list("destination", destination, device)
    if src.shape != dst.shape:
        raise ValueError(f"{src.shape[0]} sources for {dst.shape[0]} destinations")
    if P._validate_metadata and len(src) > 0:
        inside = (src >= 0) & (src < p.num_pages) & (dst >= 0) & (dst < p.num_pages)
        named = torch.cat((src[inside].unique(), dst[inside]))
        if len(named.unique()) != len(named):
            raise ValueError("a destination page is named twice or is a source")
    _call("mimir_prefixlm_pages_copy", device, p, src.data_ptr(), dst.data_ptr(), len(src))


def fork_rows(cache: PagedCache, table: PageTable, source: Tensor, destination: Tensor) -> None:
    """Row ``destination[i]`` goes on from the tokens that row ``source[i]`` held before the call (beams,
    samples, a shared prompt): it gives back its own pages, shares the source's full ones and gets a
    copy of the last, partly filled one, which it can then append to.

    All entries at once, so a permutation of beams is one call.  A last page that all rows holding
    it give back in the call (they are replaced themselves) is left to the first row that goes on from
    it, uncopied.  Entries with equal source
    and destination leave the row as it is, entries outside the table are skipped, of several
    for one destination the last counts.  Pages reserved past the source's tokens are not
    forked.  Where no page is free the destination's last page stays -1 and ``table.missing``
    counts it."""
    if _served("fork", table, cache, source, destination) is not None:
        return
    p = _params(table, cache)
    device = table.pages.device
    src, dst = _row_list("source", source, device), _row_list("destination", destination, device)
    if src.shape != dst.shape:
        raise ValueError(f"{src.shape[0]} sources for {dst.shape[0]} destinations")
    ws = _workspace(p, len(src), device)  # noqa: F841 (held until the launch)
    _call("mimir_prefixlm_pages_fork", device, p, src.data_ptr(), dst.data_ptr(), len(src))


def compact_pages(cache: PagedCache, table: PageTable) -> Tensor:
    """Move the pages in use to the front of the pool, all layers, and rename them in the table.
    Returns their number (int32 [1], on the device): the pool can be cut there."""
    used = _served("compact", table, cache)
    if used is not None:
        return used
    p = _params(table, cache)
    device = table.pages.device
    used = torch.empty(1, dtype=torch.int32, device=device)
    ws = _workspace(p, 0, device)  # noqa: F841
    _call("mimir_prefixlm_pages_compact", device, p, used.data_ptr())
    return used


def release_rows(table: PageTable, rows: Tensor) -> None:
    """The listed rows give back their pages and hold no tokens (numbers outside the table are skipped,
    one may come twice)."""
    if _served("release", table, None, rows) is not None:
        return
    p = _params(table)
    device = table.pages.device
    rows = _row_list("rows", rows, device)
    _call("mimir_prefixlm_pages_release", device, p, rows.data_ptr(), len(rows))


def reserve_pages(table: PageTable, new_lengths: Tensor) -> None:
    """Give every row the pages that it lacks for ``lengths + new_lengths`` tokens (none where
    ``new_lengths`` is 0), by row, then place, the lowest free page first.  The lengths stay: add the new ones
    when they have been appended.  Pages the pool does not have are counted in ``table.missing``."""
    if _served("reserve", table, None, new_lengths) is not None:
        return
    p = _params(table)
    device = table.pages.device
    new = _row_list("new_lengths", new_lengths, device)
    if new.shape[0] != table.pages.shape[0]:
        raise ValueError(f"new_lengths must be [{table.pages.shape[0]}], got {tuple(new.shape)}")
    ws = _workspace(p, 0, device)  # noqa: F841
    _call("mimir_prefixlm_pages_reserve", device, p, new.data_ptr())


# ---------------------------------------------------------------- attention

def _strides(t: Tensor):
    """Of batch, tokens and heads; a dim of one entry has none to speak of."""
    return tuple(s if n > 1 else 0 for n, s in zip(t.shape[:3], t.stride()))


def _rows4(t: Tensor) -> Tensor:
    return P._own_copy(t) if t.stride(-1) != 1 or any(s % 8 for s in _strides(t)) or t.data_ptr() % 16 else t


def _validate(cache, table, lens, rows, new, S: int) -> None:
    """One host read for all checks of a call's indices."""
    if table.shape[0] == 0:
        raise IndexError("a page table without rows")
    n = lens.long()
    m = torch.full_like(n, S) if new is None else new.long()
    r = torch.arange(len(n), device=n.device) if rows is None else rows.long()
    inside = (r >= 0) & (r < table.shape[0])
    at = torch.arange(table.shape[1], device=n.device)
    held = table[r.clamp(0, table.shape[0] - 1)].long()
    end = n + m.clamp(min=0)
    read = (at * PAGE_TOKENS < end[:, None]) & inside[:, None] & (m > 0)[:, None]
    written = read & ((at + 1) * PAGE_TOKENS > n[:, None])
    bad = read & ((held < 0) | (held >= cache.keys.shape[0]))
    w = held[written & ~bad]
    readers = torch.bincount(held[read & ~bad], minlength=1)  # of each page, in this call
    found = torch.stack([(n < 0).any(), ((m < 0) | (m > S)).any(), (~inside).any(), (end > table.shape[1] * PAGE_TOKENS).any(), bad.any(),
                         (readers[w] > 1).any()]).tolist()
    if found[0]:
        raise ValueError("cache_lengths must be non-negative")
    if found[1]:
        raise ValueError(f"new_lengths must lie in [0, {S}]")
    if found[2]:
        raise IndexError(f"cache_batch_indices must lie in [0, {table.shape[0]})")
    if found[3]:
        raise IndexError(f"tokens past a page table of {table.shape[1]} pages")
    if found[4]:
        raise IndexError("a row has no page for tokens that the call reads or writes")
    if found[5]:
        raise ValueError("a page that a batch row appends to is held twice in the call")


def attention_with_pages(query: Tensor, key: Tensor, value: Tensor, cache: PagedCache, layer: int, page_table: Tensor,
                         cache_lengths: Tensor, causal: bool, cache_batch_indices: Optional[Tensor] = None, *,
                         new_lengths: Optional[Tensor] = None, softmax_scale: Optional[float] = None) -> Tensor:
    """``attention_with_cache`` over one layer of a paged 8-bit cache: bf16 query [B, S, Hq, D] and
    key / value [B, S, Hkv, D]; returns [B, S, Hq, D].

    Token i of batch row b is appended at ``cache_lengths[b] + i`` of table row
    ``cache_batch_indices[b]`` (default b), in 8 bits: a page takes the smallest power-of-two scale
    that its largest magnitude fits under (448 times it), and tokens that it holds already are rounded
    again where the scale grows.  Then each query attends the tokens before ``cache_lengths[b] + S``
    (``<= cache_lengths[b] + i`` when causal) as the cache holds them, the call's own among them.

    ``new_lengths`` [B]: of a padded batch, the tokens that count; the others are not appended and
    their outputs are zeros.  A row of 0 is left alone.  ``page_table`` is int32 [rows, max_pages]
    (``PageTable.pages``); the pages must be there (:func:`reserve_pages`): tokens without one are
    dropped, and not attended.  A page that a batch row appends to must be that row's alone in the
    call, neither appended to nor read for another (fork_rows sees to that): the rows run side by
    side.  Both raise with ``mimir_amd.set_validate_metadata(True)``, which costs a host read.
    Infinite keys and values become NaN.  Scores and sums are fp32; probabilities are rounded to bf16 for
    the product with the values, and with more than 32 query rows per kv head the queries are read to 2^-22 of
    the largest of 32 columns.  For inference: the result has no gradient.
    """
    scale = (1.0 / math.sqrt(query.shape[-1]) if query.shape[-1] else 1.0) if softmax_scale is None else float(softmax_scale)
    if query.is_cuda and not P._validate_metadata:
        out = _capi.host().paged_attn(query, key, value, cache, layer, page_table, cache_lengths, causal, cache_batch_indices,
                                      new_lengths, scale, P._stream(query.device))
        if out is not None:
            return out
    if query.dtype != torch.bfloat16:
        raise TypeError(f"paged attention supports bfloat16 tensors only, got {query.dtype}")
    for name, t in (("query", query), ("key", key), ("value", value)):
        if t.dim() != 4:
            raise ValueError(f"{name} must be [batch, tokens, heads, head_dim], got shape {tuple(t.shape)}")
        P._check_device_tensor(name, t)
        if t.dtype != query.dtype or t.device != query.device:
            raise ValueError(f"{name} is {t.dtype} on {t.device}, the query {query.dtype} on {query.device}")
    B, S, hq, d = query.shape
    hkv = key.shape[2]
    if key.shape != (B, S, hkv, d) or value.shape != key.shape:
        raise ValueError(f"incompatible query / key / value shapes {tuple(query.shape)}, {tuple(key.shape)}, {tuple(value.shape)}")
    if hkv == 0 or hq % hkv:
        raise ValueError(f"Query heads {hq} must be divisible by key/value heads {hkv}.")
    device = query.device
    _check_cache(cache, device)
    pages, layers = cache.keys.shape[:2]
    if cache.keys.shape[2] != hkv or cache.keys.shape[4] != d:
        raise ValueError(f"cache must be [pages, layers, {hkv}, {PAGE_TOKENS}, {d}], got {tuple(cache.keys.shape)}")
    if not 0 <= layer < layers:
        raise IndexError(f"layer {layer} of a cache of {layers}")
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.device != device or \
            (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError(f"page_table must be int32 [rows, max_pages] on {device}, laid out row by row, got {tuple(page_table.shape)} "
                         f"{page_table.dtype} on {page_table.device}")
    # one type for all three, wide enough for each: a row number past 32 bits must not wrap to a row of the table
    index_dtype = torch.int64 if any(t is not None and t.dtype == torch.int64
                                     for t in (cache_lengths, cache_batch_indices, new_lengths)) else torch.int32

    def index(name, t):
        if t is None:
            return None
        if t.shape != (B,) or t.dtype not in _INTS:
            raise ValueError(f"{name} must be [{B}] whole numbers, got {tuple(t.shape)} {t.dtype}")
        return t.to(device=device, dtype=index_dtype).contiguous()

    lens, rows, new = (index(n, t) for n, t in (("cache_lengths", cache_lengths), ("cache_batch_indices", cache_batch_indices),
                                                ("new_lengths", new_lengths)))
    if P._validate_metadata and B > 0 and S > 0:
        _validate(cache, page_table, lens, rows, new, S)
    q, k, v = _rows4(query), _rows4(key), _rows4(value)
    out = torch.empty((B, S, hq, d), dtype=q.dtype, device=device)
    ck, cv, ke, ve = (t[:, layer] for t in cache)
    p = _capi.PagedAttnParams(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), ck.data_ptr(), cv.data_ptr(), ke.data_ptr(), ve.data_ptr(),
        page_table.data_ptr(), lens.data_ptr(), None if rows is None else rows.data_ptr(), None if new is None else new.data_ptr(),
        *_strides(q), *_strides(k), *_strides(v), *out.stride()[:3],
        ck.stride(0), cv.stride(0), ke.stride(0), ve.stride(0), page_table.stride(0),
        B, S, pages, *page_table.shape, hq, hkv, d, int(bool(causal)), _capi.DTYPE_BFLOAT16, int(index_dtype == torch.int64),
        scale, None, 0)
    lib = _capi.load()
    ws_bytes = int(lib.mimir_prefixlm_paged_attn_workspace_bytes(ctypes.byref(p)))
    ws = torch.empty(max(ws_bytes // 4, 4), dtype=torch.float32, device=device)
    p.workspace, p.workspace_bytes = ws.data_ptr(), ws_bytes
    _call("mimir_prefixlm_paged_attn", device, p)
    return out
