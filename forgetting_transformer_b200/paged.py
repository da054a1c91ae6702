"""A generation cache in pages, for requests of different lengths, and the attention of a new token over it.

``FgateCache`` (and upstream's ``FgateDynamicCache``, model/forgetting_transformer/fgate_cache.py:4-203) holds one length for a
whole batch.  Here a pool of pages of ``page_size`` tokens serves any number of requests: a page belongs to one request, a
table says which pages hold its tokens, and lengths, tables and the stack of free pages are on the device, where the kernels
read and change them: nothing here waits for the GPU, and a step can be captured in a CUDA graph.

    cache = PagedFgateCache(num_layers, num_pages, 64, num_heads, head_dim, max_requests=32, max_length=65536)
    t = cache.extend(new_tokens, max_tokens)                  # (max_requests,) int32: tokens that each request brings
    for layer in ...:                                         # k, v (max_tokens, heads, head_dim), packed
        cache.update(layer, k, v, log_fgate, t.slots)
        o = cache.attend(layer, q)                            # (max_requests, heads, head_dim): one query per request
    cache.release(finished)                                   # (max_requests,) bool

All of it works in place, so that torch.jit.trace refuses it (a trace would keep the results and drop the writes).
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib

__all__ = ["PageTables", "page_tables", "release_pages", "paged_update", "paged_forgetting_attention", "PagedFgateCache"]

_host = None


def _load_host():
    global _host
    _host = _lib.host()
    return _host


class PageTables(NamedTuple):
    """What ``page_tables`` found out, all int32: per request ``lengths`` (with the new tokens), ``granted`` (new tokens that
    have a place) and ``starts`` (R + 1: first token in the packed batch); ``num_free`` (1,); per token of the packed batch its
    request, position and slot.  A place behind the last token has request -1, position 0 and slot -1."""
    lengths: torch.Tensor
    num_free: torch.Tensor
    starts: torch.Tensor
    granted: torch.Tensor
    requests: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor


def page_tables(lengths: torch.Tensor, new_tokens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                num_free: torch.Tensor, page_size: int, max_tokens: int, *, inplace: bool = False) -> PageTables:
    """Gives every request the pages that ``new_tokens`` (R,) more tokens need, and every token of the packed batch (request 0's
    tokens first) its place.

    - lengths (R,): tokens in the cache so far; block_table (R, pages of the longest request): its entries for the pages given
      out are written, in place; free_pages (pages,): a stack whose first ``num_free`` (1,) entries are free, the last of them
      taken first.  All int32 on one device.
    - Requests are served in their order.  One whose tokens find no room (in its table row, among ``max_tokens``, or pages) is
      granted none and keeps its length; its tokens have slot -1, which ``paged_update`` leaves out.
    - Nobody overtakes: after a request that the free pages were too few for, those behind it get no page in this call either (new
      tokens that fit into their last page are granted), and tokens count towards ``max_tokens`` whether granted or not.  Set
      ``new_tokens`` to 0 for a request that is to wait.
    - ``inplace``: lengths and num_free are changed instead of returned anew.
    - page_size: a power of two from 16 to 65536."""
    return PageTables._make((_host or _load_host()).page_tables(lengths, new_tokens, block_table, free_pages, num_free, page_size,
                                                                max_tokens, inplace))


def release_pages(lengths: torch.Tensor, keep: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                  num_free: torch.Tensor, page_size: int) -> None:
    """Cuts every request to its first ``keep`` (R,) tokens (0: ends it; more than it has: as it is); pages that are not needed
    any more go back on the stack.  Everything in place, as ``page_tables`` takes it.  A page that is in two tables (the attention reads
    such tables) would go back twice: only one of them may have it when its request is cut."""
    (_host or _load_host()).release_pages(lengths, keep, block_table, free_pages, num_free, page_size)


def paged_update(k_pages: torch.Tensor, v_pages: torch.Tensor, gate_pages: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                 log_fgate: torch.Tensor, slots: torch.Tensor, *, gate_is_logit: bool = False) -> None:
    """Writes keys and values (T, Hk, D) and log gates (T, H) of T tokens into their slots.

    k_pages, v_pages (pages, Hk, page_size, D) in fp16 / bf16, rows contiguous and 16-byte aligned; gate_pages (pages, H,
    page_size) fp32, not expanded; slots (T,) int32 / int64.  A slot outside the pool (-1) leaves its token out; of tokens with the
    same slot any one's values may stay, piece by piece, and k, v may not be rows that the call writes.  ``gate_is_logit``: the
    gates are logits (fp16 / bf16 / fp32) and their log sigmoid is written.  No gradients and no tangents."""
    (_host or _load_host()).paged_update(k_pages, v_pages, gate_pages, k, v, log_fgate, slots, gate_is_logit)


def paged_forgetting_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, gate_pages: torch.Tensor,
                               block_table: torch.Tensor, lengths: torch.Tensor, *, sm_scale: Optional[float] = None,
                               return_log_normalizer: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``forgetting_attention`` of one query per request, q (R, H, D), over the first ``lengths`` (R,) tokens of its pages (the
    new token's own among them).

    Pages as for ``paged_update`` (gates 16-byte aligned too); H is a multiple of the pages' heads Hk, and H / Hk query heads
    share a key head, each with gates of its own.  A request of length 0 gets zeros.  Entries of ``block_table`` behind a request's
    length are not looked at; one in front of it that is outside the pool leaves its keys out.  ``return_log_normalizer``: also
    the (R, H) log-sum-exp of the logits (-inf without keys).  No gradients and no
    tangents."""
    return (_host or _load_host()).paged_attention(q, k_pages, v_pages, gate_pages, block_table, lengths, sm_scale,
                                                   return_log_normalizer)


class PagedFgateCache:
    """Pages, tables and lengths of all layers for up to ``max_requests`` requests of up to ``max_length`` tokens.  A request is a
    row of the table; a row of length 0 is free for a new one."""

    def __init__(self, num_layers: int, num_pages: int, page_size: int, num_heads: int, head_dim: int, max_requests: int,
                 max_length: int, *, num_kv_heads: Optional[int] = None, dtype: torch.dtype = torch.bfloat16,
                 device: Union[str, torch.device] = "cuda") -> None:
        if page_size < 16 or page_size > 65536 or page_size & (page_size - 1):
            raise ValueError(f"the page size must be a power of two from 16 to 65536, but got {page_size}")
        if min(num_layers, num_pages, num_heads, max_requests, max_length) < 1:
            raise ValueError("layers, pages, heads, requests and length must be at least 1")
        kv = num_heads if num_kv_heads is None else num_kv_heads
        if kv < 1 or num_heads % kv:
            raise ValueError(f"num_heads ({num_heads}) must be a multiple of num_kv_heads ({kv})")
        self.page_size, self.num_layers = page_size, num_layers
        i32 = dict(dtype=torch.int32, device=device)
        self.k_pages = torch.empty(num_layers, num_pages, kv, page_size, head_dim, dtype=dtype, device=device)
        self.v_pages = torch.empty_like(self.k_pages)
        self.gate_pages = torch.empty(num_layers, num_pages, num_heads, page_size, dtype=torch.float32, device=device)
        self.block_table = torch.full((max_requests, -(-max_length // page_size)), -1, **i32)
        self.lengths = torch.zeros(max_requests, **i32)
        self.free_pages = torch.arange(num_pages - 1, -1, -1, **i32)
        self.num_free = torch.full((1,), num_pages, **i32)

    def __len__(self) -> int:
        return self.num_layers

    def __getitem__(self, layer_idx: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """(k_pages, v_pages, gate_pages) of a layer."""
        return self.k_pages[layer_idx], self.v_pages[layer_idx], self.gate_pages[layer_idx]

    def extend(self, new_tokens: torch.Tensor, max_tokens: int) -> PageTables:
        """Room for ``new_tokens`` (max_requests,) int32 more tokens of every request; ``page_tables``, in place."""
        return page_tables(self.lengths, new_tokens, self.block_table, self.free_pages, self.num_free, self.page_size, max_tokens,
                           inplace=True)

    def update(self, layer_idx: int, k: torch.Tensor, v: torch.Tensor, log_fgate: torch.Tensor, slots: torch.Tensor, *,
               gate_is_logit: bool = False) -> None:
        paged_update(*self[layer_idx], k, v, log_fgate, slots, gate_is_logit=gate_is_logit)

    def attend(self, layer_idx: int, q: torch.Tensor, *, sm_scale: Optional[float] = None) -> torch.Tensor:
        """One query per request, (max_requests, heads, head_dim), against all of its tokens.  Where requests bring different numbers
        of tokens, those of their last ones: ``q[(t.starts[1:].long() - 1).clamp(0, len(q) - 1)]`` (a request that brings none, or is
        granted none, gets another's query there: its row of the result says nothing)."""
        return paged_forgetting_attention(q, *self[layer_idx], self.block_table, self.lengths, sm_scale=sm_scale)

    def crop(self, keep: torch.Tensor) -> None:
        """Cuts every request to its first ``keep`` (max_requests,) int32 tokens."""
        release_pages(self.lengths, keep, self.block_table, self.free_pages, self.num_free, self.page_size)

    def release(self, requests: torch.Tensor) -> None:
        """Ends the requests whose place in ``requests`` (max_requests,) bool is true."""
        self.crop(torch.where(requests, 0, self.lengths))

    def history(self, layer_idx: int, request: int, length: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """The first ``length`` tokens of a request, head-first: k, v (1, Hk, length, D) and log gates (1, H, length); copies, for a
        prompt that comes in several chunks.  ``forgetting_attention`` takes them as they are where Hk = H, else k and v with their
        heads repeated (``repeat_interleave(H // Hk, 1)``).  Tokens behind the request's end are zeros, not what their places last held."""
        P, most = self.k_pages.shape[1], self.block_table.shape[1] * self.page_size
        if not 0 <= length <= most:
            raise ValueError(f"a request holds 0 to {most} tokens, but got a length of {length}")
        n = -(-length // self.page_size)
        entries = self.block_table[request, :n]
        pages = entries.clamp(0, P - 1)
        at = torch.arange(n * self.page_size, device=pages.device).view(n, self.page_size)
        absent = (at >= self.lengths[request]) | (entries != pages)[:, None]

        def rows(pool: torch.Tensor, none: torch.Tensor) -> torch.Tensor:
            return pool[layer_idx][pages].masked_fill_(none, 0).transpose(0, 1).flatten(1, 2)[None, :, :length]
        # (keys and values by 8 bytes, which the masked pass takes in a fourth of the time: 16000 tokens x 24 heads of 64 in 0.16 ms)
        k, v = [rows(t.view(torch.int64), absent[:, None, :, None]).view(t.dtype) for t in (self.k_pages, self.v_pages)]
        return k, v, rows(self.gate_pages, absent[:, None])
