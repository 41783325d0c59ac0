"""Generation with a paged key/value cache: what the reference, which trains and classifies, has no counterpart of.

A cache is two tensors of pages, ``cache_k [n_pages, page_size, H, D]`` and ``cache_v [n_pages, page_size, H, Dv]`` (any strides with
unit inner one and rows on 16-byte boundaries; ``page_size`` a power of two), shared by all sequences; ``page_table [B, pages]``
(int32) says which page holds positions ``i * page_size ..`` of a sequence, ``past [B]`` (int32) how many of its tokens are in the
cache.  Both live on the device and are read there, so a step can be captured into a graph and replayed as they change.  An entry
outside ``[0, n_pages)`` names no page: its tokens are neither stored nor seen.

One step of a layer is ``paged_append`` (K, rotated, and V of the new tokens into their pages and, for a model with a depth stream,
into the token's slot of the depth cache; q rotated) and ``paged_moda`` (the new tokens attend over their sequence and their depth
slots).  When all layers are done, ``past`` grows by the new tokens.  ``PagedKVCache`` keeps the tensors of a model together.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib
from .depth_cache import DepthCache
from .ops import _check_device, _tracing
from .rotary import Rotary


def _refuse_tracing(what: str):
    if _tracing():
        raise RuntimeError(f"{what} reads and writes a cache in place: it cannot be traced")


def paged_append(k, v, cache_k, cache_v, page_table, past, new_lens=None, cu_seqlens=None, q=None, rotary: Optional[Rotary] = None,
                 moda_group_num: int = 1, cached_k=None, cached_v=None, depth_slot: int = 0) -> Optional[torch.Tensor]:
    """New token ``i`` of sequence ``b`` -- rows ``k [B, T, H, D]``, ``v [B, T, H, Dv]`` -- to position ``past[b] + i`` of the cache, in
    place.  ``new_lens [B]`` (int32): how many of the ``T`` tokens of a padded batch are real; or ``cu_seqlens [B + 1]`` (int32, on the
    device): the new tokens are packed, ``k [1, total, H, D]``.  Padded rows and rows behind the last sequence go nowhere, positions
    without a page (past the table's end, or an entry that names none) to no page.

    ``rotary``: ``k`` is rotated by its position on the way, and so is ``q [B, T*moda_group_num, HQ, D]``, which is returned (padded rows
    rotated as well, rows behind the last packed sequence as they are).  ``cached_k, cached_v [B, T*L, H, *]``: ``k, v``, as stored, also
    go to slot ``depth_slot`` of each real token, with or without a page.  No backward pass."""
    _refuse_tracing("paged_append")
    _check_device(cache_k)
    rates, dim, amplitude, interleaved = None, 0, 1.0, False
    if rotary is not None:
        rates, dim, amplitude, interleaved = rotary.rates(cache_k.device), rotary.dim, rotary.amplitude, rotary.interleaved
    return _lib.host().paged_append(k, v, cache_k, cache_v, page_table, past, new_lens, cu_seqlens, q, rates, dim, amplitude, interleaved,
                                    moda_group_num, cached_k, cached_v, depth_slot)


def paged_moda_fwd(q, cache_k, cache_v, page_table, past, new_lens=None, scale=None, cached_k=None, cached_v=None, depth_valid=None,
                   moda_group_num: int = 1) -> Tuple[torch.Tensor, torch.Tensor]:
    """``paged_moda`` with the row sums: ``(o, lse)``, lse fp32 ``[B, T*G, H]`` in base 2 as ``parallel_moda_fwd``'s."""
    _refuse_tracing("attention over a paged cache")
    _check_device(cache_k)
    return _lib.host().paged_attend(q, cache_k, cache_v, page_table, past, new_lens, scale, cached_k, cached_v, depth_valid,
                                    moda_group_num, False)


def paged_moda(q, cache_k, cache_v, page_table, past, new_lens=None, scale=None, cached_k=None, cached_v=None, depth_valid=None,
               moda_group_num: int = 1) -> torch.Tensor:
    """The rows of ``parallel_moda`` (causal) that belong to the ``T`` newest tokens of each sequence: ``q [B, T*G, H, D]``, row ``r`` of
    token ``r // G``; token ``t`` sees positions ``0 .. past[b] + t`` of its pages (its own key and value are there already, see
    ``paged_append``) and the first ``depth_valid`` (none given: all ``L``) slots of its own rows of ``cached_k, cached_v
    [B, T*L, H, *]``.  For few tokens at a time -- one, or drafted ones; a prompt goes through ``parallel_moda``.  ``new_lens [B]``
    (int32): how many of the ``T`` tokens are real.  Rows that see nothing (padded ones, or no page and no slot) are zero, their
    lse -inf.  All of q and the caches share one dtype; fp32 is computed in fp32 whatever ``set_fp32_compute`` says.  No backward."""
    return paged_moda_fwd(q, cache_k, cache_v, page_table, past, new_lens, scale, cached_k, cached_v, depth_valid, moda_group_num)[0]


def paged_attn_fwd(q, cache_k, cache_v, page_table, past, new_lens=None, scale=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``paged_attn`` with the row sums: ``(o, lse)``, lse ``[B, T, HQ]``."""
    _refuse_tracing("attention over a paged cache")
    _check_device(cache_k)
    return _lib.host().paged_attend(q, cache_k, cache_v, page_table, past, new_lens, scale, None, None, None, 1, True)


def paged_attn(q, cache_k, cache_v, page_table, past, new_lens=None, scale=None) -> torch.Tensor:
    """``parallel_attn``'s counterpart: ``q [B, T, HQ, D]`` with ``HQ`` a multiple of the cache's heads (query head ``hq`` reads
    key/value head ``hq // (HQ / H)``), no depth slots; else as ``paged_moda``."""
    return paged_attn_fwd(q, cache_k, cache_v, page_table, past, new_lens, scale)[0]


class PagedKVCache:
    """Pages of all layers of a model (``k, v [layers, n_pages, page_size, H, *]``, not initialised), the table and the counts of
    ``batch`` sequences, and which pages are free.

    ``reserve(b, n)`` gives sequence ``b`` pages for ``n`` tokens in all, ``release(b)`` takes its pages back and empties it; both write
    the table on the device.  ``append`` and ``attend`` are ``paged_append`` and ``paged_moda`` on one layer; ``advance(n)`` counts the step's
    tokens when all layers are done.  ``reserve`` and ``release`` run on the host: between steps, not in a captured one."""

    def __init__(self, layers: int, n_pages: int, page_size: int, H: int, D: int, dtype, device, batch: int = 1,
                 max_tokens: Optional[int] = None, Dv: Optional[int] = None):
        self.page_size, self.n_pages, self.batch = int(page_size), int(n_pages), int(batch)
        if self.page_size <= 0 or self.page_size & (self.page_size - 1):
            raise ValueError(f"the page size must be a power of two, got {page_size}")
        if min(layers, self.n_pages, self.batch, H, D) <= 0:
            raise ValueError("a cache has at least one layer, page, sequence and head")
        max_tokens = self.n_pages * self.page_size if max_tokens is None else int(max_tokens)
        if max_tokens <= 0:
            raise ValueError("max_tokens must be positive")
        width = -(-max_tokens // self.page_size)
        self.k = torch.empty(layers, n_pages, page_size, H, D, dtype=dtype, device=device)
        self.v = torch.empty(layers, n_pages, page_size, H, D if Dv is None else Dv, dtype=dtype, device=device)
        self.page_table = torch.full((batch, width), -1, dtype=torch.int32, device=device)
        self.past = torch.zeros(batch, dtype=torch.int32, device=device)
        self._free: List[int] = list(range(self.n_pages - 1, -1, -1))
        self._pages: List[List[int]] = [[] for _ in range(self.batch)]

    def reserve(self, b: int, tokens: int):
        """Pages for the first ``tokens`` positions of sequence ``b`` (those it has stay where they are).  Reserve before the step that needs
        them: tokens that had no page were not stored, and no longer count once there are pages behind the last one."""
        own, need = self._pages[b], -(-int(tokens) // self.page_size)
        if need > self.page_table.shape[1]:
            raise ValueError(f"{tokens} tokens are more than a sequence may have ({self.page_table.shape[1] * self.page_size})")
        more = need - len(own)
        if more <= 0:
            return
        if more > len(self._free):
            raise RuntimeError(f"the cache is full: {more} pages needed, {len(self._free)} free")
        new = [self._free.pop() for _ in range(more)]
        self.page_table[b, len(own):need] = torch.tensor(new, dtype=torch.int32).to(self.page_table.device)
        self.past[b].clamp_(max=len(own) * self.page_size)  # the new pages hold nothing yet
        own.extend(new)

    def release(self, b: int):
        """Sequence ``b`` is empty; its pages are free."""
        self.page_table[b].fill_(-1)
        self.past[b] = 0
        self._free.extend(reversed(self._pages[b]))
        self._pages[b] = []

    def check_prompts(self, tokens: int, lens: Optional[torch.Tensor] = None):
        """An error unless each sequence that a prompt of ``tokens`` (``lens [batch]``: of at most that many) goes to is empty and has pages
        for it.  Waits for the device."""
        assert lens is None or (lens.shape == self.past.shape and lens.device == self.past.device), "lens must be [batch], on the cache's device"
        new = torch.full_like(self.past, tokens) if lens is None else lens.clamp(0, tokens)
        need = (new + (self.page_size - 1)) // self.page_size
        missing = (self.page_table < 0) | (self.page_table >= self.n_pages)
        at = torch.arange(self.page_table.shape[1], device=self.past.device)
        short = (missing & (at < need[:, None])).any() | (need > at.numel()).any()
        started, short = torch.stack([((self.past > 0) & (new > 0)).any(), short]).tolist()
        if started:
            raise RuntimeError("a prompt is for an empty sequence, and one of these has tokens: release it, or go on with decode")
        if short:
            raise RuntimeError("a prompt's tokens have no pages: reserve them")

    def append(self, layer: int, k, v, new_lens=None, cu_seqlens=None, q=None, rotary: Optional[Rotary] = None, moda_group_num: int = 1,
               depth: Optional[DepthCache] = None):
        """``paged_append`` on a layer's pages; ``depth``: and as the next slot of a depth cache of the same tokens."""
        at = {} if depth is None else {"cached_k": depth.k, "cached_v": depth.v, "depth_slot": depth.n}
        assert depth is None or depth.n < depth.L_max, "depth cache is full"
        out = paged_append(k, v, self.k[layer], self.v[layer], self.page_table, self.past, new_lens, cu_seqlens, q, rotary, moda_group_num,
                           **at)
        if depth is not None:
            depth.n += 1
        return out

    def attend(self, layer: int, q, new_lens=None, scale=None, cached_k=None, cached_v=None, depth_valid=None, moda_group_num: int = 1):
        """``paged_moda`` on a layer's pages."""
        return paged_moda(q, self.k[layer], self.v[layer], self.page_table, self.past, new_lens, scale, cached_k, cached_v, depth_valid,
                          moda_group_num)

    def advance(self, n):
        """The step's tokens count from now on: an int for all sequences, or int32 ``[batch]``, as they are (``new_lens`` that may be out of
        the call's range are bounded by it there: pass ``new_lens.clamp(0, T)``; negative ones take tokens back)."""
        self.past.add_(n)
