"""Pages of a cache on the device, over llmk_pages_update, llmk_pages_compact
and llmk_pages_copy (include/llmk_sampler.h).

Reference: llm-scheduler/src/block_allocator.rs keeps the pool of pages and
their reference counts on the host, and the scheduler's step calls it next to
the sampling loop (llm-scheduler/src/scheduler.rs:162-187).  Here the tables,
counts and free pages stay on the GPU beside the token histories, so a step
that samples, verifies and appends on the device needs no round trip for them.
PyTorch only provides device memory and the stream.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from . import _lib
from .sampler import _I32, HipSampler, SamplerError, _flat, _on_device, _output, _ptr, _raw_stream


class PagePools:
    """Tensors that hold the pages of a cache: pool[i][p] is page p of pool i
    (a layer's keys, its values, their scales, ...).  All are contiguous and
    have the same number of pages; a page's size may differ between them."""

    def __init__(self, pools: Sequence[torch.Tensor]):
        if not pools:
            raise SamplerError(_lib.LLMK_ERR_INVALID_ARGUMENT, "no pools")
        self.tensors = list(pools)  # kept alive
        dev, n = pools[0].device, pools[0].shape[0] if pools[0].dim() else 0
        if dev.type != "cuda":
            raise SamplerError(_lib.LLMK_ERR_INVALID_ARGUMENT, "pools must be CUDA (HIP) tensors")
        for t in pools:
            if t.device != dev or not t.is_contiguous() or t.dim() < 1 or t.shape[0] != n \
                    or t.numel() == 0:
                raise SamplerError(_lib.LLMK_ERR_INVALID_ARGUMENT,
                                   "pools must be contiguous tensors of one device and number of pages")
        size = [t.numel() * t.element_size() // n for t in pools]
        self.count, self.num_pages, self.page_bytes = len(pools), n, max(size)
        self.addresses = torch.tensor([[t.data_ptr(), b] for t, b in zip(pools, size)],
                                      dtype=torch.int64, device=dev)


class PageCache:
    """The rows of a paged cache: their tables, lengths, the pages' reference
    counts, and the pools the pages lie in (llmk_page_cache).

    `state` holds counts, bitmap, lengths and table in one int32 tensor, of
    which refs [num_pages], used, lengths [rows] and table [rows, max_pages] are
    views: a copy of it is a snapshot of the cache without the pages' contents.
    A new cache is empty."""

    def __init__(self, sampler: HipSampler, rows: int, max_pages: int, page_tokens: int,
                 num_pages: int, pools: Sequence[torch.Tensor] = ()):
        self.sampler, self._lib = sampler, _lib.load()
        words = ctypes.c_uint64()
        self._check(self._lib.llmk_pages_work_words(rows, num_pages, ctypes.byref(words)))
        dev = torch.device("cuda", sampler.device)
        self.pools = PagePools(pools) if pools else None
        if self.pools is not None:
            if self.pools.num_pages != num_pages:
                raise SamplerError(_lib.LLMK_ERR_INVALID_ARGUMENT,
                                   f"pools of {self.pools.num_pages} pages, num_pages {num_pages}")
            sampler._same_device(self.pools.addresses)
        if max_pages <= 0 or page_tokens <= 0:
            raise SamplerError(_lib.LLMK_ERR_INVALID_ARGUMENT,
                               "max_pages and page_tokens must be > 0")
        self.rows, self.max_pages = rows, max_pages
        self.page_tokens, self.num_pages = page_tokens, num_pages
        sizes = (num_pages, (num_pages + 31) // 32, rows, rows * max_pages)
        self.state = torch.zeros(sum(sizes), dtype=torch.int32, device=dev)
        self.refs, self.used, self.lengths, table = self.state.split(sizes)
        self.table = table.view(rows, max_pages)
        self._work = torch.zeros(words.value, dtype=torch.int32, device=dev)
        a = _lib.PageCacheArgs()
        a.rows, a.max_pages, a.page_tokens, a.num_pages = rows, max_pages, page_tokens, num_pages
        a.table, a.lengths, a.refs = _ptr(self.table), _ptr(self.lengths), _ptr(self.refs)
        a.used, a.work = _ptr(self.used), _ptr(self._work)
        if self.pools is not None:
            a.n_pools, a.page_bytes = self.pools.count, self.pools.page_bytes
            a.pools = _ptr(self.pools.addresses)
        self._args = a

    @staticmethod
    def _check(rc: int) -> None:
        if rc != 0:
            raise SamplerError(rc, _lib.last_error())

    def _stream(self, stream: Optional[torch.cuda.Stream]) -> int:
        return _raw_stream(self.sampler.device, stream)

    def load(self, table: torch.Tensor, lengths: torch.Tensor) -> None:
        """The rows of a cache kept elsewhere (a checkpoint, another process):
        the counts follow from the tables.  Waits for the GPU."""
        if tuple(table.shape) != (self.rows, self.max_pages) or lengths.numel() != self.rows:
            raise SamplerError(_lib.LLMK_ERR_INVALID_ARGUMENT,
                               f"table must be [{self.rows}, {self.max_pages}], lengths [{self.rows}]")
        t, n = table.to(self.state.device).long(), lengths.to(self.state.device).long()
        held = torch.arange(self.max_pages, device=t.device)[None, :] \
            < ((n + self.page_tokens - 1) // self.page_tokens)[:, None]
        pages = t[held]
        if bool((n < 0).any()) or int(n.max()) > self.max_pages * self.page_tokens or \
                (pages.numel() and (int(pages.min()) < 0 or int(pages.max()) >= self.num_pages)):
            raise SamplerError(_lib.LLMK_ERR_INVALID_ARGUMENT, "a length or a page out of range")
        refs = torch.bincount(pages, minlength=self.num_pages)
        bits = torch.zeros(self.used.numel() * 32, dtype=torch.int64, device=t.device)
        bits[:self.num_pages] = (refs > 0).long()
        words = (bits.view(-1, 32) << torch.arange(32, device=t.device)).sum(1)
        self.refs.copy_(refs)
        self.used.copy_(torch.where(words >= 2**31, words - 2**32, words))
        self.lengths.copy_(n)
        self.table.copy_(t)

    def update(self, new_lengths: Optional[torch.Tensor] = None,
               parents: Optional[torch.Tensor] = None,
               stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
        """llmk_pages_update: rows fork from parents[r], shrink, end (length 0)
        and grow to new_lengths[r] (int32 [rows], negative: nothing asked of the
        row).  Returns int32 [rows]: 1, or 0 where a row did not get what it
        asked for (too few pages, or an invalid request)."""
        for name, t in (("new_lengths", new_lengths), ("parents", parents)):
            if t is None:
                continue
            if t.get_device() != self.sampler.device:
                _on_device(self.state.device, **{name: t})
            _flat(name, t, _I32)
            if t.numel() != self.rows:
                raise SamplerError(_lib.LLMK_ERR_INVALID_ARGUMENT, f"{name} needs an entry per row")
        granted = _output(stream, self.rows, dtype=torch.int32, device=self.state.device)
        self._check(self._lib.llmk_pages_update(
            self.sampler._h, ctypes.byref(self._args), _ptr(parents), _ptr(new_lengths),
            granted.data_ptr(), self._stream(stream)))
        return granted

    def compact(self, stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
        """llmk_pages_compact: the pages in use move to the front.  Returns
        int32 [num_pages]: where each page's contents are now."""
        out = _output(stream, self.num_pages, dtype=torch.int32, device=self.state.device)
        self._check(self._lib.llmk_pages_compact(self.sampler._h, ctypes.byref(self._args),
                                                 out.data_ptr(), self._stream(stream)))
        return out

    def copy(self, src: torch.Tensor, dst: torch.Tensor,
             stream: Optional[torch.cuda.Stream] = None) -> None:
        """HipSampler.copy_pages on this cache's pools (contents alone)."""
        if self.pools is None:
            raise SamplerError(_lib.LLMK_ERR_INVALID_ARGUMENT, "the cache has no pools")
        self.sampler.copy_pages(self.pools, src, dst, stream)
