"""Copies of pages inside the paged cache."""
from __future__ import annotations

from typing import Iterable, Sequence

import torch

from . import _C, _count


class CacheBlocks:
    """The tensors of a paged cache, as :func:`copy_blocks` addresses them: each [pages, rows, dim] or
    [pages, heads, rows, dim] with the rows of a head one after another, the same number of pages and rows in all."""

    def __init__(self, tensors: Sequence[torch.Tensor]) -> None:
        self.tensors = list(tensors)
        if not self.tensors:
            raise ValueError("CacheBlocks: no tensors")
        first = self.tensors[0]
        self.num_blocks, self.block_size, self.device = first.shape[0], first.shape[-2] if first.dim() > 2 else 0, first.device
        desc, self._max_vecs = [], 0
        for t in self.tensors:
            if t.dim() not in (3, 4) or t.shape[0] != self.num_blocks or t.shape[-2] != self.block_size \
                    or t.device != self.device:
                raise ValueError(f"CacheBlocks: a tensor {tuple(t.shape)} on {t.device} beside {tuple(first.shape)} on "
                                 f"{self.device}")
            size = t.element_size()
            row, heads = t.shape[-1] * size, t.shape[1] if t.dim() == 4 else 1
            head = (t.stride(1) if t.dim() == 4 else t.stride(0)) * size
            if t.stride(-1) != 1 or t.stride(-2) != t.shape[-1] or row % 16 or head % 16 or t.stride(0) * size % 16 \
                    or t.data_ptr() % 16 or t.numel() == 0:
                raise ValueError("CacheBlocks: rows of a head lie one after another and are multiples of 16 bytes, not none")
            span = t.shape[-2] * t.shape[-1]                   # elements of a head, then from the first to the last of several
            outer = () if t.is_contiguous() else range(t.dim() - 2)
            for stride, n in sorted((t.stride(i), t.shape[i]) for i in outer if t.shape[i] > 1):
                if stride < span:
                    raise ValueError("CacheBlocks: pages or heads of a tensor overlap")
                span += (n - 1) * stride
            desc.append([t.data_ptr(), t.stride(0) * size, head, heads | (row // 16) << 32])
            self._max_vecs = max(self._max_vecs, heads * self.block_size * (row // 16))
        self._desc = torch.tensor(desc, dtype=torch.int64, device=self.device) if first.is_cuda else None


def copy_blocks(cache: CacheBlocks, pairs: Iterable[Sequence[int]]) -> None:
    """Copy pages of every tensor of the cache in one launch.  ``pairs``: (source, destination) for whole pages or (source,
    destination, rows) for the first ``rows`` token rows; the destination's other rows keep what they hold.  A destination
    may neither appear twice nor be the source of another pair (ValueError: the result would depend on an order)."""
    flat = []
    for p in pairs:
        flat.extend(p)
        if len(p) == 2:
            flat.append(cache.block_size)
        elif len(p) != 3:
            raise ValueError("copy_blocks: pairs are (source, destination) or (source, destination, rows)")
    if not flat:
        return
    if cache._desc is not None:
        _count(_C().cache_copy(cache._desc, flat, cache.num_blocks, cache.block_size, cache._max_vecs))
        return
    src, dst, rows = flat[0::3], flat[1::3], flat[2::3]
    if min(flat) < 0 or max(src + dst) >= cache.num_blocks or max(rows) > cache.block_size:
        raise ValueError(f"copy_blocks: a page outside 0 .. {cache.num_blocks - 1} or more than {cache.block_size} rows")
    if len(set(dst)) != len(dst) or not set(dst).isdisjoint(src):
        raise ValueError("copy_blocks: a destination is named twice or is a source")
    for s, d, n in zip(src, dst, rows):
        for t in cache.tensors:
            t[d, ..., :n, :] = t[s, ..., :n, :]
