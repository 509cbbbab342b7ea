"""A paged K/V cache for batches of requests whose drafts are token trees.

The cache owns one page pool per layer, the block tables and the free list,
all on the device; nothing here reads a length back to the host, so a step
can be captured in a CUDA graph.  One step of tree decoding:

>>> rows = cache.extend(counts, max_tokens)          # room behind each context
>>> for layer in range(n_layers):
...     cache.write(layer, k, v, rows)
...     out, lse = cache.attend(layer, q, rows, tree_mask)
>>> cache.accept(path, path_lens)                    # keep one path of each tree

A prompt is a step whose rows are all kept: ``extend``, ``write``, the
prompt's own attention, then ``accept(None, counts)``.  No counterpart in the
reference (its caches hold one tensor per layer and one token a step).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from halo_b200 import _lib as L
from halo_b200 import ops


class PagedRows(NamedTuple):
    """Rows of one step, in the places of the counts they were asked by:
    request ``r``'s begin at ``counts[:r].sum()``, whether or not the requests
    before it were granted theirs.  ``cu`` counts those granted:
    ``cu[r + 1] - cu[r]`` is 0 for a request whose rows the pool cannot hold,
    whose places hold -1 and are neither written nor attended."""
    slots: torch.Tensor        # int64 (max_tokens,), -1 for a row that is not there
    positions: torch.Tensor    # int64 (max_tokens,), -1 for a row that is not there
    cu: torch.Tensor           # int32 (max_requests + 1,)


class PagedKVCache:
    """``n_pages`` pages of ``page_size`` rows a layer, shared by up to
    ``max_requests`` (8192) requests of up to ``max_len`` rows.  Rows of any
    ``head_dim``, page size and floating type can be written, moved and given
    back; ``attend`` takes bf16 and fp16, a ``head_dim`` of 64 or 128 and a
    page size that is a multiple of 8."""

    def __init__(self, n_layers: int, n_pages: int, n_kv_heads: int, head_dim: int, *,
                 max_requests: int, max_len: int, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if min(n_layers, n_pages, n_kv_heads, head_dim, max_requests, max_len, page_size) < 1:
            raise L.HaloError("cache dimensions must be positive", L.HALO_ERR_INVALID_ARG)
        blocks = -(-max_len // page_size)
        # what no step could be begun in is refused before the pools are allocated
        if max_requests > 8192 or n_pages > 2 ** 30 or max_requests * blocks >= 2 ** 31 or \
                (blocks + 1) * page_size >= 2 ** 31:
            raise L.HaloError(f"{max_requests} requests of {max_len} rows on {n_pages} pages of "
                              f"{page_size} are too many", L.HALO_ERR_UNSUPPORTED)
        L.halo_dtype(dtype)
        self.page_size = page_size
        shape = (n_pages, n_kv_heads, page_size, head_dim)
        self.k = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(n_layers)]
        self.v = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(n_layers)]
        dev = self.k[0].device
        self.block_tables = torch.zeros(max_requests, blocks, dtype=torch.int32, device=dev)
        self.free_pages = torch.arange(n_pages, dtype=torch.int32, device=dev)
        self.n_free = torch.full((1,), n_pages, dtype=torch.int32, device=dev)
        # rows of each request's context, of the step under way (and where they
        # begin in it), and rows whose pages the request holds
        self.lens = torch.zeros(max_requests, dtype=torch.int32, device=dev)
        self.step = torch.zeros(max_requests, dtype=torch.int32, device=dev)
        self.starts = torch.zeros(max_requests, dtype=torch.int32, device=dev)
        self.held = torch.zeros(max_requests, dtype=torch.int32, device=dev)

    def extend(self, counts: torch.Tensor, max_tokens: int) -> PagedRows:
        """Begin a step: room for ``counts[r]`` (int32, at most ``max_tokens`` in
        all; a single count is every request's) rows behind each request's
        context.  A step that was begun before and not accepted is given up:
        its rows are room again."""
        if counts.numel() == 1:
            counts = counts.expand(self.lens.shape)
        return PagedRows(*ops.extend_block_tables(
            self.block_tables, self.held, self.lens, counts.contiguous(), self.step, self.starts,
            self.free_pages, self.n_free, page_size=self.page_size, max_tokens=max_tokens))

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, rows: PagedRows) -> None:
        """Store the step's K/V rows ``(max_tokens, H_kv, D)``."""
        ops.write_kv_pages(k, v, self.k[layer], self.v[layer], rows.slots)

    def attend(self, layer: int, q: torch.Tensor, rows: PagedRows, tree_mask: torch.Tensor,
               **kwargs):
        """``ops.tree_attention`` of the step's rows over ``layer``; rows of a
        request that was refused are not written."""
        return ops.tree_attention(q, self.k[layer], self.v[layer], self.block_tables, self.lens,
                                  rows.cu, tree_mask, node_starts=self.starts, **kwargs)

    def accept(self, path: Optional[torch.Tensor], path_lens: torch.Tensor) -> None:
        """End the step: request ``r`` keeps the rows ``path[r, :path_lens[r]]``
        of its step (``None``: its first ``path_lens[r]`` rows; never more than
        the step gave it) and gives the other pages back.  A node that is not
        of the step moves nothing: row ``i`` of the step stays in its place."""
        # neither a path's steps nor its nodes may reach behind the rows of the
        # step: table entries there name pages that another request may own by now
        keep = torch.minimum(path_lens.clamp(0, None if path is None else path.shape[1]), self.step)
        if path is not None:
            path = path.masked_fill(path >= self.step[:, None], 0)
            for k, v in zip(self.k, self.v):
                ops.commit_tree_path(k, v, self.block_tables, self.lens, path, keep)
        self.lens.copy_(self._resize(self.lens + keep))
        self.step.zero_()

    def release(self, ended: torch.Tensor) -> None:
        """Empty the requests where ``ended (max_requests,)`` is true; others
        keep their rows, those of a step under way too (an ended request's
        rows of that step are nobody's: they may not be written any more)."""
        self._resize(self.held.masked_fill(ended, 0))
        self.lens.masked_fill_(ended, 0)
        self.step.masked_fill_(ended, 0)

    def _resize(self, lens: torch.Tensor) -> torch.Tensor:
        _, _, _, held = ops.update_block_tables(
            self.block_tables, self.held, lens, self.free_pages, self.n_free,
            page_size=self.page_size, max_tokens=0)
        return self.held.copy_(held)
