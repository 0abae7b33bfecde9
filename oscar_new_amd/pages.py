"""Pages of a model's caches: free pages, forked requests, compaction (``csrc/pages.hip``).

No reference counterpart: the reference refuses page copies (backend.py:30-38), because the first
page of a request holds its BF16 window and so has one owner. Its other pages hold INT2 records that
nothing writes again once a page is full, so requests that continue the same tokens may map them
together. A fork does that: it copies the first page and an unfinished last one and shares the rest.
``kernels.shared_history`` then computes the attention over the shared positions once for all of
them.

Everything stays on the device: no call reads back, synchronizes or allocates anything but its
outputs, so calls can be captured in a graph. Page numbers are physical pages (a block table's entry
divided by the kernel blocks of a page). All calls take the block table and the token counts of the
scheduler's rows: row r holds ``seq_lens[r]`` tokens in the blocks of ``block_tables[r]``, and the
rows below ``counts[0]`` are live. Those tokens are the ones that stay: a fork of a request whose
draft tokens are not yet accepted takes its count without them, since records of a shared page are
not written again. A page that a row maps past its tokens counts as free: ``free_pages`` and
``compact_pages`` take, for a row whose next tokens already have pages, the count with those tokens.
"""

from __future__ import annotations

import torch

from . import _ext
from .kernels import _device_check, _int32, _launch, _same_device, layout_struct

__all__ = ["PageCaches", "free_pages", "fork_requests", "compact_pages"]


class PageCaches:
    """The caches of a model's layers, for page copies in all of them with one launch.

    ``kv_caches``: one native ``(K, V)`` cache view pair per layer (``CacheLayout.tensor_views``),
    all of the same page count on one device. Keeps the views and a device table of their
    addresses.
    """

    def __init__(self, kv_caches, layout):
        views = [layout.tensor_views(pair) for pair in kv_caches]
        if not views:
            raise ValueError("PageCaches needs at least one layer's cache")
        history, window = views[0]
        _device_check(*(t for pair in views for t in pair))
        for pair in views:
            if any(t.device != history.device for t in pair):
                raise ValueError("all layers' caches must be on one device")
            if pair[0].numel() != history.numel():
                raise ValueError("all layers' caches must have the same number of pages")
            if any(t.data_ptr() % 16 for t in pair):
                raise ValueError("cache stripes must be 16-byte aligned")
        self.layout = layout
        self.layout_struct = layout_struct(layout)
        self.views = views
        self.device = history.device
        self.num_pages = history.numel() // layout.stripe_page_bytes
        if not self.num_pages:
            raise ValueError("the caches hold no pages")
        self.stripes = torch.tensor([[t.data_ptr() for t in pair] for pair in views],
                                    dtype=torch.int64, device=self.device)


def _table(caches, block_tables, seq_lens, counts=None, **others):
    """Checks of the scheduler's tensors; the arguments of the block table."""
    _same_device(caches.stripes, block_tables=block_tables, seq_lens=seq_lens, counts=counts,
                 **others)
    if block_tables.dim() != 2 or 0 in block_tables.shape:
        raise ValueError("block_tables must be [rows, columns]")
    if _int32(block_tables, "block_tables").stride(1) != 1 and block_tables.shape[1] > 1:
        raise ValueError("block table rows must be contiguous")
    rows, columns = block_tables.shape
    stride = block_tables.stride(0) if rows > 1 else max(block_tables.stride(0), columns)
    if stride < columns:
        raise ValueError("block table rows must not overlap")
    if _int32(seq_lens, "seq_lens").dim() != 1 or not seq_lens.is_contiguous():
        raise ValueError("seq_lens must be a contiguous vector")
    if seq_lens.shape[0] < rows:
        raise ValueError("seq_lens must hold one count per block table row")
    if counts is not None and (_int32(counts, "counts").numel() < 1 or not counts.is_contiguous()):
        raise ValueError("counts must hold the number of live rows first")
    return block_tables.data_ptr(), stride, columns, rows


def free_pages(caches, block_tables, seq_lens, counts):
    """Pages that no token of a live row is mapped to: ``(pages, count)``, int32 ``[num_pages]`` with
    the free pages in ascending order and -1 behind them, and int32 ``[1]``."""
    table = _table(caches, block_tables, seq_lens, counts)
    n = caches.num_pages
    pages, count, used = seq_lens.new_empty(2 * n + 1).split((n, 1, n))
    _launch(
        _ext.library().oscar_free_pages, "free_pages", caches.device, caches.num_pages, *table,
        seq_lens.data_ptr(), counts.data_ptr(), caches.layout_struct, used.data_ptr(),
        pages.data_ptr(), count.data_ptr(),
    )
    return pages, count


def fork_requests(caches, block_tables, seq_lens, parents, children, fresh):
    """Rows ``children[i]`` become requests that continue the tokens of rows ``parents[i]``.

    ``parents``, ``children``: int32 ``[forks]`` rows of ``block_tables``, which is changed in place,
    as is ``seq_lens``; ``fresh``: int32 ``[forks, 2]`` free pages (such as the first ones of
    ``free_pages``), the child's first page and its copy of an unfinished last page (not used when
    the parent's tokens end with a page, or in the first one). In every layer the parent's records
    and window rows of those pages are copied, nothing else of them is written; table columns past
    the parent's last page keep their values.

    Returns int32 ``[forks]``: 1, or 0 for a fork that was refused and wrote nothing (a row outside
    the table, more tokens than its columns hold, a parent that is also some fork's child, a child
    row or a needed page that an earlier fork lists too, a needed page outside the pool or among the
    parent's own, a parent's page outside the pool). At most 4096 forks a call.
    """
    table = _table(caches, block_tables, seq_lens, parents=parents, children=children, fresh=fresh)
    forks = parents.numel()
    for name, t, shape in (("parents", parents, (forks,)), ("children", children, (forks,)),
                           ("fresh", fresh, (forks, 2))):
        if _int32(t, name).shape != shape or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor of shape {shape}")
    status = children.new_empty(forks)
    _launch(
        _ext.library().oscar_fork_requests, "fork_requests", caches.device,
        caches.stripes.data_ptr(), len(caches.views), caches.num_pages, *table,
        seq_lens.data_ptr(), parents.data_ptr(), children.data_ptr(), fresh.data_ptr(), forks,
        caches.layout_struct, status.data_ptr(),
    )
    return status


def compact_pages(caches, block_tables, seq_lens, counts):
    """Moves the pages in use to the pool's start in every layer.

    Returns ``(tables, live)``: int32 ``[1]`` the number of pages in use, and the block table with
    every live token's blocks where they are now, all below page ``live``, and -1 behind a live row's
    last page; the pages from there on are free. Rows that are not live come as they were. Pages below
    ``live`` that were in use stay, the k-th one above moves to the k-th free one below.
    ``block_tables`` is not changed (a caller with fixed buffers copies the new one in), slot
    mappings made from it are stale.
    """
    table = _table(caches, block_tables, seq_lens, counts)
    scratch = seq_lens.new_empty(5 * caches.num_pages + 1)
    tables, live = scratch.new_empty(block_tables.shape), scratch.new_empty(1)
    _launch(
        _ext.library().oscar_compact_pages, "compact_pages", caches.device,
        caches.stripes.data_ptr(), len(caches.views), caches.num_pages, *table,
        seq_lens.data_ptr(), counts.data_ptr(), caches.layout_struct, scratch.data_ptr(),
        tables.data_ptr(), live.data_ptr(),
    )
    return tables, live
