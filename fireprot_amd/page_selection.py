"""Attention over the pages that matter, on gfx950: bounds of each page's keys, and the
choice of pages by them.

``PageBounds`` holds, for every page and head of a ``PagedCache``, the least and the
greatest value of each channel of its keys.  ``update_page_bounds`` forms them for the
pages of the newest tokens (``fpx_page_bounds``), ``select_pages`` takes, for one new
token's queries, the pages on which a key may score highest (``fpx_select_pages``), and
``paged_attention(q, cache, chosen.table, chosen.lengths)`` attends to those alone: of a
long context a step reads the bounds (two rows a page) and ``count`` pages of keys and
values for each cache head.  There is no counterpart in the reference.

No call records an autograd graph: queries that require a gradient are refused under
grad mode, those with a forward-mode tangent always.
"""
from __future__ import annotations

import dataclasses

import torch

from . import _native
from .kv_cache import (CACHE_DTYPES, CODED_DTYPES, HEAD_DIMS, PAGE_SIZES, ROW_DTYPES, PagedCache)
from .paged_attention import _aligned_rows

NO_WORKSPACE = 256  # the size that stands for none


def bounds_dtype(cache_dtype: torch.dtype) -> torch.dtype:
    """The type of a cache's bounds: its own, bfloat16 for a cache in 8 or 4 bits."""
    return torch.bfloat16 if cache_dtype in CODED_DTYPES else cache_dtype


@dataclasses.dataclass(frozen=True, eq=False)
class PageBounds:
    """``values`` contiguous ``[pages, heads, 2, head_dim]``: the least, then the
    greatest value of each channel of a page's keys; ``page_size`` of the cache."""

    values: torch.Tensor
    page_size: int

    def __post_init__(self) -> None:
        t = self.values
        if t.dim() != 4 or t.shape[2] != 2 or t.shape[3] not in HEAD_DIMS or (
                t.dtype not in ROW_DTYPES or 0 in t.shape):
            raise ValueError("values must be float32, bfloat16 or float16 [pages, heads, 2, "
                             f"head_dim] with head_dim in {HEAD_DIMS}")
        if self.page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}")
        if not t.is_contiguous() or t.data_ptr() % 16:
            raise ValueError("values must be contiguous and 16-byte aligned")
        if t.requires_grad:
            raise ValueError("bounds record no gradient: detach values")

    @classmethod
    def allocate(cls, cache: PagedCache) -> "PageBounds":
        """Zeros for ``cache``: ``update_page_bounds`` fills in what sequences hold."""
        pages, heads, page_size, head_dim = cache.sizes
        return cls(torch.zeros((pages, heads, 2, head_dim), dtype=bounds_dtype(cache.dtype),
                               device=cache.device), page_size)


@dataclasses.dataclass(frozen=True, eq=False)
class PageSelection:
    """``table`` int32 ``[batch, heads, count]``: the chosen pages, in the order of the
    sequence; ``index`` their places in it; both -1 past a sequence's pages.
    ``lengths`` int32 ``[batch]``: the keys on them."""

    table: torch.Tensor
    lengths: torch.Tensor
    index: torch.Tensor


def _sequences(block_table, lengths, device, batch, page_size, max_length):
    """(table, its stride, its pages a sequence, lengths, max_length), checked, rows of
    unit stride."""
    shape = block_table.shape
    if (len(shape) != 2 or shape[0] != batch or block_table.dtype != torch.int32
            or block_table.get_device() != device):
        raise ValueError("block_table must be int32 [batch, pages] on the cache's device")
    if lengths.shape != (batch,) or lengths.dtype != torch.int32 or lengths.get_device() != device:
        raise ValueError("lengths must be int32 [batch] on the cache's device")
    columns = shape[1]
    held = columns * page_size
    if max_length is None:
        max_length = held
    if not 0 <= max_length <= held:
        raise ValueError(f"needs 0 <= max_length ({max_length}) <= {held}, the block table's slots")
    row, one = block_table.stride()
    if one != 1 and columns > 1:
        block_table = block_table.contiguous()
        row = columns
    if not lengths.is_contiguous():
        lengths = lengths.contiguous()
    return block_table, row, columns, lengths, max_length


def update_page_bounds(bounds: PageBounds, cache: PagedCache, block_table: torch.Tensor,
                       lengths: torch.Tensor, *, new: int = 1,
                       max_length: int | None = None) -> None:
    """Form the bounds of the pages that hold the last ``new`` tokens of each sequence
    (a step: 1; a prompt: its length, or the longest of a batch), from the keys below
    its length.  Pages of earlier tokens keep theirs.  (A page that several sequences
    hold must be full in all of them: its bounds are those of its keys in one.)

    ``block_table``, ``lengths`` and ``max_length`` as ``paged_attention``'s.  A
    sequence whose length is negative or above ``max_length``, and an entry that names
    no page of the cache, is passed over.  A NaN among the keys makes its channel's
    bounds NaN.
    """
    lib = _native.library()
    pages, heads, page_size, head_dim = cache.sizes
    device = cache.k.get_device()
    values = bounds.values
    if device < 0 or values.get_device() != device:
        raise ValueError("the cache and its bounds must be on one HIP device")
    if (values.shape != (pages, heads, 2, head_dim) or bounds.page_size != page_size
            or values.dtype != bounds_dtype(cache.k.dtype)):
        raise ValueError("the bounds are not of this cache: PageBounds.allocate(cache)")
    batch = lengths.shape[0] if lengths.dim() == 1 else -1
    block_table, row, columns, lengths, max_length = _sequences(
        block_table, lengths, device, batch, page_size, max_length)
    if new < 1:
        raise ValueError(f"needs new ({new}) >= 1")
    k_scale = cache.k_scale
    code = _native.launch(
        device, lib.fpx_page_bounds, CACHE_DTYPES[cache.k.dtype], cache.k.data_ptr(),
        None if k_scale is None else k_scale.data_ptr(), pages, heads, page_size, head_dim,
        block_table.data_ptr(), row, columns, lengths.data_ptr(), batch, max_length,
        min(new, max_length + 1), values.data_ptr())
    if code:
        _native.check(code, "fpx_page_bounds")


def select_pages(q: torch.Tensor, bounds: PageBounds, block_table: torch.Tensor,
                 lengths: torch.Tensor, count: int, *, sinks: int = 0, recent: int = 1,
                 max_length: int | None = None,
                 workspace: torch.Tensor | None = None) -> PageSelection:
    """The ``count`` pages that each sequence's queries attend to, for each cache head.

    The first ``sinks`` and the last ``recent`` (at least one: the new token's own) pages
    of a sequence are always among them; the others are those with the highest ``max
    over the head's queries of sum_c max(q_c lo_c, q_c hi_c)``, which no key of the page
    exceeds.  The sum is taken in FP64 and rounded to FP32; of equal pages the lower
    comes first, NaN and pages outside the cache above all (NaN are zero times an infinite
    bound and a sum of both infinities).  A sequence of no more than ``count`` pages keeps
    them all; the outputs have ``count`` places whatever the table holds, and an attention
    over them plans for as many unless its ``max_length`` says less.

    * ``q`` ``[batch, q_heads, head_dim]`` as ``paged_attention``'s, ``q_heads`` a
      multiple of the bounds' heads; for a negative ``scale`` of the scores pass ``-q``.
    * ``block_table``, ``lengths`` (with the new token), ``max_length``: as there.  A
      length that is negative or above ``max_length`` gives -1, whose attention is NaN.
    * ``workspace``: uint8, ``select_workspace_bytes`` of them, 256-byte aligned and not
      shared with a call that may overlap this one (by default each call, and each
      captured graph, takes its own from the caching allocator).
    """
    lib = _native.library()
    values, page_size = bounds.values, bounds.page_size
    pages, heads, _, head_dim = values.shape
    device = values.get_device()
    kind = ROW_DTYPES.get(q.dtype)
    if q.dim() != 3 or kind is None or device < 0 or q.get_device() != device:
        raise ValueError("q must be float32, bfloat16 or float16 [batch, q_heads, head_dim] on "
                         "the bounds' HIP device")
    batch, q_heads, q_dim = q.shape
    if q_dim != head_dim or q_heads < heads or q_heads % heads:
        raise ValueError(f"q must have head_dim {head_dim} and a multiple of {heads} heads, got "
                         f"{tuple(q.shape)}")
    block_table, row, columns, lengths, max_length = _sequences(
        block_table, lengths, device, batch, page_size, max_length)
    if sinks < 0 or recent < 1 or count < sinks + recent:
        raise ValueError(f"needs sinks ({sinks}) >= 0, recent ({recent}) >= 1 and count ({count}) "
                         ">= their sum")
    if count * page_size >= 1 << 30:
        raise ValueError(f"count ({count}) pages of {page_size} slots are 2^30 keys or more")
    if _native.differentiated(q):
        raise ValueError("no autograd graph is recorded: detach q")
    if not _aligned_rows(q):
        q = q.clone(memory_format=torch.contiguous_format)
    size = lib.fpx_select_pages_workspace_bytes(batch, heads, page_size, max_length, count)
    if size == 0:
        raise ValueError(f"unsupported sizes: batch {batch}, max_length {max_length}")
    if workspace is not None:
        if (workspace.dtype != torch.uint8 or workspace.get_device() != device
                or workspace.numel() < size or not workspace.is_contiguous()):
            raise ValueError(f"workspace must be {size} contiguous bytes on q's device")
    elif size > NO_WORKSPACE:
        workspace = q.new_empty(size, dtype=torch.uint8)
    table = lengths.new_empty((batch, heads, count))
    index, kept = torch.empty_like(table), torch.empty_like(lengths)
    code = _native.launch(
        device, lib.fpx_select_pages, kind, ROW_DTYPES[values.dtype], q.data_ptr(),
        *q.stride()[:2], q_heads, values.data_ptr(), pages, heads, page_size, head_dim,
        block_table.data_ptr(), row, columns, lengths.data_ptr(), batch, max_length, count,
        sinks, recent, index.data_ptr(), table.data_ptr(), kept.data_ptr(),
        None if workspace is None else workspace.data_ptr(), size)
    if code:
        _native.check(code, "fpx_select_pages")
    return PageSelection(table, kept, index)


def select_workspace_bytes(q: torch.Tensor, bounds: PageBounds, max_length: int,
                           count: int) -> int:
    """Device workspace of one ``select_pages`` call (any contents); 0 for unsupported
    sizes, ``NO_WORKSPACE`` where none is used."""
    return int(_native.library().fpx_select_pages_workspace_bytes(
        q.shape[0], bounds.values.shape[1], bounds.page_size, max_length, count))
