"""A paged key-value cache on gfx950, plain or in 8 bits.

``PagedCache`` holds keys and values in pages of a power of two of slots, one
head's rows of a page contiguous: ``[pages, heads, page_size, head_dim]``.  A
sequence's tokens sit in any pages, in the order of its row of a block table;
``cache_slots`` gives the slots of positions.  ``cache_write`` puts the rows of
new tokens at their slots, converted or quantised as they are written
(float8_e4m3fn with a power-of-two scale per row, int8 with a scale per row),
``cache_read`` brings rows back, and ``paged_attention`` attends to them where
they are.  There is no counterpart in the reference.

No call records an autograd graph: rows that require a gradient are refused
under grad mode, those with a forward-mode tangent always.
"""
from __future__ import annotations

import dataclasses
from typing import Any

import torch

from . import _native

HEAD_DIMS = (32, 64, 128, 256)
PAGE_SIZES = tuple(1 << i for i in range(4, 13))
ROW_DTYPES = {torch.float32: _native.FPX_F32, torch.bfloat16: _native.FPX_BF16,
              torch.float16: _native.FPX_F16}
CODED_DTYPES = {torch.float8_e4m3fn: _native.FPX_F8E4M3, torch.int8: _native.FPX_I8}
CACHE_DTYPES = {**ROW_DTYPES, **CODED_DTYPES}


@dataclasses.dataclass(frozen=True, eq=False)
class PagedCache:
    """``k`` and ``v`` contiguous ``[pages, heads, page_size, head_dim]``;
    ``k_scale`` and ``v_scale`` float32 ``[pages, heads, page_size]`` for the
    8-bit types, None for the others."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor | None = None
    v_scale: torch.Tensor | None = None

    def __post_init__(self) -> None:
        k, v = self.k, self.v
        if k.dim() != 4 or k.dtype not in CACHE_DTYPES:
            raise ValueError("k must be [pages, heads, page_size, head_dim] of a type in "
                             f"{[str(t) for t in CACHE_DTYPES]}")
        if v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
            raise ValueError("v must have k's shape, type and device")
        pages, heads, page_size, head_dim = k.shape
        if head_dim not in HEAD_DIMS or page_size not in PAGE_SIZES or pages < 1 or heads < 1:
            raise ValueError(f"needs head_dim in {HEAD_DIMS}, page_size in {PAGE_SIZES}, and at "
                             "least one page and head")
        if k.requires_grad or v.requires_grad:
            raise ValueError("a cache records no gradient: detach k and v")
        scales = (self.k_scale, self.v_scale)
        if k.dtype in CODED_DTYPES:
            if any(s is None or s.shape != k.shape[:3] or s.dtype != torch.float32
                   or s.device != k.device for s in scales):
                raise ValueError("an 8-bit cache needs float32 scales [pages, heads, page_size] "
                                 "on its device")
        elif any(s is not None for s in scales):
            raise ValueError("only an 8-bit cache has scales")
        for t in (k, v, *scales):
            if t is not None and (not t.is_contiguous() or t.data_ptr() % 16):
                raise ValueError("the cache's tensors must be contiguous and 16-byte aligned")
        ranges = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size())
                        for t in (k, v, *scales) if t is not None)
        if any(end > begin for (_, end), (begin, _) in zip(ranges, ranges[1:])):
            raise ValueError("k, v and their scales must not share memory")

    @classmethod
    def allocate(cls, pages: int, heads: int, page_size: int, head_dim: int, *,
                 dtype: torch.dtype, device: Any = "cuda") -> "PagedCache":
        """A cache of zeros."""
        def zeros(shape, kind):
            return torch.zeros(shape, dtype=kind, device=device)

        shape = (pages, heads, page_size, head_dim)
        coded = dtype in CODED_DTYPES
        scales = [zeros(shape[:3], torch.float32) if coded else None for _ in range(2)]
        return cls(zeros(shape, dtype), zeros(shape, dtype), *scales)

    @property
    def pages(self) -> int:
        return self.k.shape[0]

    @property
    def heads(self) -> int:
        return self.k.shape[1]

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    @property
    def head_dim(self) -> int:
        return self.k.shape[3]

    @property
    def dtype(self) -> torch.dtype:
        return self.k.dtype

    @property
    def device(self) -> torch.device:
        return self.k.device

    def pointers(self) -> tuple[int | None, ...]:
        return (self.k.data_ptr(), self.v.data_ptr(),
                None if self.k_scale is None else self.k_scale.data_ptr(),
                None if self.v_scale is None else self.v_scale.data_ptr())


def cache_slots(block_table: torch.Tensor, positions: torch.Tensor,
                page_size: int) -> torch.Tensor:
    """Slots (int64, ``[batch, n]``) of ``positions`` ``[batch, n]`` of
    sequences whose pages are the rows of ``block_table`` ``[batch, p]``.
    A negative position is no token (slot -1); one past the table, or whose entry
    there is negative and so names no page, gets a slot past every cache."""
    if block_table.dim() != 2 or positions.dim() != 2 or len(positions) != len(block_table):
        raise ValueError("block_table must be [batch, p] and positions [batch, n]")
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}")
    room = block_table.shape[1] * page_size
    if room == 0:
        inside = torch.full_like(positions, torch.iinfo(torch.int64).max, dtype=torch.int64)
    else:
        held = positions.long().clamp(0, room - 1)
        page = block_table.long().gather(1, held // page_size)
        outside = (positions >= room) | (page < 0)
        inside = torch.where(outside, torch.iinfo(torch.int64).max,
                             page * page_size + held % page_size)
    return torch.where(positions < 0, -1, inside)


def _check_rows(t: torch.Tensor, name: str, shape: tuple[int, int, int], device: int) -> None:
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {tuple(t.shape)}")
    if t.dtype not in ROW_DTYPES or t.get_device() != device:
        raise ValueError(f"{name} must be float32, bfloat16 or float16 on the cache's device")


def _check_slots(slots: torch.Tensor, device: int) -> torch.Tensor:
    if device < 0:
        raise ValueError("the cache must be on a HIP device")
    if slots.dim() != 1 or slots.dtype != torch.int64 or slots.get_device() != device:
        raise ValueError("slots must be an int64 vector on the cache's device")
    return slots if slots.is_contiguous() else slots.contiguous()


def _call(entry, what, device, row_dtype, cache, k, v, slots):
    code = _native.launch(
        device, entry, ROW_DTYPES[row_dtype], CACHE_DTYPES[cache.k.dtype],
        k.data_ptr(), *k.stride()[:2], v.data_ptr(), *v.stride()[:2],
        slots.data_ptr(), slots.shape[0], *cache.pointers(), *cache.k.shape)
    if code:
        _native.check(code, what)


def cache_write(cache: PagedCache, k: torch.Tensor, v: torch.Tensor,
                slots: torch.Tensor) -> None:
    """Put token ``t``'s rows ``k[t]`` and ``v[t]`` (``[tokens, heads,
    head_dim]``, float32, bfloat16 or float16, any strides) at ``slots[t]``.

    A token with a negative slot (padding) or one past the cache is not
    written; everything else in the cache stays as it is.  The other slots
    must be distinct, as with ``torch.Tensor.index_copy_``: of two tokens with
    one slot it is not defined what the slot holds.  ``k`` and ``v`` may not be
    rows of this cache (the library refuses them).
    """
    lib = _native.library()
    _, heads, _, head_dim = cache.k.shape
    device = cache.k.get_device()
    slots = _check_slots(slots, device)
    shape = (slots.shape[0], heads, head_dim)
    _check_rows(k, "k", shape, device)
    _check_rows(v, "v", shape, device)
    if v.dtype != k.dtype:
        raise ValueError("k and v must have one type")
    if _native.differentiated(k, v):
        raise ValueError("a cache records no gradient: detach k and v")
    if k.stride(2) != 1:
        k = k.contiguous()
    if v.stride(2) != 1:
        v = v.contiguous()
    _call(lib.fpx_cache_write, "fpx_cache_write", device, k.dtype, cache, k, v, slots)


def cache_read(cache: PagedCache, slots: torch.Tensor, *, dtype: torch.dtype | None = None,
               k_out: torch.Tensor | None = None, v_out: torch.Tensor | None = None
               ) -> tuple[torch.Tensor, torch.Tensor]:
    """``(k, v)``, each ``[tokens, heads, head_dim]`` of ``dtype`` (the outputs'
    where given, the cache's own for a plain cache, float32 for an 8-bit one):
    the rows at ``slots``, dequantised in 32 bits and rounded once.  A negative
    slot gives zeros, one past the cache NaN.  Slots may repeat.  Outputs that share
    an element with each other, themselves or the cache are refused, views that only
    interleave are not."""
    lib = _native.library()
    _, heads, _, head_dim = cache.k.shape
    device = cache.k.get_device()
    slots = _check_slots(slots, device)
    if dtype is None:
        given = k_out if k_out is not None else v_out
        dtype = (given.dtype if given is not None
                 else torch.float32 if cache.dtype in CODED_DTYPES else cache.dtype)
    if dtype not in ROW_DTYPES:
        raise ValueError("rows are read as float32, bfloat16 or float16")
    outs, shape = [], (slots.shape[0], heads, head_dim)
    for out, name in ((k_out, "k_out"), (v_out, "v_out")):
        if out is None:
            out = slots.new_empty(shape, dtype=dtype)
        else:
            _check_rows(out, name, shape, device)
            if out.dtype != dtype or out.stride(2) != 1 or _native.repeats(out):
                raise ValueError(f"{name} must be {dtype} with unit channel stride and no "
                                 "repeated elements")
            if _native.differentiated(out):
                raise ValueError("a cache records no gradient: detach the outputs")
        outs.append(out)
    if outs[0].data_ptr() == outs[1].data_ptr() and outs[0].numel():
        raise ValueError("k_out and v_out must not share memory")
    _call(lib.fpx_cache_read, "fpx_cache_read", device, dtype, cache, outs[0], outs[1], slots)
    return outs[0], outs[1]
