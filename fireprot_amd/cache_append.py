"""New tokens into the paged cache on gfx950, turned by their positions, in one launch.

``cache_append(cache, q, k, v, positions, frequencies, block_table=...)`` is the write
half of a decoding step (or of a prompt): queries and keys turned as ``apply_rotary``
turns them, keys and values put at their slots as ``cache_write`` puts them, the slots
found in the block table as ``cache_slots`` finds them (``fpx_cache_append``).  The
turned keys exist only in the cache: they are converted from FP32, with one rounding,
where the three calls round to the rows' type in between.  There is no counterpart in
the reference.
"""
from __future__ import annotations

import torch

from . import _native
from .kv_cache import CACHE_DTYPES, ROW_DTYPES, PagedCache
from .rotary import LAYOUTS, POSITION_DTYPES, RotaryFrequencies, _output

# (Shapes and strides are asked for once each below: a question to a tensor takes 0.1 to
# 0.2 us, and a step's call is some 40 of them beside its launch.)


def _placed(t: torch.Tensor) -> tuple[torch.Tensor, tuple[int, ...]]:
    """``t``, of three or four axes, with unit channel stride, and what its pointer
    comes with: strides of (batch, token, head)."""
    strides = t.stride()
    if strides[-1] != 1:
        t = t.contiguous()
        strides = t.stride()
    return t, strides[:3] if len(strides) == 4 else (0, *strides[:2])


def cache_append(cache: PagedCache, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor,
                 positions: torch.Tensor, frequencies: RotaryFrequencies, *,
                 block_table: torch.Tensor | None = None, slots: torch.Tensor | None = None,
                 layout: str = "half", q_out: torch.Tensor | None = None):
    """The turned queries (None where ``q`` is None); the keys, turned, and the values
    go into the cache.

    * ``q`` ``[batch, tokens, q_heads, head_dim]``, ``k`` and ``v`` ``[batch, tokens,
      heads, head_dim]`` (or all without the batch axis): float32, bfloat16 or float16,
      one type, any non-negative strides; the cache may be of any type.
    * ``positions`` ``[batch, tokens]`` or ``[tokens]``, int32 or int64: what rows are
      turned by, and with ``block_table`` also their places in the sequences.
    * ``block_table`` int32 ``[batch, p]``, the sequences' pages in order, or ``slots``
      int64 ``[batch, tokens]`` (``[tokens]`` without the batch axis): one of the two.
      By ``block_table`` a token with a negative position (padding), past the table, or on
      a page outside the cache is not written; by ``slots`` one with a negative slot, or
      past the cache (its position, negative or not, only turns it, so padding has to show
      in ``slots``).  Its query is turned all the same.  The other tokens' slots must be
      distinct.
    * ``q_out=q`` works in place; an output that shares an element with anything else is
      refused, as are inputs that are rows of this cache.

    Records no autograd graph: tensors that require a gradient are refused under grad
    mode, those with a forward-mode tangent always.
    """
    lib = _native.library()
    mode = LAYOUTS.get(layout)
    if mode is None:
        raise ValueError(f"layout must be one of {sorted(LAYOUTS)}")
    _, heads, _, head_dim = cache.sizes
    held, dtype, shape = cache.k, k.dtype, k.shape
    device, kind = held.get_device(), ROW_DTYPES.get(dtype)
    if kind is None or device < 0 or k.get_device() != device:
        raise ValueError("k must be float32, bfloat16 or float16 on the cache's HIP device")
    axes = len(shape)
    if axes not in (3, 4) or shape[-2] != heads or shape[-1] != head_dim:
        raise ValueError(f"k must be [batch, tokens, {heads}, {head_dim}] or [tokens, {heads}, "
                         f"{head_dim}], got {tuple(shape)}")
    if v.shape != shape or v.dtype != dtype or v.get_device() != device:
        raise ValueError("v must have k's shape, type and device")
    batch, tokens = (shape[0], shape[1]) if axes == 4 else (1, shape[0])
    inv_freq = frequencies.inv_freq
    rotary_dim = 2 * inv_freq.shape[0]
    if rotary_dim > head_dim:
        raise ValueError(f"needs rotary_dim ({rotary_dim}) <= head_dim ({head_dim})")
    strides = positions.stride()
    wide = len(strides) == 2
    place = POSITION_DTYPES.get(positions.dtype)
    if (place is None or positions.get_device() != device or inv_freq.get_device() != device
            or positions.shape != ((batch, tokens) if wide else (tokens,))):
        raise ValueError("positions must be int32 or int64 [batch, tokens] or [tokens], and they "
                         "and inv_freq on the cache's device")
    if (block_table is None) == (slots is None):
        raise ValueError("needs either block_table or slots")
    if slots is not None:
        if slots.shape != shape[:-2] or slots.dtype != torch.int64 or (
                slots.get_device() != device):
            raise ValueError(f"slots must be int64 {list(shape[:-2])} on the cache's device")
        if not slots.is_contiguous():
            slots = slots.contiguous()
        where = (slots.data_ptr(), None, 0, 0)
    else:
        pages = block_table.shape
        if (len(pages) != 2 or pages[0] != batch or block_table.dtype != torch.int32
                or block_table.get_device() != device):
            raise ValueError("block_table must be int32 [batch, pages] on the cache's device")
        columns = pages[1]
        if columns == 0:  # (every token is past it, but it needs an address)
            block_table = block_table.new_empty((batch, 1))
        elif columns > 1 and block_table.stride(1) != 1:
            block_table = block_table.contiguous()
        where = (None, block_table.data_ptr(), block_table.stride(0), columns)
    if _native.differentiated(q, k, v, q_out):
        raise ValueError("no autograd graph is recorded: call without gradients "
                         "(torch.no_grad, detach)")
    given = None
    q_args = out_args = (None, 0, 0, 0)
    q_heads = 0
    if q is not None:
        sizes = q.shape
        if (q.dtype != dtype or q.get_device() != device or len(sizes) != axes
                or sizes[:-2] != shape[:-2] or sizes[-1] != head_dim):
            raise ValueError("q must have k's type, device, batch, tokens and head_dim")
        z, apart = _placed(q)
        q_heads = sizes[-2]
        if q_out is None:
            given = torch.empty_like(q, memory_format=torch.contiguous_format)
            out_apart = (tokens * q_heads * head_dim, q_heads * head_dim, head_dim)
        else:
            given = _output(q_out, q, z, "q_out")[1]
            out_apart = _placed(given)[1]
        if q_heads:
            q_args = (z.data_ptr(), *apart)
            out_args = (given.data_ptr(), *out_apart)
    elif q_out is not None:
        raise ValueError("q_out needs q")
    if batch == 0 or tokens == 0:
        return given
    x, x_apart = _placed(k)
    y, y_apart = _placed(v)
    code = _native.launch(
        device, lib.fpx_cache_append, kind, CACHE_DTYPES[held.dtype], mode, *q_args, *out_args,
        q_heads, x.data_ptr(), *x_apart, y.data_ptr(), *y_apart,
        positions.data_ptr(), place, strides[0] if wide else 0, strides[-1],
        inv_freq.data_ptr(), frequencies.scale, rotary_dim, *where, batch, tokens,
        *cache.pointers(), *cache.sizes)
    if code:
        _native.check(code, "fpx_cache_append")
    return given
