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
from .rotary import LAYOUTS, POSITION_DTYPES, RotaryFrequencies, _output, _rows


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
      A token with a negative slot or position (padding), past the table, or on a page
      outside the cache is not written; its query is turned all the same.  The other
      tokens' slots must be distinct.
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
    device, kind = cache.k.get_device(), ROW_DTYPES.get(k.dtype)
    if kind is None or device < 0 or k.get_device() != device:
        raise ValueError("k must be float32, bfloat16 or float16 on the cache's HIP device")
    if k.dim() not in (3, 4) or k.shape[-2:] != (heads, head_dim):
        raise ValueError(f"k must be [batch, tokens, {heads}, {head_dim}] or [tokens, {heads}, "
                         f"{head_dim}], got {tuple(k.shape)}")
    if v.shape != k.shape or v.dtype != k.dtype or v.get_device() != device:
        raise ValueError("v must have k's shape, type and device")
    x, y = _rows(k, "k"), _rows(v, "v")
    batch, tokens = x.shape[:2]
    inv_freq = frequencies.inv_freq
    rotary_dim = 2 * inv_freq.shape[0]
    if rotary_dim > head_dim:
        raise ValueError(f"needs rotary_dim ({rotary_dim}) <= head_dim ({head_dim})")
    wide = positions.dim() == 2
    place = POSITION_DTYPES.get(positions.dtype)
    if (place is None or positions.get_device() != device or inv_freq.get_device() != device
            or positions.shape != ((batch, tokens) if wide else (tokens,))):
        raise ValueError("positions must be int32 or int64 [batch, tokens] or [tokens], and they "
                         "and inv_freq on the cache's device")
    if (block_table is None) == (slots is None):
        raise ValueError("needs either block_table or slots")
    if slots is not None:
        if slots.shape != k.shape[:-2] or slots.dtype != torch.int64 or (
                slots.get_device() != device):
            raise ValueError(f"slots must be int64 {list(k.shape[:-2])} on the cache's device")
        if not slots.is_contiguous():
            slots = slots.contiguous()
        where = (slots.data_ptr(), None, 0, 0)
    else:
        if (block_table.dim() != 2 or block_table.shape[0] != batch
                or block_table.dtype != torch.int32 or block_table.get_device() != device):
            raise ValueError("block_table must be int32 [batch, pages] on the cache's device")
        if block_table.stride(1) != 1 and block_table.shape[1] > 1:
            block_table = block_table.contiguous()
        columns = block_table.shape[1]
        if columns == 0:  # (every token is past it, but it needs an address)
            block_table = block_table.new_empty((batch, 1))
        where = (None, block_table.data_ptr(), block_table.stride(0), columns)
    if _native.differentiated(q, k, v, q_out):
        raise ValueError("no autograd graph is recorded: call without gradients "
                         "(torch.no_grad, detach)")
    given = None
    q_args = out_args = (None, 0, 0, 0)
    q_heads = 0
    if q is not None:
        if (q.dtype != k.dtype or q.get_device() != device or q.dim() != k.dim()
                or q.shape[:-2] != k.shape[:-2] or q.shape[-1] != head_dim):
            raise ValueError("q must have k's type, device, batch, tokens and head_dim")
        z = _rows(q, "q")
        out, given = _output(q_out, q, z, "q_out")
        q_heads = z.shape[2]
        if q_heads:
            q_args = (z.data_ptr(), *z.stride()[:3])
            out_args = (out.data_ptr(), *out.stride()[:3])
    elif q_out is not None:
        raise ValueError("q_out needs q")
    if batch == 0 or tokens == 0:
        return given
    code = _native.launch(
        device, lib.fpx_cache_append, kind, CACHE_DTYPES[cache.k.dtype], mode, *q_args, *out_args,
        q_heads, x.data_ptr(), *x.stride()[:3], y.data_ptr(), *y.stride()[:3],
        positions.data_ptr(), place, positions.stride(0) if wide else 0, positions.stride(-1),
        inv_freq.data_ptr(), frequencies.scale, rotary_dim, *where, batch, tokens,
        *cache.pointers(), *cache.sizes)
    if code:
        _native.check(code, "fpx_cache_append")
    return given
