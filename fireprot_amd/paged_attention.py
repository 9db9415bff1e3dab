"""Attention of one new token per sequence over a paged key-value cache.

``paged_attention(q, cache, block_table, lengths)`` is the decoding step's
attention: each sequence's query heads attend to the keys its row of the block
table names, ``lengths[b]`` of them (the new token's own among them), where
they lie in the ``PagedCache`` (``fpx_paged_attention``).  Query heads share
cache heads in groups; 8-bit caches are dequantised on the way; scores, softmax
and sums are FP32, and so are the weights that meet the values of an FP32 output
(16-bit outputs: cut to 22 bits over an FP16 cache, to 16 over others).  All
sequences' keys are dealt out evenly to the card's
work-groups, and a second launch joins what several of them share.  There is no
counterpart in the reference.
"""
from __future__ import annotations

import torch

from . import _native
from .kv_cache import CACHE_DTYPES, CODED_DTYPES, ROW_DTYPES, PagedCache

NO_WORKSPACE = 256  # the size that stands for none


def workspace_bytes(q: torch.Tensor, cache: PagedCache, max_length: int, window: int = 0) -> int:
    """Device workspace of one call (any contents); 0 for unsupported sizes,
    ``NO_WORKSPACE`` where none is used."""
    return int(_native.library().fpx_paged_attention_workspace_bytes(
        CACHE_DTYPES[cache.k.dtype], q.shape[0], q.shape[1], cache.k.shape[1], cache.k.shape[3],
        max_length, window))


def _aligned_rows(t: torch.Tensor) -> bool:
    s0, s1, s2 = t.stride()
    e = 16 // t.element_size()
    return s2 == 1 and s0 % e == 0 and s1 % e == 0 and t.data_ptr() % 16 == 0


def paged_attention(q: torch.Tensor, cache: PagedCache, block_table: torch.Tensor,
                    lengths: torch.Tensor, *, scale: float | None = None, window: int = 0,
                    max_length: int | None = None, out: torch.Tensor | None = None,
                    return_lse: bool = False, workspace: torch.Tensor | None = None):
    """``out`` ``[batch, q_heads, head_dim]`` of q's type, or ``(out, lse)``.

    * ``q`` ``[batch, q_heads, head_dim]``, any strides; ``q_heads`` a multiple
      of the cache's heads, each of which serves consecutive query heads.  A
      plain cache has q's type, an 8-bit one takes float32 (below 2^110: products
      with the codes are formed in FP32), bfloat16 and float16 queries.
    * ``block_table`` int32 ``[batch, p]``: a sequence's pages in order.
      Entries past its length, or before its window, are not used.
    * ``lengths`` int32 ``[batch]``, up to ``max_length`` (default: what the
      table holds; a captured graph keeps the bound it was captured with).
    * ``scale`` of the scores, ``head_dim ** -0.5`` by default; ``window`` > 0
      keeps the last ``window`` keys only.
    * ``lse`` float32 ``[batch, q_heads]``: the logarithm of the softmax's sum.

    * ``workspace``: uint8, ``workspace_bytes`` of them, 256-byte aligned and not
      shared with a call that may overlap this one (by default each call, and
      each captured graph, takes its own from the caching allocator).

    A sequence of length 0 gives zeros (lse -inf).  One whose length is
    negative or above ``max_length``, or whose table names a page outside the
    cache, gives NaN.  ``out`` may be ``q`` itself; it and the workspace may share
    no other element with the call's tensors.  Records no autograd graph:
    a ``q`` that requires a gradient is refused under grad mode, one with a
    forward-mode tangent always.
    """
    lib = _native.library()
    k = cache.k
    device = k.get_device()
    if q.dim() != 3 or q.dtype not in ROW_DTYPES or device < 0 or q.get_device() != device:
        raise ValueError("q must be float32, bfloat16 or float16 [batch, q_heads, head_dim] on "
                         "the cache's HIP device")
    batch, q_heads, head_dim = q.shape
    pages, heads, page_size, cache_dim = k.shape
    if head_dim != cache_dim or q_heads < heads or q_heads % heads:
        raise ValueError(f"q must have head_dim {cache_dim} and a multiple of {heads} heads, "
                         f"got {tuple(q.shape)}")
    if k.dtype not in CODED_DTYPES and k.dtype != q.dtype:
        raise ValueError(f"a {k.dtype} cache needs {k.dtype} queries")
    if (block_table.dim() != 2 or block_table.shape[0] != batch or block_table.dtype != torch.int32
            or block_table.get_device() != device):
        raise ValueError("block_table must be int32 [batch, pages] on q's device")
    if lengths.shape != (batch,) or lengths.dtype != torch.int32 or lengths.get_device() != device:
        raise ValueError("lengths must be int32 [batch] on q's device")
    held = block_table.shape[1] * page_size
    if max_length is None:
        max_length = held
    if not 0 <= max_length <= held or window < 0:
        raise ValueError(f"needs 0 <= max_length ({max_length}) <= {held}, the block table's "
                         f"slots, and window ({window}) >= 0")
    if _native.differentiated(q, out):
        raise ValueError("no autograd graph is recorded: detach q (and out)")
    if not _aligned_rows(q):
        q = q.clone(memory_format=torch.contiguous_format)
    if block_table.stride(1) != 1 and block_table.shape[1] > 1:
        block_table = block_table.contiguous()
    if not lengths.is_contiguous():
        lengths = lengths.contiguous()
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif (out.shape != q.shape or out.dtype != q.dtype or out.get_device() != device
          or not _aligned_rows(out) or _native.repeats(out)):
        raise ValueError("out must have q's shape, type and device, 16-byte aligned rows and "
                         "no repeated elements")
    lse = q.new_empty((batch, q_heads), dtype=torch.float32) if return_lse else None
    size = lib.fpx_paged_attention_workspace_bytes(CACHE_DTYPES[k.dtype], batch, q_heads, heads,
                                                   head_dim, max_length, window)
    if size == 0:
        raise ValueError(f"unsupported sizes: batch {batch}, {q_heads} query heads, "
                         f"max_length {max_length}, window {window}")
    if workspace is not None:
        if (workspace.dtype != torch.uint8 or workspace.get_device() != device
                or workspace.numel() < size or not workspace.is_contiguous()):
            raise ValueError(f"workspace must be {size} contiguous bytes on q's device")
    elif size > NO_WORKSPACE:
        # of the current stream, and of the graph where one is captured: no two
        # calls that may overlap share it
        workspace = q.new_empty(size, dtype=torch.uint8)
    code = _native.launch(
        device, lib.fpx_paged_attention, ROW_DTYPES[q.dtype], CACHE_DTYPES[k.dtype],
        q.data_ptr(), *q.stride()[:2], *cache.pointers(), pages, heads, page_size, head_dim,
        block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
        lengths.data_ptr(), batch, q_heads, max_length, window,
        head_dim ** -0.5 if scale is None else scale, out.data_ptr(), *out.stride()[:2],
        None if lse is None else lse.data_ptr(),
        None if workspace is None else workspace.data_ptr(), size)
    if code:
        _native.check(code, "fpx_paged_attention")
    return (out, lse) if return_lse else out
