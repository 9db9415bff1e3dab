"""Tensors that share memory: the refusals of PagedCache."""
from __future__ import annotations

import pytest
import torch

from fireprot_amd import kv_cache


def test_caches_whose_tensors_overlap_are_refused():
    buffer = torch.zeros(3, 3, 16, 64, dtype=torch.int8)
    other, scales = torch.zeros(2, 3, 16, 64, dtype=torch.int8), torch.zeros(3, 3, 16)
    s, t = scales[:2], torch.zeros(2, 3, 16)
    kv_cache.PagedCache(buffer[:2], other, s, t)
    for args in ((buffer[:2], other, s, s), (buffer[:2], other, s, scales[1:]),
                 (buffer[:2], buffer[1:], s, t), (buffer[:2], buffer[:2], s, t),
                 (buffer[:2], other, buffer.view(torch.float32).flatten()[:96].view(2, 3, 16), t)):
        with pytest.raises(ValueError, match="share memory"):
            kv_cache.PagedCache(*args)
    # side by side in one buffer
    both = torch.zeros(4, 3, 16, 64, dtype=torch.float16)
    kv_cache.PagedCache(both[:2], both[2:])
    kv_cache.PagedCache(both[2:], both[:2])
