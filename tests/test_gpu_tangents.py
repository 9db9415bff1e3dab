"""Forward-mode tangents on the device: refused by every decoding entry, by functional
transforms too."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from fireprot_amd import kv_cache, rotary
from fireprot_amd.paged_attention import paged_attention

pytestmark = pytest.mark.gpu


def test_entries_refuse_a_tangent():
    cache = kv_cache.PagedCache.allocate(4, 2, 16, 64, dtype=torch.float32)
    rows = torch.randn(5, 2, 64, device="cuda")
    slots = torch.arange(5, device="cuda")
    table = torch.arange(4, device="cuda", dtype=torch.int32).view(1, 4)
    lengths = torch.tensor([5], device="cuda", dtype=torch.int32)
    q = torch.randn(1, 2, 64, device="cuda")
    f = rotary.rotary_frequencies(64, device="cuda")
    position = torch.arange(1, device="cuda")
    kv_cache.cache_write(cache, rows, rows.clone(), slots)
    want, kept = paged_attention(q, cache, table, lengths), cache.k.clone()
    with forward_ad.dual_level(), torch.no_grad():
        assert torch.equal(paged_attention(q, cache, table, lengths), want)
        dual, dual_q = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (rows, q))
        for call in (lambda: kv_cache.cache_write(cache, dual, rows, slots),
                     lambda: kv_cache.cache_write(cache, rows, dual, slots),
                     lambda: kv_cache.cache_read(cache, slots, v_out=dual),
                     lambda: paged_attention(dual_q, cache, table, lengths),
                     lambda: paged_attention(q, cache, table, lengths, out=dual_q),
                     lambda: rotary.apply_rotary(dual_q[None], None, position, f)):
            with pytest.raises(ValueError, match="gradient|autograd"):
                call()
    with torch.no_grad(), pytest.raises((ValueError, RuntimeError)):
        torch.func.jvp(lambda x: paged_attention(x, cache, table, lengths), (q,),
                       (torch.ones_like(q),))
    torch.cuda.synchronize()
    assert torch.equal(cache.k, kept)
