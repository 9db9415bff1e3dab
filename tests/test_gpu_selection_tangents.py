"""Forward-mode tangents and gradients on the device: refused by ``cache_append`` and by
``select_pages``, which then have written nothing."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from fireprot_amd import rotary
from fireprot_amd.cache_append import cache_append
from fireprot_amd.kv_cache import FP4, PagedCache
from fireprot_amd.page_selection import PageBounds, select_pages, update_page_bounds
from fireprot_amd.paged_attention import paged_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", (torch.float32, FP4))
def test_entries_refuse_a_tangent_and_a_gradient(dtype):
    cache = PagedCache.allocate(4, 2, 16, 64, dtype=dtype)
    bounds = PageBounds.allocate(cache)
    rows = torch.randn(1, 40, 2, 64, device="cuda")
    table = torch.arange(4, device="cuda", dtype=torch.int32).view(1, 4)
    lengths = torch.tensor([40], device="cuda", dtype=torch.int32)
    f = rotary.rotary_frequencies(64, device="cuda")
    positions = torch.arange(40, device="cuda")

    def append(q, k, v, out=None):
        return cache_append(cache, q, k, v, positions, f, block_table=table, q_out=out)

    def codes():
        return [t.view(torch.uint8).clone() for t in (cache.k, cache.v, bounds.values)]

    turned = append(rows, rows.clone(), rows.clone())
    update_page_bounds(bounds, cache, table, lengths, new=40)
    q = turned[:, -1].contiguous()
    chosen, kept = select_pages(q, bounds, table, lengths, 2), codes()
    for need in (q.clone().requires_grad_(), rows.clone().requires_grad_()):
        calls = ((lambda: select_pages(need, bounds, table, lengths, 2),
                  lambda: paged_attention(need, cache, chosen.table, chosen.lengths))
                 if need.dim() == 3 else
                 (lambda: append(need, rows, rows), lambda: append(rows, need, rows),
                  lambda: append(rows, rows, need), lambda: append(None, need, rows)))
        for call in calls:
            with pytest.raises(ValueError, match="gradient|autograd"):
                call()
    with forward_ad.dual_level(), torch.no_grad():
        dual_q, dual = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (q, rows))
        assert torch.equal(select_pages(q, bounds, table, lengths, 2).index, chosen.index)
        for call in (lambda: select_pages(dual_q, bounds, table, lengths, 2),
                     lambda: paged_attention(dual_q, cache, chosen.table, chosen.lengths),
                     lambda: append(dual, rows, rows), lambda: append(rows, dual, rows),
                     lambda: append(rows, rows, dual), lambda: append(rows, rows, rows, dual)):
            with pytest.raises(ValueError, match="gradient|autograd"):
                call()
    with torch.no_grad(), pytest.raises((ValueError, RuntimeError)):
        torch.func.jvp(lambda x: select_pages(x, bounds, table, lengths, 2).index, (q,),
                       (torch.ones_like(q),))
    torch.cuda.synchronize()
    assert all(map(torch.equal, codes(), kept))
    # without gradients asked for, the same tensors are taken
    with torch.no_grad():
        assert torch.equal(append(rows.clone().requires_grad_(), rows, rows), turned)
