"""Outputs that share memory, on the device: those that share an element with another
tensor of the call are refused and leave everything as it was; views of one buffer
that interleave come out as separate tensors do."""
from __future__ import annotations

import pytest
import torch

from fireprot_amd import kv_cache, rotary
from fireprot_amd.paged_attention import paged_attention, workspace_bytes

pytestmark = pytest.mark.gpu


def test_rotary_outputs():
    f = rotary.rotary_frequencies(64, device="cuda")
    fused = torch.randn(2, 9, 10 * 64, device="cuda").bfloat16()
    q, k = fused[..., :6 * 64].view(2, 9, 6, 64), fused[..., 6 * 64:8 * 64].view(2, 9, 2, 64)
    positions = torch.arange(9, device="cuda")
    want = rotary.apply_rotary(q, k, positions, f)
    out = torch.zeros(2, 9, 8, 64, device="cuda", dtype=torch.bfloat16)
    rotary.apply_rotary(q, k, positions, f, q_out=out[:, :, :6], k_out=out[:, :, 6:])
    assert torch.equal(out[:, :, :6], want[0]) and torch.equal(out[:, :, 6:], want[1])
    before = fused.clone()
    flat = out.flatten()
    for kw in (dict(q_out=out[:, :, 1:7], k_out=out[:, :, 6:]),
               dict(q_out=fused[..., 32:6 * 64 + 32].view(2, 9, 6, 64)),
               dict(k_out=fused[..., 4 * 64:6 * 64].view(2, 9, 2, 64)),
               dict(q_out=flat.as_strided((2, 9, 6, 64), (9 * 6 * 64, 5 * 64, 64, 1)))):
        with pytest.raises(RuntimeError, match="overlap"):
            rotary.apply_rotary(q, k, positions, f, **kw)
    torch.cuda.synchronize()
    assert torch.equal(fused, before) and torch.equal(out[:, :, :6], want[0])
    # in place through one buffer, whose halves interleave
    rotary.apply_rotary(q, k, positions, f, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(fused[..., 8 * 64:], before[..., 8 * 64:])


def test_rows_read_and_written():
    cache = kv_cache.PagedCache.allocate(4, 2, 16, 64, dtype=torch.bfloat16)
    rows = torch.randn(2, 20, 2, 64, device="cuda").bfloat16()
    slots = torch.arange(20, device="cuda") + 3
    kv_cache.cache_write(cache, rows[0], rows[1], slots)
    both = torch.zeros(20, 4, 64, device="cuda", dtype=torch.bfloat16)
    kv_cache.cache_read(cache, slots, k_out=both[:, :2], v_out=both[:, 2:])
    assert torch.equal(both[:, :2], rows[0]) and torch.equal(both[:, 2:], rows[1])
    kept = cache.k.clone(), both.clone()
    inside = cache.k.flatten()[64:64 + 20 * 2 * 64].view(20, 2, 64)
    for kw in (dict(k_out=both[:, :2], v_out=both[:, 1:3]), dict(k_out=inside),
               dict(k_out=both.flatten().as_strided((20, 2, 64), (64, 64, 1)))):
        with pytest.raises(RuntimeError, match="overlap"):
            kv_cache.cache_read(cache, slots, **kw)
    with pytest.raises(RuntimeError, match="overlap"):
        kv_cache.cache_write(cache, inside, rows[1], slots)
    torch.cuda.synchronize()
    assert torch.equal(cache.k, kept[0]) and torch.equal(both, kept[1])


def test_attention_outputs():
    cache = kv_cache.PagedCache.allocate(400, 2, 16, 64, dtype=torch.bfloat16)
    kv_cache.cache_write(cache, *torch.randn(2, 6400, 2, 64, device="cuda").bfloat16(),
                         torch.arange(6400, device="cuda"))
    table = torch.arange(400, device="cuda", dtype=torch.int32).view(2, 200)
    lengths = torch.tensor([3200, 77], device="cuda", dtype=torch.int32)
    buffer = torch.randn(2, 8, 64, device="cuda").bfloat16()
    q = buffer[:, :4]
    want = paged_attention(q, cache, table, lengths)
    paged_attention(q, cache, table, lengths, out=buffer[:, 4:])
    assert torch.equal(buffer[:, 4:], want)
    size = workspace_bytes(q, cache, 3200)
    assert size > 256
    kept = buffer.clone()
    for kw in (dict(out=buffer[:, 1:5]), dict(out=cache.v[0, :, :4].transpose(0, 0)),
               dict(workspace=cache.k.view(torch.uint8).flatten()[:size]),
               dict(out=buffer.flatten().as_strided((2, 4, 64), (64, 64, 1)))):
        with pytest.raises((RuntimeError, ValueError), match="overlap|out must"):
            paged_attention(q, cache, table, lengths, **kw)
    torch.cuda.synchronize()
    assert torch.equal(buffer, kept)
    paged_attention(q, cache, table, lengths, out=q)
    assert torch.equal(buffer[:, :4], want) and torch.equal(buffer[:, 4:], want)
