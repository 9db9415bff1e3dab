"""Paths of cache_append and of the 4-bit cache that only large or odd calls take: several
tokens to a work-group, with a last one of fewer and ones that cross sequences; queries in
place where a neighbouring lane has the other channel of a pair; rows that are streamed; and
more work-groups than a launch has.  Compared byte for byte with the calls they stand for, as
test_gpu_cache_append.py has them, or with the same rows in small calls."""
from __future__ import annotations

import pytest
import torch

from fireprot_amd import rotary
from fireprot_amd.cache_append import cache_append
from fireprot_amd.kv_cache import FP4, PagedCache, cache_read, cache_slots, cache_write
from tests.test_gpu_cache_append import check, expect, randn, raw, tensors, two_caches

pytestmark = pytest.mark.gpu

F32, BF16, F16, INT8 = torch.float32, torch.bfloat16, torch.float16, torch.int8
KINDS = [(BF16, BF16), (F32, INT8), (F16, FP4)]


def offset_rows(shape, dtype, seed, offset):
    """Rows that begin `offset` elements past an aligned address."""
    x = randn((torch.Size(shape).numel() // shape[-1], shape[-1]), dtype, seed).flatten()
    held = torch.zeros(x.numel() + 8, dtype=dtype, device="cuda")
    held[offset:offset + x.numel()] = x
    return held[offset:offset + x.numel()].view(shape)


# 4, 4, 4, 16, 8 and 2 tokens to a work-group
SIZES = [(3, 2731, 2, 1, 32, 32), (3, 2731, 2, 1, 64, 16), (3, 2731, 2, 1, 64, 26),
         (5, 6555, 2, 1, 32, 18), (5, 3301, 1, 1, 64, 32), (3, 2731, 4, 3, 128, 96)]


@pytest.mark.parametrize("row,form", KINDS)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("batch,tokens,q_heads,heads,dim,rot", SIZES)
def test_several_tokens_to_a_work_group(row, form, layout, offset, batch, tokens, q_heads, heads,
                                        dim, rot):
    print(f"tokens {row}->{form} {layout} +{offset} {batch, tokens, q_heads, heads, dim, rot}",
          flush=True)
    page = 64
    columns = -(-(tokens + 40) // page)
    one, two = two_caches(batch * columns, heads, page, dim, dtype=form)
    table = torch.randperm(batch * columns, generator=torch.Generator().manual_seed(dim))
    table = table.view(batch, columns).int().cuda()
    f = rotary.rotary_frequencies(rot, device="cuda")
    q, k, v = (offset_rows((batch, tokens, h, dim), row, j, offset)
               for j, h in enumerate((q_heads, heads, heads)))
    positions = (torch.arange(batch)[:, None] * 17 + torch.arange(tokens)).cuda()
    positions[-1, -1] = positions[0, 5] = -3
    slots = cache_slots(table, positions, page)
    before = q.clone()
    want = expect(two, q, k, v, positions, f, slots, layout)
    got = cache_append(one, q, k, v, positions, f, block_table=table, layout=layout)
    assert torch.equal(q, before)
    check(got, want, one, two, slots)
    # the queries in place
    one = two_caches(batch * columns, heads, page, dim, dtype=form)[0]
    assert cache_append(one, q, k, v, positions, f, slots=slots, layout=layout,
                        q_out=q).data_ptr() == q.data_ptr()
    assert torch.equal(raw(q.contiguous()), raw(got))
    check(None, (None, want[1]), one, two, slots)


@pytest.mark.parametrize("row", [F32, BF16, F16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("dim,rot", [(32, 16), (64, 32), (64, 26), (128, 64), (256, 128),
                                     (256, 250), (256, 256)])
def test_queries_in_place(row, layout, offset, dim, rot):
    """Rows of a fused product, the head turned in part: what a lane writes another reads."""
    n, h = 301, 6
    f = rotary.rotary_frequencies(rot, device="cuda")
    x = offset_rows((n, 3 * h, dim), row, dim, offset)
    one, two = two_caches(32, h, 16, dim, dtype=row)
    slots = torch.randperm(512, generator=torch.Generator().manual_seed(1))[:n].cuda()
    positions = torch.arange(7, 7 + n).cuda()
    q, k, v = x[:, :h], x[:, h:2 * h], x[:, 2 * h:]
    want = cache_append(two, q, k, v, positions, f, slots=slots, layout=layout)
    exact = rotary.apply_rotary(q.float(), None, positions, f, layout=layout)
    rest = x[:, h:].clone()
    for _ in range(3):
        y = offset_rows((n, 3 * h, dim), row, dim, offset)
        got = cache_append(one, y[:, :h], y[:, h:2 * h], y[:, 2 * h:], positions, f, slots=slots,
                           layout=layout, q_out=y[:, :h])
        assert got.data_ptr() == y.data_ptr()
        assert torch.equal(raw(got.contiguous()), raw(want))
        assert torch.equal(raw(y[:, h:].contiguous()), raw(rest))
        for a, b in zip(tensors(one), tensors(two)):
            assert torch.equal(raw(a), raw(b))
    gap = (want.double() - exact.double()).abs()
    # one rounding to the type; FP16's may come from the sum before its rounding to 32 bits
    assert (gap <= exact.double().abs() * (torch.finfo(row).eps / 2 + 2.0 ** -23)
            + torch.finfo(row).smallest_normal * torch.finfo(row).eps).all()


@pytest.mark.parametrize("row,form,dim,layout,rot", [
    (BF16, FP4, 128, "half", 128), (F16, INT8, 64, "interleaved", 26), (F32, F32, 256, "half", 256),
    (BF16, torch.float8_e4m3fn, 32, "half", 32), (F32, FP4, 64, "interleaved", 64)])
def test_streamed_rows(row, form, dim, layout, rot):
    """More than 64 MB of rows in one call, and the same in calls of 1000 tokens."""
    q_heads, heads, page = 8, 4, 64
    n = (65 << 20) // ((q_heads + 2 * heads) * dim * row.itemsize) + 3
    print(f"streamed {row}->{form} {dim} {n} tokens", flush=True)
    one, two = two_caches(-(-n // page), heads, page, dim, dtype=form)
    f = rotary.rotary_frequencies(rot, device="cuda")
    x = randn((n, q_heads + 2 * heads, dim), row, dim)
    q, k, v = x.split([q_heads, heads, heads], 1)
    positions = torch.arange(n).cuda()
    slots = torch.randperm(one.pages * page, generator=torch.Generator().manual_seed(2))[:n].cuda()
    got = cache_append(one, q, k, v, positions, f, slots=slots, layout=layout)
    for i in range(0, n, 1000):
        part = slice(i, i + 1000)
        want = cache_append(two, q[part], k[part], v[part], positions[part], f, slots=slots[part],
                            layout=layout)
        assert torch.equal(raw(got[part]), raw(want)), i
    for a, b in zip(tensors(one), tensors(two)):
        assert torch.equal(raw(a), raw(b))


def test_more_tokens_than_a_launch_has_work_groups():
    """2^22 + 9 sequences of one token, of which a few, first and last, have a place."""
    batch, heads, dim, page = (1 << 22) + 9, 32, 64, 16
    one, two = two_caches(4, heads, page, dim, dtype=BF16)
    k, v = (randn((1, 1, heads, dim), F16, j).expand(batch, 1, heads, dim) for j in (1, 2))
    f = rotary.rotary_frequencies(dim, device="cuda")
    positions = torch.arange(batch, dtype=torch.int32, device="cuda")[:, None]
    at = torch.tensor([0, 1, 77, (1 << 22) - 1, 1 << 22, (1 << 22) + 1, batch - 1]).cuda()
    slots = torch.full((batch, 1), -1, device="cuda")
    slots[at, 0] = torch.tensor([3, 60, 17, 33, 0, 50, 16]).cuda()
    cache_append(one, None, k, v, positions, f, slots=slots)
    expect(two, None, k[at].contiguous(), v[at].contiguous(), positions[at].contiguous(), f,
           slots[at], "half")
    for a, b in zip(tensors(one), tensors(two)):
        assert torch.equal(raw(a), raw(b))


@pytest.mark.parametrize("dim,row", [(128, BF16), (256, F32), (32, F16)])
def test_streamed_rows_in_4_bits(dim, row):
    """Written and read back in one call of more than 64 MB, and in calls of 1000 tokens."""
    heads, page = 8, 64
    n = (33 << 20) // (heads * dim // 2) + 5
    print(f"4 bits streamed {row} {dim} {n} tokens", flush=True)
    one, two = two_caches(-(-n // page), heads, page, dim, dtype=FP4)
    k, v = (randn((n, heads, dim), row, j) for j in range(2))
    slots = torch.randperm(one.pages * page, generator=torch.Generator().manual_seed(3))[:n].cuda()
    slots[11], slots[n - 2] = -1, one.pages * page + 5
    cache_write(one, k, v, slots)
    whole = cache_read(one, slots, dtype=row)
    for i in range(0, n, 1000):
        part = slice(i, i + 1000)
        cache_write(two, k[part], v[part], slots[part])
        for a, b in zip(cache_read(two, slots[part], dtype=row), whole):
            assert torch.equal(raw(a), raw(b[part])), i
    for a, b in zip(tensors(one), tensors(two)):
        assert torch.equal(raw(a), raw(b))
    assert (whole[0][11] == 0).all() and torch.isnan(whole[1][n - 2]).all()
