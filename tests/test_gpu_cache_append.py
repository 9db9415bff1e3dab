"""New tokens appended to the paged cache on the GPU.

The rotation is apply_rotary's arithmetic (its own tests hold it to 64 bits), and what
enters the cache is the FP32 rotation converted once: so the queries, and every byte of
the cache, are determined by apply_rotary on FP32 copies of the rows, torch's conversion
of its FP32 results and cache_write of them, bit for bit, and compared with them.  FP16
numbers may differ where the sum is within FP32's rounding of half way between two: the
hardware's fused multiply-add to FP16 rounds once where the two steps round twice.  One
test goes without any of that, by the 64-bit definition: a rotated FP32 value is off by
at most 2^-21 (|x1| + |x2|)."""
from __future__ import annotations

import pytest
import torch

from fireprot_amd import kv_cache, rotary
from fireprot_amd.cache_append import cache_append
from fireprot_amd.kv_cache import FP4, PagedCache, cache_slots, cache_write

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
FORMATS = [F32, BF16, F16, torch.float8_e4m3fn, torch.int8, FP4]


def raw(t):
    return t.view(torch.uint8)


def randn(shape, dtype, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda")
            * torch.exp(torch.randn((*shape[:-1], 1), generator=g, device="cuda"))).to(dtype)


def two_caches(*args, dtype):
    """Equal caches of random bytes."""
    one, two = (PagedCache.allocate(*args, dtype=dtype) for _ in range(2))
    g = torch.Generator("cuda").manual_seed(9)
    for a, b in zip(tensors(one), tensors(two)):
        raw(a).random_(0, 100, generator=g)
        raw(b).copy_(raw(a))
    return one, two


def tensors(cache):
    return [t for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]


def expect(cache, q, k, v, positions, f, slots, layout):
    """What a call does, by the operators it stands for, from FP32 rows: the cache
    written, the FP32 queries returned."""
    lead = positions.shape if positions.dim() == 2 else k.shape[:-2]
    positions = positions.expand(lead)
    kr = rotary.apply_rotary(k.float(), None, positions, f, layout=layout)
    cache_write(cache, kr.flatten(0, -3), v.float().flatten(0, -3), slots.flatten())
    if q is None:
        return None, kr
    return rotary.apply_rotary(q.float(), None, positions, f, layout=layout), kr


def same(got, exact, want):
    """FP32 values converted, or as near to them as the conversion."""
    if got.dtype != F16:
        return torch.equal(raw(got.contiguous()), raw(want.contiguous()))
    gap, least = ((t.double() - exact.double()).abs() for t in (got, want))
    return bool((gap <= least + 2.0 ** -23 * exact.double().abs()).all())


def check(got, expected, one, two, slots):
    """The queries, and two caches byte for byte."""
    q, k = expected
    if q is not None:
        assert same(got, q, q.to(got.dtype))
    a, b = tensors(one), tensors(two)
    if one.dtype == F16:
        page = one.page_size
        at, kept = slots.flatten(), (slots.flatten() >= 0) & (slots.flatten() < one.pages * page)
        at = at[kept]
        rows = (at // page, slice(None), at % page)
        assert same(one.k[rows], k.flatten(0, -3)[kept], two.k[rows])
        one.k[rows] = two.k[rows]
    for x, y in zip(a, b):
        assert torch.equal(raw(x), raw(y))


SIZES = [  # batch, tokens, q_heads, heads, head_dim, page, rotary_dim
    (1, 1, 1, 1, 32, 16, 32), (3, 37, 8, 2, 64, 32, 64), (2, 65, 5, 5, 128, 16, 96),
    (7, 1, 32, 8, 128, 64, 128), (2, 19, 6, 3, 256, 32, 256), (1, 130, 4, 1, 64, 16, 26),
    (5, 3, 3, 3, 32, 128, 2), (2, 21, 16, 1, 256, 16, 64)]


@pytest.mark.parametrize("row", [F32, BF16, F16])
@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_against_the_calls_it_stands_for(row, form, layout):
    for i, (batch, tokens, q_heads, heads, dim, page, rot) in enumerate(SIZES):
        print(f"append {row}->{form} {layout} {SIZES[i]}", flush=True)
        columns = -(-(tokens + 11) // page) + 1
        one, two = two_caches(batch * columns + 2, heads, page, dim, dtype=form)
        table = torch.randperm(batch * columns + 2, generator=torch.Generator().manual_seed(i))
        table = table[:batch * columns].view(batch, columns).int().cuda()
        f = rotary.rotary_frequencies(rot, scaling="by_parts", factor=4.0, original_length=64,
                                      device="cuda")
        q, k, v = (randn((batch, tokens, h, dim), row, 10 * i + j)
                   for j, h in enumerate((q_heads, heads, heads)))
        start = torch.arange(batch)[:, None] * 3 % 11
        positions = (start + torch.arange(tokens)).cuda()
        if tokens > 2:
            positions[-1, -2:] = torch.tensor([-1, -2 ** 40])
        if i % 2:
            positions = positions.clamp(min=-7).int()
        slots = cache_slots(table, positions, page)
        got = cache_append(one, q, k, v, positions, f, block_table=table, layout=layout)
        check(got, expect(two, q, k, v, positions, f, slots, layout), one, two, slots)
        # the slots given, and no queries
        one, two = two_caches(batch * columns + 2, heads, page, dim, dtype=form)
        assert cache_append(one, None, k, v, positions, f, slots=slots, layout=layout) is None
        check(None, expect(two, None, k, v, positions, f, slots, layout), one, two, slots)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rot", [10, 32, 64])
def test_by_definition(layout, rot):
    batch, tokens, dim, page = 2, 33, 64, 16
    f = rotary.rotary_frequencies(rot, device="cuda")
    cache = PagedCache.allocate(8, 2, page, dim, dtype=F32)
    table = torch.tensor([[5, 1, 7], [0, 6, 3]], dtype=torch.int32).cuda()
    q, k, v = (randn((batch, tokens, h, dim), F32, h + j) for j, h in enumerate((4, 2, 2)))
    positions = torch.arange(tokens).cuda()
    out = cache_append(cache, q, k, v, positions, f, block_table=table, layout=layout)
    angle = (positions.double()[:, None] * f.inv_freq)[None, :, None]
    one, two = ((slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half"
                else (slice(0, rot, 2), slice(1, rot, 2)))
    held = cache.k[table.long()].transpose(2, 3).flatten(1, 2)[:, :tokens]
    for got, x in ((out, q.double()), (held, k.double())):
        want, size = x.clone(), x.abs()
        a, b = x[..., one], x[..., two]
        want[..., one] = a * torch.cos(angle) - b * torch.sin(angle)
        want[..., two] = b * torch.cos(angle) + a * torch.sin(angle)
        size[..., one] = size[..., two] = a.abs() + b.abs()
        assert ((got.double() - want).abs() <= 2.0 ** -21 * size).all()
        assert torch.equal(got[..., rot:], x[..., rot:].float())
    assert torch.equal(cache.v[table.long()].transpose(2, 3).flatten(1, 2)[:, :tokens], v)


@pytest.mark.parametrize("row,form", [(BF16, BF16), (F32, torch.int8), (F16, FP4)])
@pytest.mark.parametrize("view", ["fused", "offset", "odd", "heads_first", "broadcast",
                                  "channel_stride"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_strides_and_alignment(row, form, view, layout):
    b, n, h, d = 3, 13, 4, 64
    if view == "fused":
        x = randn((b, n, 4 * h, d), row, 1)
        q, k, v = x[:, :, :2 * h], x[:, :, 2 * h:3 * h], x[:, :, 3 * h:]
    elif view == "offset":
        x = randn((3, b * n * h * d + 1), row, 2)
        q, k, v = (t[1:].view(b, n, h, d) for t in x)
    elif view == "odd":
        x = randn((b, n, h, 3 * d + 5), row, 3)
        q, k, v = x[..., 1:d + 1], x[..., d + 2:2 * d + 2], x[..., 2 * d + 5:]
    elif view == "heads_first":
        q, k, v = (randn((b, h, n, d), row, 4 + j).transpose(1, 2) for j in range(3))
    elif view == "broadcast":
        q, k = (randn((b, n, 1, d), row, 7 + j).expand(b, n, h, d) for j in range(2))
        v = randn((1, n, h, d), row, 9).expand(b, n, h, d)
    else:
        q, k, v = randn((b, n, h, 3 * d), row, 10).view(b, n, h, d, 3).unbind(-1)
    one, two = two_caches(7, h, 16, d, dtype=form)
    f = rotary.rotary_frequencies(d, device="cuda")
    positions = torch.randint(-1000, 1 << 20, (n,)).cuda()
    slots = torch.randperm(7 * 16, generator=torch.Generator().manual_seed(3))[:b * n]
    slots[5], slots[7] = -1, 7 * 16
    slots = slots.view(n, b).cuda().t()  # not contiguous
    got = cache_append(one, q, k, v, positions, f, slots=slots, layout=layout)
    want = expect(two, q.contiguous().clone(), k.contiguous().clone(), v.contiguous().clone(),
                  positions, f, slots, layout)
    check(got, want, one, two, slots)


def test_in_place_outputs_and_no_batch_axis():
    n, h, d = 9, 4, 128
    f = rotary.rotary_frequencies(d, device="cuda")
    x = randn((n, 3 * h, d), BF16, 1)
    one, two = two_caches(2, h, 16, d, dtype=BF16)
    slots, positions = torch.arange(3, 3 + n).cuda(), torch.arange(n).cuda()
    want = expect(two, x[:, :h], x[:, h:2 * h], x[:, 2 * h:], positions, f, slots, "half")
    out = torch.zeros(n, 2 * h, d, dtype=BF16, device="cuda")
    got = cache_append(one, x[:, :h], x[:, h:2 * h], x[:, 2 * h:], positions, f, slots=slots,
                       q_out=out[:, ::2])
    assert got.data_ptr() == out.data_ptr() and (out[:, 1::2] == 0).all()
    check(got, want, one, two, slots)
    turned, before = got.clone(), x[:, h:].clone()
    got = cache_append(one, x[:, :h], x[:, h:2 * h], x[:, 2 * h:], positions, f,
                       block_table=torch.tensor([[1]], dtype=torch.int32).cuda(), q_out=x[:, :h])
    assert torch.equal(x[:, :h], turned) and torch.equal(x[:, h:], before)
    assert torch.equal(one.k[1, :, :n], two.k[0, :, 3:3 + n])


def test_places_that_are_no_slots():
    """Past the table, on entries that name no page, in an empty table: not written."""
    one, two = two_caches(4, 2, 16, 32, dtype=torch.int8)
    f = rotary.rotary_frequencies(32, device="cuda")
    q, k, v = (randn((2, 6, 2, 32), F32, j) for j in range(3))
    positions = torch.tensor([[0, 15, 16, 31, 32, 2 ** 40], [47, 3, 48, -1, -2 ** 62, 40]]).cuda()
    table = torch.tensor([[2, -1, 0], [1, 5, 4]], dtype=torch.int32).cuda()
    slots = torch.tensor([[32, 47, -1, -1, 0, -1], [-1, 19, -1, -1, -1, -1]]).cuda()
    got = cache_append(one, q, k, v, positions, f, block_table=table)
    check(got, expect(two, q, k, v, positions, f, slots, "half"), one, two, slots)
    before = [raw(t).clone() for t in tensors(one)]
    got = cache_append(one, q, k, v, positions, f, block_table=table[:, :0])
    assert torch.equal(got, rotary.apply_rotary(q, None, positions, f))
    assert all(torch.equal(raw(t), b) for t, b in zip(tensors(one), before))
    # nothing to do
    none = cache_append(one, q[:, :0], k[:, :0], v[:, :0], positions[:, :0], f, block_table=table)
    assert none.shape == (2, 0, 2, 32)
    assert cache_append(one, None, k[:0], v[:0], positions[:0], f, block_table=table[:0]) is None


def test_many_tokens_and_large_offsets():
    """Groups of 16 tokens, and a cache of more than 2^31 elements."""
    page, dim = 4096, 32
    pages = 2 ** 31 // (page * dim) + 2
    cache = PagedCache.allocate(pages, 1, page, dim, dtype=torch.int8)
    n = 40_000
    f = rotary.rotary_frequencies(dim, device="cuda")
    k, v = randn((n, 1, dim), F16, 1), randn((n, 1, dim), F16, 2)
    slots = pages * page - 1 - torch.arange(n).cuda()
    cache_append(cache, None, k, v, torch.arange(n).cuda(), f, slots=slots)
    small = PagedCache.allocate(-(-n // page), 1, page, dim, dtype=torch.int8)
    at = torch.arange(n).cuda()
    expect(small, None, k, v, at, f, at, "half")
    for a, b in zip(kv_cache.cache_read(cache, slots), kv_cache.cache_read(small, at)):
        assert torch.equal(a, b)


def test_refusals():
    cache = PagedCache.allocate(2, 2, 16, 32, dtype=BF16)
    f = rotary.rotary_frequencies(32, device="cuda")
    q, k, v = (randn((3, 4, h, 32), BF16, h) for h in (4, 2, 2))
    good = dict(q=q, k=k, v=v, positions=torch.arange(4).cuda(), frequencies=f,
                block_table=torch.zeros(3, 1, dtype=torch.int32, device="cuda"), slots=None)
    bad = [dict(k=k[0]), dict(k=k[..., :16]), dict(v=v.float()), dict(v=v[:2]), dict(v=v.cpu()),
           dict(q=q.float()), dict(q=q[:2]), dict(q=q[..., :16]), dict(q=q.cpu()),
           dict(k=k.double()), dict(k=k.expand(2, 3, 4, 2, 32)),
           dict(positions=torch.arange(5).cuda()), dict(positions=torch.arange(4)),
           dict(positions=torch.arange(4.0).cuda()), dict(block_table=None),
           dict(slots=torch.zeros(3, 4, dtype=torch.int64, device="cuda")),
           dict(block_table=torch.zeros(3, 1, dtype=torch.int64, device="cuda")),
           dict(block_table=torch.zeros(2, 1, dtype=torch.int32, device="cuda")),
           dict(block_table=torch.zeros(3, 1, dtype=torch.int32)),
           dict(block_table=None, slots=torch.zeros(12, dtype=torch.int64, device="cuda")),
           dict(block_table=None, slots=torch.zeros(3, 4, dtype=torch.int32, device="cuda")),
           dict(frequencies=rotary.rotary_frequencies(64, device="cuda")),
           dict(frequencies=rotary.rotary_frequencies(32)), dict(layout="quarter"),
           dict(q_out=q[:, :1]), dict(q_out=q.float()), dict(q=None, q_out=q),
           dict(q_out=q[:, :, :1].expand(3, 4, 4, 32)),
           dict(k=k.clone().requires_grad_()), dict(q=q.clone().requires_grad_())]
    for change in bad:
        with pytest.raises(ValueError):
            cache_append(cache, **{**good, **change})
    x = randn((3, 4, 8, 32), BF16, 5)
    for change in (dict(q=x[:, :, :4], k=x[:, :, 4:6], v=x[:, :, 6:], q_out=x[:, :, 1:5]),
                   dict(k=cache.k.view(1, 16, 2, 2, 32).expand(3, 16, 2, 2, 32)[:, :4, 0])):
        with pytest.raises(RuntimeError, match="status 2"):
            cache_append(cache, **{**good, **change})
    with torch.no_grad():
        cache_append(cache, **{**good, "k": k.clone().requires_grad_()})


def test_on_another_stream_and_captured():
    """Replays follow the eager call, on a side stream too."""
    f = rotary.rotary_frequencies(64, device="cuda")
    one, two = two_caches(12, 2, 16, 64, dtype=FP4)
    table = torch.randperm(12, generator=torch.Generator().manual_seed(1)).view(3, 4).int().cuda()
    q, k, v = (torch.zeros(3, 1, h, 64, dtype=BF16, device="cuda") for h in (4, 2, 2))
    positions = torch.zeros(3, 1, dtype=torch.int32, device="cuda")

    def call(cache):
        return cache_append(cache, q, k, v, positions, f, block_table=table)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(one)
        call(two)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(one)
    g = torch.Generator("cuda").manual_seed(4)
    for rep in range(8):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, device="cuda", generator=g))
        positions.copy_(torch.tensor([[rep], [9 * rep], [63 - rep]]))
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want = call(two)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for a, b in zip(tensors(one), tensors(two)):
            assert torch.equal(raw(a), raw(b)), f"replay {rep}"
