"""The paged cache on the GPU against its definition.

A plain cache holds its rows rounded once: equal bit for bit to torch's own
conversion.  The 8-bit codes and scales are determined bit for bit by the
definition (a division by a power of two is exact; the INT8 scale, its
reciprocal and each product are single 32-bit operations, the same here and on
the CPU), and so is what is read back: one 32-bit product, one rounding.
"""
from __future__ import annotations

import pytest
import torch

from fireprot_amd import kv_cache
from fireprot_amd.kv_cache import PagedCache, cache_read, cache_write

pytestmark = pytest.mark.gpu

ROWS = [torch.float32, torch.bfloat16, torch.float16]
CODED = [torch.float8_e4m3fn, torch.int8]


def raw(t):
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def quantised(x, dtype):
    """Codes (as raw bytes) and scales of the rows of x, on the CPU."""
    x = x.cpu().float()
    top = x.abs().amax(-1)
    finite = torch.isfinite(x).all(-1)
    top = torch.where(finite, top, torch.zeros_like(top))
    live = top >= 2.0 ** -100
    safe = torch.where(live, top, torch.ones_like(top))
    if dtype == torch.float8_e4m3fn:
        e = torch.ceil(torch.log2(safe.double() / 448.0))
        e = torch.where(safe.double() > 448.0 * torch.exp2(e), e + 1, e)
        e = torch.where(safe.double() <= 448.0 * torch.exp2(e - 1), e - 1, e)
        scale = torch.exp2(e).float()
        y = torch.where((live & finite)[..., None], x.double() / scale[..., None].double(), 0.0)
        codes = y.float().to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        scale = safe * torch.tensor(1.0 / 127.0)
        y = torch.where((live & finite)[..., None], x * (1.0 / scale)[..., None], 0.0)
        codes = torch.round(y).to(torch.int8).view(torch.uint8)
    scale = torch.where(live, scale, torch.zeros_like(scale))
    return codes, torch.where(finite, scale, torch.full_like(scale, float("nan")))


def rows(tokens, heads, dim, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, heads, dim, generator=g)
    return (x * torch.exp(torch.randn(tokens, heads, 1, generator=g))).to(dtype).cuda()


def random_cache(pages, heads, page, dim, dtype, seed=9):
    """A cache whose every byte is random, to see what a write leaves alone."""
    cache = PagedCache.allocate(pages, heads, page, dim, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(seed)
    for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        if t is not None:
            raw(t).random_(0, 100, generator=g)
    return cache


def clone(cache):
    return [None if t is None else raw(t).clone()
            for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]


@pytest.mark.parametrize("row", ROWS)
@pytest.mark.parametrize("dtype", ROWS + CODED)
@pytest.mark.parametrize("tokens,heads,page,dim", [(1, 1, 16, 32), (37, 3, 16, 64),
                                                   (130, 8, 64, 128), (67, 5, 32, 256)])
def test_write_and_read_back(row, dtype, tokens, heads, page, dim):
    print(f"cache {row}->{dtype} {tokens, heads, page, dim}", flush=True)
    pages = tokens // page + 4
    cache = random_cache(pages, heads, page, dim, dtype)
    k, v = rows(tokens, heads, dim, row), rows(tokens, heads, dim, row, 2)
    g = torch.Generator().manual_seed(4)
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    if tokens > 4:
        slots[1], slots[2], slots[3] = -1, -2 ** 62, pages * page  # no token, no token, outside
    before = clone(cache)
    cache_write(cache, k, v, slots.cuda())
    torch.cuda.synchronize()
    after = clone(cache)
    kept = (slots >= 0) & (slots < pages * page)
    p, o = slots[kept] // page, slots[kept] % page
    for w, x in ((0, k), (1, v)):
        want, want_scale = before[w].cpu(), before[w + 2]
        if dtype in CODED:
            codes, scale = quantised(x[kept.cuda()], dtype)
            want[p, :, o] = codes
            want_scale = want_scale.cpu()
            want_scale[p, :, o] = raw(scale)
            assert torch.equal(after[w + 2].cpu(), want_scale)
        else:
            want[p, :, o] = raw(x[kept.cuda()].to(dtype).cpu())
        assert torch.equal(after[w].cpu(), want), "written rows and nothing else"
    # back in each row type, in another order, some slots twice
    order = torch.randint(0, tokens, (2 * tokens,), generator=g)
    back = slots[order]
    for out_type in ROWS:
        got = cache_read(cache, back.cuda(), dtype=out_type)
        for w, y in enumerate(got):
            data, scale = (cache.k, cache.k_scale) if w == 0 else (cache.v, cache.v_scale)
            at = back.clamp(0, pages * page - 1)
            held = raw(data).cpu()[at // page, :, at % page].view(data.dtype).float()
            if scale is not None:
                held = held * scale.cpu()[at // page, :, at % page][..., None]
            held[back < 0] = 0.0
            held[back >= pages * page] = float("nan")
            want = held.to(out_type)
            assert torch.equal(torch.isnan(y.cpu()), torch.isnan(want))
            assert torch.equal(torch.nan_to_num(y.cpu()), torch.nan_to_num(want))


@pytest.mark.parametrize("dtype", CODED)
def test_rows_at_the_edges_of_the_codes(dtype):
    dim = 32
    x = torch.zeros(14, 1, dim)
    x[0] = 0.0
    x[1, 0, 3] = 448.0
    x[2, 0, 3] = 448.0001
    x[3, 0, 3] = -447.9999
    x[4] = torch.linspace(-1, 1, dim)
    x[5, 0, 0] = 2.0 ** -100
    x[6, 0, 0] = 2.0 ** -100 * (1 - 2 ** -24)
    x[7, 0, 1] = 3.0e38
    x[8, 0, 5], x[8, 0, 6] = float("inf"), 1.0
    x[9, 0, 31] = float("nan")
    x[10, 0, 0], x[10, 0, 1], x[10, 0, 2] = 256.0, 17.0, 0.0146484375  # ties, a subnormal code
    x[11] = -0.0
    x[12, 0, 0], x[12, 0, 1], x[12, 0, 2] = 127.0, 0.5, 1.5
    x[13, 0, 0] = 2.0 ** -149
    cache = PagedCache.allocate(1, 1, 16, dim, dtype=dtype)
    slots = torch.arange(14).cuda()
    cache_write(cache, x.cuda(), -x.cuda(), slots)
    for data, scale, source in ((cache.k, cache.k_scale, x), (cache.v, cache.v_scale, -x)):
        codes, want = quantised(source, dtype)
        got = scale[0, 0, :14, None].cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
        assert torch.equal(data.view(torch.uint8)[0, 0, :14].cpu(), codes[:, 0])
    k, _ = cache_read(cache, slots)
    assert torch.isnan(k[8:10]).all() and (k[6] == 0).all() and (k[0] == 0).all()
    # a code is off by half a step: 2^-4 of the value (or of the smallest
    # normal code), half a unit of the scale
    fine = [1, 2, 3, 4, 5, 7, 10, 12]
    s = cache.k_scale[0, 0, fine, None, None].cpu().double()
    step = (2.0 ** -4 * x[fine].double().abs().clamp(min=0) + s * 2.0 ** -10
            if dtype == torch.float8_e4m3fn else s * 0.5 * (1 + 2.0 ** -16))
    assert ((k[fine].cpu().double() - x[fine].double()).abs() <= step).all()


@pytest.mark.parametrize("row", ROWS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("view", ["fused", "offset", "odd_stride", "broadcast", "channel_stride"])
def test_strided_rows(row, dtype, view):
    t, h, d = 21, 4, 64
    if view == "fused":
        x = rows(t, 3 * h, d, row)
        k, v = x[:, h:2 * h], x[:, 2 * h:]
    elif view == "offset":
        k = rows(t, h, d, row).reshape(-1)
        k = torch.cat([k[:1], k])[1:].view(t, h, d)
        v = k
    elif view == "odd_stride":
        x = rows(t, h, 2 * d + 3, row)
        k, v = x[..., 1:d + 1], x[..., d + 2:2 * d + 2]
    elif view == "broadcast":
        k = rows(t, 1, d, row).expand(t, h, d)
        v = rows(1, h, d, row).expand(t, h, d)
    else:
        x = rows(t, h, 2 * d, row).view(t, h, d, 2)
        k, v = x[..., 0], x[..., 1]
    slots = torch.randperm(48, generator=torch.Generator().manual_seed(2))[:t].cuda()
    a = PagedCache.allocate(3, h, 16, d, dtype=dtype)
    b = PagedCache.allocate(3, h, 16, d, dtype=dtype)
    cache_write(a, k, v, slots)
    cache_write(b, k.contiguous().clone(), v.contiguous().clone(), slots)
    for one, two in zip(clone(a), clone(b)):
        assert one is None or torch.equal(one, two)
    wide = torch.full((t, h, 2 * d + 2), 7.0, dtype=row, device="cuda")
    cache_read(a, slots, k_out=wide[..., 1:d + 1], v_out=wide[..., d + 2:])
    want = cache_read(b, slots, dtype=row)
    assert torch.equal(wide[..., 1:d + 1], want[0]) and torch.equal(wide[..., d + 2:], want[1])
    assert (wide[..., 0] == 7).all() and (wide[..., d + 1] == 7).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8])
def test_offsets_past_32_bits(dtype):
    page, dim = 4096, 256
    pages = 2 ** 31 // (page * dim) + 3  # more than 2^31 elements
    cache = PagedCache.allocate(pages, 1, page, dim, dtype=dtype)
    slots = torch.tensor([0, pages * page - 1, 2 ** 31 // dim, 2 ** 31 // dim - 1]).cuda()
    k, v = rows(4, 1, dim, torch.float32), rows(4, 1, dim, torch.float32, 3)
    cache_write(cache, k, v, slots)
    small = PagedCache.allocate(1, 1, 16, dim, dtype=dtype)
    cache_write(small, k, v, torch.arange(4).cuda())
    got, want = cache_read(cache, slots), cache_read(small, torch.arange(4).cuda())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert int((raw(cache.k) != 0).any(-1).sum()) == 4


def test_source_offsets_past_32_bits():
    pitch = 2 ** 31 + 32
    buffer = torch.empty(pitch + 64, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(buffer, (2, 1, 32), (pitch, 32, 1))
    x.copy_(rows(2, 1, 32, torch.bfloat16))
    cache = PagedCache.allocate(1, 1, 16, 32, dtype=torch.bfloat16)
    slots = torch.tensor([3, 5]).cuda()
    cache_write(cache, x, x, slots)
    assert torch.equal(cache.k[0, 0, [3, 5]], x[:, 0])
    saved = x.clone()
    x.zero_()
    cache_read(cache, slots, k_out=x, v_out=torch.empty(2, 1, 32, dtype=torch.bfloat16,
                                                        device="cuda"))
    assert torch.equal(x, saved)


def test_more_rows_than_one_grid():
    # 2^27 rows of 32 channels and some: more groups of rows than the grid's
    # limit, so the kernels walk on
    tokens, heads, dim = 2 ** 23 + 5, 16, 32
    cache = PagedCache.allocate(tokens // 4096 + 1, heads, 4096, dim, dtype=torch.int8)
    x = torch.randint(-127, 128, (tokens, 1, dim), device="cuda", dtype=torch.int8,
                      generator=torch.Generator(device="cuda").manual_seed(1)).to(torch.bfloat16)
    x[..., 0] = 127  # so each row's scale is that of 127
    x = x.expand(tokens, heads, dim)
    slots = torch.arange(tokens, device="cuda")
    cache_write(cache, x, x, slots)
    k, v = cache_read(cache, slots, dtype=torch.bfloat16)
    assert torch.equal(k, x) and torch.equal(v, x)


def test_empty_calls():
    cache = PagedCache.allocate(1, 2, 16, 32, dtype=torch.bfloat16)
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    x = torch.zeros(0, 2, 32, device="cuda")
    cache_write(cache, x, x, none)
    k, v = cache_read(cache, none)
    assert k.shape == v.shape == (0, 2, 32) and k.dtype == torch.bfloat16


def test_refusals_on_the_device():
    cache = PagedCache.allocate(2, 3, 16, 64, dtype=torch.float8_e4m3fn)
    x, slots = rows(4, 3, 64, torch.bfloat16), torch.arange(4).cuda()
    grad = x.clone().requires_grad_()
    for bad in (lambda: cache_write(cache, x, x.half(), slots),
                lambda: cache_write(cache, x[:3], x, slots),
                lambda: cache_write(cache, x[..., :32], x, slots),
                lambda: cache_write(cache, x.double(), x.double(), slots),
                lambda: cache_write(cache, x, x, slots.int()),
                lambda: cache_write(cache, x, x, slots.cpu()),
                lambda: cache_write(cache, x.cpu(), x.cpu(), slots),
                lambda: cache_write(cache, grad, x, slots),
                lambda: cache_read(cache, slots, dtype=torch.float64),
                lambda: cache_read(cache, slots, dtype=torch.float32, k_out=x),
                lambda: cache_read(cache, slots, k_out=x[:3]),
                lambda: cache_read(cache, slots, k_out=x[:1].expand_as(x)),
                lambda: cache_read(cache, slots[None])):
        with pytest.raises(ValueError):
            bad()
    assert cache_read(cache, slots)[0].dtype == torch.float32


def test_other_stream_and_graph():
    cache = PagedCache.allocate(4, 2, 16, 64, dtype=torch.float8_e4m3fn)
    other = PagedCache.allocate(4, 2, 16, 64, dtype=torch.float8_e4m3fn)
    x, slots = rows(9, 2, 64, torch.bfloat16), torch.arange(9).cuda()
    out = [torch.empty_like(x) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache_write(cache, x, -x, slots)
        cache_read(cache, slots, k_out=out[0], v_out=out[1])
    torch.cuda.current_stream().wait_stream(side)
    cache_write(other, x, -x, slots)
    want = cache_read(other, slots, dtype=torch.bfloat16)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache_write(cache, x, -x, slots)
        cache_read(cache, slots, k_out=out[0], v_out=out[1])
    for rep in range(4):
        x.copy_(rows(9, 2, 64, torch.bfloat16, 30 + rep))
        slots.copy_(torch.randperm(64, generator=torch.Generator().manual_seed(rep))[:9])
        graph.replay()
        torch.cuda.synchronize()
        cache_write(other, x, -x, slots)
        want = cache_read(other, slots, dtype=torch.bfloat16)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    for one, two in zip(clone(cache), clone(other)):
        assert torch.equal(one, two), "every replay wrote what the eager calls did"


def test_slots_of_positions_on_the_device():
    table = torch.tensor([[2, 0], [1, 3]], dtype=torch.int32).cuda()
    positions = torch.tensor([[0, 17, -1], [31, 32, 5]]).cuda()
    top = torch.iinfo(torch.int64).max
    assert kv_cache.cache_slots(table, positions, 16).tolist() == [[32, 1, -1], [63, top, 21]]


def test_outputs_of_a_read_share_no_memory():
    cache = PagedCache(*(torch.zeros(2, 1, 16, 32, device="cuda", dtype=torch.float16)
                         for _ in range(2)))
    x = torch.empty(3, 1, 32, device="cuda", dtype=torch.float16)
    slots = torch.arange(3, device="cuda")
    with pytest.raises(ValueError):
        cache_read(cache, slots, k_out=x, v_out=x)
    with pytest.raises(ValueError):
        cache_read(cache, slots, k_out=x, v_out=x.view(3, 1, 32))
    pair = torch.empty(3, 2, 32, device="cuda", dtype=torch.float16)
    k, v = cache_read(cache, slots, k_out=pair[:, :1], v_out=pair[:, 1:])
    assert (pair == 0).all() and k.data_ptr() != v.data_ptr()
