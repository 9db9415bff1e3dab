"""Bounds of pages, the selection by them and the attention to what is selected, on the
GPU.

Bounds are determined exactly: the least and greatest of the FP32 values that cache_read
gives, rounded outward to BF16 for coded caches.  A score is an FP64 sum rounded to FP32:
the reference sums in FP64 in another order, off by at most 2 D 2^-53 of the sum of
magnitudes, so that the FP32 numbers agree but for one sum in some 10^7, and the order of
the pages with them.  The attention's tolerance is that of whole sequences
(test_gpu_paged_attention.py), over the selected keys."""
from __future__ import annotations

import pytest
import torch

from fireprot_amd import kv_cache, rotary
from fireprot_amd.cache_append import cache_append
from fireprot_amd.kv_cache import FP4, PagedCache, cache_write
from fireprot_amd.page_selection import (PageBounds, bounds_dtype, select_pages,
                                         select_workspace_bytes, update_page_bounds)
from fireprot_amd.paged_attention import paged_attention

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
FP8, INT8 = torch.float8_e4m3fn, torch.int8
FORMATS = [F32, BF16, F16, FP8, INT8, FP4]


def raw(t):
    return t.view(torch.uint8)


def same(a, b):
    """Equal numbers, zeros of either sign among them, and NaN in the same places."""
    return (torch.equal(torch.isnan(a), torch.isnan(b))
            and torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float())))


def outward(x, kind, upper):
    """FP32 values as the nearest number of a type that is not inside them."""
    y = x.to(kind)
    if kind == BF16:
        wrong = y.float() < x if upper else y.float() > x
        bits = y.view(torch.int16)
        bits = torch.where(wrong, bits + torch.where((x > 0) == upper, 1, -1).to(torch.int16), bits)
        y = bits.view(BF16)
    return y


def filled(form, heads, page, dim, lengths, seed=1, spare=3):
    """(cache of rubbish where no sequence has a token, table, lengths)."""
    g = torch.Generator().manual_seed(seed)
    columns = max(1, -(-max([0, *lengths]) // page)) + 1
    pages = len(lengths) * columns + spare
    cache = PagedCache.allocate(pages, heads, page, dim, dtype=form)
    for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        if t is not None:
            raw(t).fill_(255)
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(lengths), columns), -9, dtype=torch.int32)
    slots, at = [], 0
    for b, n in enumerate(lengths):
        held = -(-n // page)
        table[b, :held] = order[at:at + held]
        at += held
        j = torch.arange(n)
        slots.append(table[b, j // page].long() * page + j % page)
    slots = torch.cat(slots)
    kv = torch.randn(2, len(slots), heads, dim, generator=g)
    kv *= torch.exp(0.4 * torch.randn(2, len(slots), heads, 1, generator=g))
    kv = kv.to(form if form in (F32, BF16, F16) else F32).cuda()
    cache_write(cache, kv[0], kv[1], slots.cuda())
    return cache, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()


def page_rows(cache, page, rows):
    """Keys and values of a page's first slots as cache_read has them, [rows, heads, d]."""
    slots = page * cache.page_size + torch.arange(rows, device="cuda")
    return kv_cache.cache_read(cache, slots, dtype=F32)


def expected_bounds(cache, table, lengths, new, values):
    """values with the bounds of the newest tokens' pages brought up to date."""
    values, page = values.clone(), cache.page_size
    for b, n in enumerate(lengths.tolist()):
        for i in range(max(0, n - new) // page, -(-n // page)):
            k, _ = page_rows(cache, int(table[b, i]), min(page, n - i * page))
            values[table[b, i], :, 0] = outward(k.amin(0), values.dtype, False)
            values[table[b, i], :, 1] = outward(k.amax(0), values.dtype, True)
    return values


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("heads,page,dim", [(2, 16, 32), (3, 64, 64), (1, 32, 128), (2, 128, 256),
                                            (5, 4096, 32)])
def test_bounds(form, heads, page, dim):
    print(f"bounds {form} {heads, page, dim}", flush=True)
    lengths = [0, 1, page - 1, page, page + 1, 3 * page + 7]
    cache, table, n = filled(form, heads, page, dim, lengths)
    bounds = PageBounds.allocate(cache)
    assert bounds.values.dtype == bounds_dtype(form)
    for new in (1, 5, page + 2, 1 << 40):
        bounds.values.copy_(torch.randn(bounds.values.shape))
        want = expected_bounds(cache, table, n, new, bounds.values)
        update_page_bounds(bounds, cache, table, n, new=new)
        assert same(bounds.values, want), new


def test_bounds_hold_for_scales_of_any_kind():
    """Scales that no BF16 holds: the bounds are not inside the values."""
    cache, table, n = filled(FP8, 2, 16, 64, [100])
    cache.k_scale.copy_(torch.rand(cache.k_scale.shape) + 0.01)
    cache.k.view(torch.uint8).random_(0, 127)
    bounds = PageBounds.allocate(cache)
    update_page_bounds(bounds, cache, table, n, new=100)
    for i in range(7):
        k, _ = page_rows(cache, int(table[0, i]), min(16, 100 - 16 * i))
        edge = bounds.values[table[0, i]].float()
        assert (edge[:, 0] <= k.amin(0)).all() and (edge[:, 1] >= k.amax(0)).all()
        assert (edge[:, 1] <= k.amax(0).abs() * (1 + 2.0 ** -7) + 1e-30).all()


def test_what_gets_no_bounds():
    cache, table, n = filled(F32, 2, 16, 32, [40, 40, 40])
    cache.k[table[0, 1].long(), 1, 3, 5] = float("nan")
    cache.k[table[0, 2].long(), 0, 2, 7] = float("inf")
    bounds = PageBounds.allocate(cache)
    bounds.values.fill_(7.0)
    want = expected_bounds(cache, table[:1], n[:1], 40, bounds.values)
    n[1] = -1
    table[2, 0], table[2, 1], table[2, 2] = -1, cache.pages, 2 ** 31 - 1
    update_page_bounds(bounds, cache, table, n, new=40)
    assert same(bounds.values, want)
    assert torch.isnan(want[table[0, 1], 1, :, 5]).all() and torch.isnan(want).sum() == 2
    n[1] = 33
    update_page_bounds(bounds, cache, table, n, new=40, max_length=32)  # all are longer
    assert same(bounds.values, want)


def test_bounds_of_more_pages_than_a_launch_has_work_groups():
    """2048 sequences, 64 heads, up to 33 pages each: 4.3 million (sequence, head, page)."""
    cache = PagedCache.allocate(40, 64, 16, 32, dtype=F16)
    cache.k.normal_(generator=torch.Generator("cuda").manual_seed(2))
    lengths = torch.zeros(2048, dtype=torch.int32)
    table = torch.full((2048, 33), -1, dtype=torch.int32)
    lengths[0], lengths[1023], lengths[2047] = 5, 300, 17
    table[0, 0] = 7
    table[1023, :19] = torch.arange(10, 29)
    table[2047, :2] = torch.tensor([31, 3])
    table, lengths = table.cuda(), lengths.cuda()
    bounds = PageBounds.allocate(cache)
    want = expected_bounds(cache, table, lengths, 1 << 20, bounds.values)
    update_page_bounds(bounds, cache, table, lengths, new=528)
    assert same(bounds.values, want)


# ---------------------------------------------------------------- selection

def expected_index(q, values, table, lengths, page, count, sinks, recent, max_length):
    """(index, lengths) by the definition, on the CPU."""
    q, values, table = q.cpu().double(), values.cpu().double(), table.cpu().long()
    pages, heads = values.shape[:2]
    index = torch.full((len(q), heads, count), -1, dtype=torch.int32)
    kept = torch.zeros(len(q), dtype=torch.int32)
    for b, n in enumerate(lengths.tolist()):
        if not 0 <= n <= max_length:
            kept[b] = -1
            continue
        total = -(-n // page)
        m = min(total, count)
        kept[b] = n - (total - m) * page
        held = table[b, :total]
        inside = (held >= 0) & (held < pages)
        edge = values[held.clamp(0, pages - 1)]
        for h in range(heads):
            x = q[b].unflatten(0, (heads, -1))[h]
            lo, hi = edge[:, h, 0], edge[:, h, 1]
            score = (x.clamp(min=0) @ hi.T + x.clamp(max=0) @ lo.T).amax(0).float()
            # NaN above all, the lowest place first
            order = torch.where(torch.isnan(score) | ~inside, float("inf"), score)
            sure = torch.isnan(score) | ~inside
            forced = torch.zeros(total, dtype=torch.bool)
            forced[:sinks], forced[max(0, total - recent):] = True, True
            rank = sorted(range(total), key=lambda i: (not forced[i], not sure[i], -order[i].item(),
                                                       i))
            index[b, h, :m] = torch.tensor(sorted(rank[:m]), dtype=torch.int32)
    return index, kept


def check_selection(got, want, table):
    index, kept = want
    assert torch.equal(got.lengths.cpu(), kept)
    assert torch.equal(got.index.cpu(), index)
    pages = table.cpu().gather(1, index.flatten(1).clamp(min=0).long()).view(index.shape)
    assert torch.equal(got.table.cpu(), torch.where(index < 0, -1, pages))


def random_bounds(pages, heads, dim, kind, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(pages, heads, 2, dim, generator=g, device="cuda")
    return x.sort(dim=2)[0].to(kind)


@pytest.mark.parametrize("q_type", [F32, BF16, F16])
@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("q_heads,heads,dim,page", [
    (1, 1, 32, 16), (8, 2, 64, 32), (15, 3, 128, 64), (16, 1, 256, 16), (17, 1, 128, 4096),
    (80, 2, 64, 16)])
def test_selection(q_type, kind, q_heads, heads, dim, page):
    print(f"select {q_type} {kind} {q_heads, heads, dim, page}", flush=True)
    held = [0, 1, 2, 7, 8, 9, 15, 16, 17, 63, 64, 65, 130, 300]
    g = torch.Generator().manual_seed(dim)
    lengths = torch.tensor([max(0, p * page - int(torch.randint(0, page, (1,), generator=g)))
                            for p in held], dtype=torch.int32)
    pages = sum(held) + 5
    bounds = PageBounds(random_bounds(pages, heads, dim, kind, 3), page)
    table = torch.full((len(held), 301), -3, dtype=torch.int32)
    order, at = torch.randperm(pages, generator=g), 0
    for b, p in enumerate(held):
        table[b, :p] = order[at:at + p]
        at += p
    table = table.cuda()
    q = torch.randn(len(held), q_heads, dim, generator=g).to(q_type).cuda()
    for count, sinks, recent in ((1, 0, 1), (8, 1, 2), (16, 0, 1), (7, 3, 4), (64, 2, 1),
                                 (301, 1, 1), (1000, 0, 5)):
        got = select_pages(q, bounds, table, lengths.cuda(), count, sinks=sinks, recent=recent)
        check_selection(got, expected_index(q, bounds.values, table, lengths, page, count, sinks,
                                            recent, 301 * page), table)
        again = select_pages(q, bounds, table, lengths.cuda(), count, sinks=sinks, recent=recent,
                             max_length=300 * page)
        assert torch.equal(got.index, again.index) and torch.equal(got.table, again.table)


@pytest.mark.parametrize("total", [127, 128, 129, 255, 256, 257, 1023, 1024, 1025, 2048, 2049, 8192, 8193, 20011])
def test_many_pages(total):
    bounds = PageBounds(random_bounds(total, 2, 64, BF16, 5), 16)
    table = torch.randperm(total, generator=torch.Generator().manual_seed(1)).int()[None].cuda()
    q = torch.randn(1, 8, 64, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    for n in (total * 16, total * 16 - 15, min(total, 600) * 16):
        lengths = torch.tensor([n], dtype=torch.int32)
        for count in (1, 100, total // 2, total - 1):
            got = select_pages(q, bounds, table, lengths.cuda(), count)
            check_selection(got, expected_index(q, bounds.values, table, lengths, 16, count, 0, 1,
                                                total * 16), table)


def test_equal_scores_and_special_values():
    """Pages alike go by their place; infinities, NaN and -0 have theirs."""
    total, dim = 700, 32
    values = torch.zeros(total, 1, 2, dim)
    g = torch.Generator().manual_seed(4)
    values[:, 0, :, 0] = torch.randint(-2, 3, (total, 1), generator=g).float()
    values[5:9, 0, :, 1] = float("inf")
    values[20:23, 0, :, 1] = float("nan")
    values[30:33, 0, :, 1] = float("-inf")
    values[40:60, 0, :, 2] = -1e-38
    table = torch.arange(total).int()[None].cuda()
    lengths = torch.tensor([total * 16], dtype=torch.int32)
    for x in (1.0, -1.0, 1e-30, 0.0, 3e38):
        q = torch.zeros(1, 2, dim)
        q[0, :, 0], q[0, 1, 1], q[0, 1, 2] = x, 0.5, 1e-30
        bounds = PageBounds(values.cuda(), 16)
        for count in (2, 10, 150, 350, 699):
            got = select_pages(q.cuda(), bounds, table, lengths.cuda(), count, sinks=1)
            check_selection(got, expected_index(q, values, table, lengths, 16, count, 1, 1,
                                                total * 16), table)
    q.fill_(float("nan"))  # every score is NaN: the first pages
    got = select_pages(q.cuda(), bounds, table, lengths.cuda(), 50, recent=3)
    assert got.index[0, 0].tolist() == [*range(47), 697, 698, 699]


def test_sequences_that_cannot_be_read():
    bounds = PageBounds(random_bounds(40, 2, 64, F16, 6), 32)
    table = torch.arange(36).int().view(3, 12).cuda()
    table[1, 3], table[1, 7] = -1, 40
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(3)).cuda()
    lengths = torch.tensor([-5, 300, 12 * 32 + 1], dtype=torch.int32)
    got = select_pages(q, bounds, table, lengths.cuda(), 4)
    want = expected_index(q, bounds.values, table, lengths, 32, 4, 0, 1, 12 * 32)
    check_selection(got, want, table)
    assert want[1].tolist()[::2] == [-1, -1]
    for chosen in want[0][1].tolist():  # the newest page, those that cannot be read, one more
        assert {3, 7, 9} < set(chosen)
    cache = PagedCache.allocate(40, 2, 32, 64, dtype=F32)
    out = paged_attention(q, cache, got.table, got.lengths)
    assert torch.isnan(out).all()


def test_offsets_past_32_bits():
    dim, pages = 256, 2 ** 31 // 512 + 40  # more than 2^31 bounds
    values = torch.zeros(pages, 1, 2, dim, dtype=BF16, device="cuda")
    bounds = PageBounds(values, 16)
    values[-30:] = random_bounds(30, 1, dim, BF16, 8)
    table = (pages - 1 - torch.randperm(30, generator=torch.Generator().manual_seed(1))).int()
    q = torch.randn(1, 4, dim, generator=torch.Generator().manual_seed(2)).cuda()
    lengths = torch.tensor([30 * 16 - 3], dtype=torch.int32)
    got = select_pages(q, bounds, table[None].cuda(), lengths.cuda(), 9)
    small = expected_index(q, values[-30:], table[None] - (pages - 30), lengths, 16, 9, 0, 1, 480)
    check_selection(got, small, table[None])


# ---------------------------------------------------------------- attention

def check_attention(q, cache, chosen, got):
    out, lse = (t.cpu().double() for t in got)
    heads, d = cache.heads, cache.head_dim
    scale, info = d ** -0.5, torch.finfo(q.dtype)
    x = q.cpu().double().unflatten(1, (heads, -1))
    out, lse = out.unflatten(1, (heads, -1)), lse.unflatten(1, (heads, -1))
    for b, n in enumerate(chosen.lengths.tolist()):
        if n == 0:
            assert (out[b] == 0).all() and (lse[b] == float("-inf")).all()
            continue
        for h in range(heads):
            pages = [p for p in chosen.table[b, h].tolist() if p >= 0]
            rows = [page_rows(cache, p, cache.page_size) for p in pages]
            k, v = (torch.cat([r[i] for r in rows])[:n, h].cpu().double() for i in range(2))
            s, size = scale * x[b, h] @ k.T, scale * x[b, h].abs() @ k.abs().T
            w = torch.softmax(s, -1)
            want, a, total = w @ v, w @ v.abs(), torch.logsumexp(s, -1)
            relative = ((d + 8) * 2.0 ** -23 * size.amax(-1) + 2.0 ** -22 * s.abs().amax(-1)
                        + 2.0 ** -23 + (2 * n / 128 + 300) * 2.0 ** -23)
            tol = (2 * a * relative[:, None] + a * 2.0 ** -17
                   + info.eps / 2 * want.abs().clamp(min=info.tiny))
            assert ((out[b, h] - want).abs() <= tol).all(), (b, h)
            assert ((lse[b, h] - total).abs() <= 2 * relative + 2.0 ** -22 * total.abs()).all()


@pytest.mark.parametrize("q_type,form", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, FP8),
                                         (F16, INT8), (F32, INT8), (BF16, FP4), (F32, FP4)])
@pytest.mark.parametrize("q_heads,heads,dim,page,count", [
    (4, 2, 64, 16, 5), (6, 1, 128, 32, 12), (40, 2, 32, 64, 3), (3, 3, 256, 16, 40)])
def test_attention_to_the_selected(q_type, form, q_heads, heads, dim, page, count):
    print(f"selected {q_type} {form} {q_heads, heads, dim, page, count}", flush=True)
    cache, table, lengths = filled(form, heads, page, dim,
                                   [0, 1, page, 5 * page + 3, 47 * page - 1, 60 * page])
    bounds = PageBounds.allocate(cache)
    update_page_bounds(bounds, cache, table, lengths, new=60 * page)
    q = 2 * torch.randn(6, q_heads, dim, generator=torch.Generator().manual_seed(5))
    q = q.to(q_type).cuda()
    chosen = select_pages(q, bounds, table, lengths, count, sinks=1, recent=2)
    check_attention(q, cache, chosen, paged_attention(q, cache, chosen.table, chosen.lengths,
                                                      return_lse=True))
    # every page: the whole sequence, bit for bit
    every = select_pages(q, bounds, table, lengths, table.shape[1])
    for a, b in zip(paged_attention(q, cache, every.table, every.lengths, return_lse=True),
                    paged_attention(q, cache, table, lengths, return_lse=True)):
        assert torch.equal(a, b)


def test_lists_for_each_head():
    """Any lists will do, in any strides, also where the work goes by equal shares."""
    cache, table, lengths = filled(BF16, 4, 16, 64, [3000] * 24)
    q = torch.randn(24, 8, 64, generator=torch.Generator().manual_seed(6)).bfloat16().cuda()
    g = torch.Generator("cuda").manual_seed(7)
    lists = torch.stack([table[:, torch.randperm(188, generator=g, device="cuda")]
                         for _ in range(4)], 1)[:, :, :60]
    kept = torch.randint(0, 60 * 16 + 1, (24,), generator=g, device="cuda").int()
    strided = torch.empty(60, 24, 4, dtype=torch.int32, device="cuda")
    strided.copy_(lists.permute(2, 0, 1))
    got = paged_attention(q, cache, lists, kept, return_lse=True)
    for a, b in zip(got, paged_attention(q, cache, strided.permute(1, 2, 0), kept,
                                         return_lse=True)):
        assert torch.equal(a, b)
    for h in range(4):  # one list for all heads is the plain table
        one = paged_attention(q, cache, lists[:, h].contiguous(), kept, return_lse=True)
        for a, b in zip(got, one):
            assert torch.equal(a[:, 2 * h:2 * h + 2], b[:, 2 * h:2 * h + 2])
    big, big_table, n = filled(FP8, 2, 64, 256, [30000, 50000, 1, 40001, 30000, 50000], spare=0)
    lists = torch.stack([big_table, big_table.flip(0)], 1)
    n = torch.full((6,), 1, dtype=torch.int32, device="cuda")
    n[1], n[4] = 30000, 29999
    q = torch.randn(6, 32, 256, generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    got = paged_attention(q, big, lists, n)
    for h, t in enumerate((big_table, big_table.flip(0))):
        assert torch.equal(got[:, 16 * h:16 * h + 16],
                           paged_attention(q, big, t.contiguous(), n)[:, 16 * h:16 * h + 16])


def test_refusals():
    cache, table, lengths = filled(BF16, 2, 16, 32, [40, 20])
    bounds = PageBounds.allocate(cache)
    q = torch.randn(2, 4, 32).bfloat16().cuda()
    good = dict(bounds=bounds, cache=cache, block_table=table, lengths=lengths)
    other = PageBounds.allocate(PagedCache.allocate(cache.pages, 2, 16, 32, dtype=F32))
    for change in (dict(bounds=other), dict(bounds=PageBounds(bounds.values, 32)),
                   dict(bounds=PageBounds(bounds.values[1:].clone(), 16)),
                   dict(bounds=PageBounds(bounds.values.cpu(), 16)), dict(block_table=table[:1]),
                   dict(block_table=table.long()), dict(block_table=table.cpu()),
                   dict(lengths=lengths.long()), dict(lengths=lengths[:1]), dict(new=0),
                   dict(lengths=lengths[None]), dict(max_length=table.shape[1] * 16 + 1)):
        with pytest.raises(ValueError):
            update_page_bounds(**{**good, **change})
    good = dict(q=q, bounds=bounds, block_table=table, lengths=lengths, count=2)
    for change in (dict(q=q[0]), dict(q=q.double()), dict(q=q.cpu()), dict(q=q[:, :3]),
                   dict(q=q[..., :16]), dict(q=q[:1]), dict(count=0), dict(count=1 << 26),
                   dict(count=(1 << 32) + 2), dict(count=1, sinks=1),
                   dict(recent=0), dict(sinks=-1), dict(max_length=-1),
                   dict(max_length=table.shape[1] * 16 + 1), dict(block_table=table.long()),
                   dict(lengths=lengths.long()), dict(lengths=lengths.cpu()),
                   dict(q=q.clone().requires_grad_()),
                   dict(bounds=PageBounds(bounds.values.cpu(), 16)),
                   dict(workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(ValueError):
            select_pages(**{**good, **change})
    lists = table[:, None].expand(2, 2, -1)
    for bad in (lists[:, :1], lists[:1], lists[None], lists.long(), table[0]):
        with pytest.raises(ValueError):
            paged_attention(q, cache, bad, lengths)
    with pytest.raises(ValueError):
        paged_attention(q, cache, lists, lengths, window=5)
    assert select_workspace_bytes(q, bounds, 64, 4) == 256
    assert select_pages(q[:0], bounds, table[:0], lengths[:0], 2).table.shape == (0, 2, 2)
    none = select_pages(q, bounds, table[:, :0], torch.zeros_like(lengths), 2)
    assert (none.index == -1).all() and (none.lengths == 0).all()


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("dtype,form", [(BF16, BF16), (F16, FP4), (F32, INT8)])
def test_decoding_with_selected_pages(dtype, form):
    """Prompts and steps: append, bounds, selection, attention; one graph of the step,
    replayed beside the eager one on a cache of its own."""
    batch, q_heads, heads, dim, page, columns, count = 3, 8, 2, 64, 16, 30, 6
    f = rotary.rotary_frequencies(dim, device="cuda")
    table = torch.randperm(batch * columns, generator=torch.Generator().manual_seed(3))
    table = table.view(batch, columns).int().cuda()
    caches = [PagedCache.allocate(batch * columns, heads, page, dim, dtype=form) for _ in range(2)]
    bounds = [PageBounds.allocate(c) for c in caches]
    g = torch.Generator("cuda").manual_seed(4)
    prompts = torch.tensor([1, 77, 200])
    k, v = (torch.randn(batch, 200, heads, dim, generator=g, device="cuda").to(dtype)
            for _ in range(2))
    positions = torch.arange(200).repeat(batch, 1)
    positions[positions >= prompts[:, None]] = -1
    lengths = prompts.int().cuda()
    for c, e in zip(caches, bounds):
        cache_append(c, None, k, v, positions.cuda(), f, block_table=table)
        update_page_bounds(e, c, table, lengths, new=200)
    q, k, v = (torch.zeros(batch, 1, h, dim, dtype=dtype, device="cuda")
               for h in (q_heads, heads, heads))
    position = torch.zeros(batch, 1, dtype=torch.int64, device="cuda")

    def step(c, e):
        turned = cache_append(c, q, k, v, position, f, block_table=table)[:, 0]
        n = (position[:, 0] + 1).int()
        update_page_bounds(e, c, table, n)
        chosen = select_pages(turned, e, table, n, count, sinks=1)
        return turned, chosen, paged_attention(turned, c, chosen.table, chosen.lengths,
                                               return_lse=True)

    def fill(rep):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, device="cuda", generator=g))
        position.copy_((prompts + rep)[:, None])

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[0], bounds[0])
        step(caches[1], bounds[1])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turned, chosen, out = step(caches[0], bounds[0])
    for rep in range(1, 40):
        fill(rep)
        graph.replay()
        torch.cuda.synchronize()
        _, other, want = step(caches[1], bounds[1])
        assert torch.equal(chosen.index, other.index), rep
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), rep
        if rep % 13 == 0:
            n = (prompts + rep + 1).int().cuda()
            assert same(bounds[0].values, expected_bounds(caches[0], table, n, 1 << 30,
                                                          bounds[0].values))
            check_selection(chosen, expected_index(turned, bounds[0].values, table, n.cpu(), page,
                                                   count, 1, 1, columns * page), table)
            check_attention(turned, caches[0], chosen, out)
