"""The 4-bit cache on the GPU: written and read rows bit for bit as defined (a division
by a power of two is exact, so the codes are determined), and attention over them
against softmax in 64 bits.

The attention's tolerance is that of the other caches, derived in
test_gpu_paged_attention.py: the codes times their scales are exact in BF16, so nothing
is added to it."""
from __future__ import annotations

import pytest
import torch

from tests import fp4
from fireprot_amd import kv_cache
from fireprot_amd.kv_cache import FP4, PagedCache, cache_read, cache_write
from fireprot_amd.paged_attention import paged_attention, workspace_bytes

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ROWS = [F32, BF16, F16]


def raw(t):
    return t.view(torch.uint8)


def random_cache(pages, heads, page, dim, seed=9):
    cache = PagedCache.allocate(pages, heads, page, dim, dtype=FP4)
    g = torch.Generator(device="cuda").manual_seed(seed)
    for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        raw(t).random_(0, 250, generator=g)
    return cache


def rows(tokens, heads, dim, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, heads, dim, generator=g)
    return (x * torch.exp(torch.randn(tokens, heads, dim // 32, generator=g)).repeat_interleave(
        32, -1)).to(dtype).cuda()


def held(data, scale, slots):
    """Values at slots, [n, heads, d] in float64."""
    page = data.shape[2]
    at = slots.cpu().clamp(0, data.shape[0] * page - 1)
    index = (at // page, slice(None), at % page)
    return fp4.values(raw(data).cpu()[index], raw(scale).cpu()[index])


@pytest.mark.parametrize("row", ROWS)
@pytest.mark.parametrize("tokens,heads,page,dim", [(1, 1, 16, 32), (37, 3, 16, 64),
                                                   (130, 8, 64, 128), (67, 5, 32, 256)])
def test_write_and_read_back(row, tokens, heads, page, dim):
    print(f"fp4 cache {row} {tokens, heads, page, dim}", flush=True)
    pages = tokens // page + 4
    cache = random_cache(pages, heads, page, dim)
    k, v = rows(tokens, heads, dim, row), rows(tokens, heads, dim, row, 2)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(4))[:tokens]
    if tokens > 4:
        slots[1], slots[2], slots[3] = -1, -2 ** 62, pages * page
    want = [raw(t).cpu() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    cache_write(cache, k, v, slots.cuda())
    kept = (slots >= 0) & (slots < pages * page)
    p, o = slots[kept] // page, slots[kept] % page
    for w, x in ((0, k), (1, v)):
        want[w][p, :, o], want[w + 2][p, :, o] = fp4.quantise(x.cpu()[kept])
    for t, x in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), want):
        assert torch.equal(raw(t).cpu(), x), "written rows and nothing else"
    back = slots[torch.randint(0, tokens, (2 * tokens,), generator=torch.Generator().manual_seed(5))]
    for out_type in ROWS:
        for got, data, scale in zip(cache_read(cache, back.cuda(), dtype=out_type),
                                    (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
            x = held(data, scale, back)
            x[back < 0], x[back >= pages * page] = 0.0, float("nan")
            x = x.to(out_type)
            assert torch.equal(torch.isnan(got.cpu()), torch.isnan(x))
            assert torch.equal(torch.nan_to_num(got.cpu()), torch.nan_to_num(x))
    assert cache_read(cache, back.cuda())[0].dtype == F32


def test_rows_at_the_edges_of_the_codes():
    up, down = (lambda x: torch.nextafter(torch.tensor(x), torch.tensor(9e9)).item(),
                lambda x: torch.nextafter(torch.tensor(x), torch.tensor(0.0)).item())
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    x = torch.zeros(16, 1, 64)
    x[1, 0, :8] = torch.tensor([6.0, *ties])
    x[2, 0, :8] = torch.tensor([6.0, *map(up, ties)])
    x[3, 0, :8] = -torch.tensor([6.0, *map(down, ties)])
    x[4, 0, 0], x[4, 0, 1] = 7.0, 6.5
    x[5, 0, 0], x[5, 0, 1] = up(7.0), 6.5
    x[6, 0, 0], x[6, 0, 33] = down(7.0), 1e-3     # two blocks, unlike scales
    x[7, 0, 0] = 2.0 ** -100
    x[8, 0, 0] = down(2.0 ** -100)
    x[9, 0, 1], x[9, 0, 2] = torch.finfo(F32).max, -3.0e38
    x[10, 0, 5], x[10, 0, 6], x[10, 0, 40] = float("inf"), 1.0, 1.0
    x[11, 0, 63], x[11, 0, 0] = float("nan"), 2.0
    x[12] = -0.0
    x[13, 0, 0] = 2.0 ** -149
    x[14, 0] = torch.linspace(-3, 3, 64)
    x[15, 0, 0], x[15, 0, 1] = 1.75 * 2.0 ** 127, -(2.0 ** 125)
    cache = PagedCache.allocate(1, 1, 16, 64, dtype=FP4)
    cache_write(cache, x.cuda(), -x.cuda(), torch.arange(16).cuda())
    for data, scale, source in ((cache.k, cache.k_scale, x), (cache.v, cache.v_scale, -x)):
        codes, scales = fp4.quantise(source)
        assert torch.equal(raw(scale)[0, 0].cpu(), scales[:, 0])
        assert torch.equal(raw(data)[0, 0].cpu(), codes[:, 0])
    k = cache_read(cache, torch.arange(16).cuda())[0].cpu()
    bad = torch.isnan(k)
    assert bad[10, 0, :32].all() and bad[11, 0, 32:].all() and bad.sum() == 64
    assert torch.isfinite(k[9]).all() and torch.isfinite(k[15]).all()
    # a code is off by at most a quarter of its value, or of the smallest's half step
    fine = [1, 2, 3, 4, 5, 6, 7, 14]
    scale = torch.exp2(raw(cache.k_scale)[0, 0, fine].cpu().double() - 127)
    step = x[fine].double().abs() / 4 + scale.repeat_interleave(32, -1)[:, None] / 4
    assert ((k[fine].double() - x[fine].double()).abs() <= step).all()


def test_every_code_and_scale_is_read():
    cache = PagedCache.allocate(16, 1, 16, 32, dtype=FP4)  # a scale byte to each slot
    codes = torch.arange(256 * 16, dtype=torch.int64) * 73 % 256
    raw(cache.k).copy_(codes.view(16, 1, 16, 16).to(torch.uint8))
    raw(cache.v).copy_(255 - raw(cache.k))
    for t in (cache.k_scale, cache.v_scale):
        raw(t).copy_(torch.arange(256).view(16, 1, 16, 1).to(torch.uint8))
    slots = torch.arange(256)
    for got, data, scale in zip(cache_read(cache, slots.cuda()), (cache.k, cache.v),
                                (cache.k_scale, cache.v_scale)):
        want = held(data, scale, slots).float()  # (infinite past 2^128)
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
        assert torch.equal(got.cpu()[:255], want[:255])


@pytest.mark.parametrize("view", ["fused", "odd", "broadcast", "channel_stride"])
def test_strided_rows(view):
    t, h, d = 21, 4, 64
    if view == "fused":
        x = rows(t, 3 * h, d, BF16)
        k, v = x[:, h:2 * h], x[:, 2 * h:]
    elif view == "odd":
        x = rows(t, h, 4 * d, F16)
        k, v = x[..., 1:d + 1], x[..., d + 3:2 * d + 3]
    elif view == "broadcast":
        k, v = rows(t, 1, d, F32).expand(t, h, d), rows(1, h, d, F32).expand(t, h, d)
    else:
        x = rows(t, h, 2 * d, BF16).view(t, h, d, 2)
        k, v = x[..., 0], x[..., 1]
    slots = torch.randperm(48, generator=torch.Generator().manual_seed(2))[:t].cuda()
    one, two = (PagedCache.allocate(3, h, 16, d, dtype=FP4) for _ in range(2))
    cache_write(one, k, v, slots)
    cache_write(two, k.contiguous().clone(), v.contiguous().clone(), slots)
    for a, b in zip((one.k, one.v, one.k_scale, one.v_scale),
                    (two.k, two.v, two.k_scale, two.v_scale)):
        assert torch.equal(raw(a), raw(b))
    wide = torch.full((t, h, 2 * d + 2), 7.0, dtype=F16, device="cuda")
    cache_read(one, slots, k_out=wide[..., 1:d + 1], v_out=wide[..., d + 2:])
    want = cache_read(two, slots, dtype=F16)
    assert torch.equal(wide[..., 1:d + 1], want[0]) and torch.equal(wide[..., d + 2:], want[1])
    assert (wide[..., 0] == 7).all() and (wide[..., d + 1] == 7).all()


def test_offsets_past_32_bits():
    page, dim = 4096, 256
    pages = 2 ** 32 // (page * dim // 2) + 3  # more than 2^32 bytes of codes
    cache = PagedCache.allocate(pages, 1, page, dim, dtype=FP4)
    slots = torch.tensor([0, pages * page - 1, 2 ** 32 // 128, 2 ** 32 // 128 - 1])
    k, v = rows(4, 1, dim, F32), rows(4, 1, dim, F32, 3)
    cache_write(cache, k, v, slots.cuda())
    for got, x in zip(cache_read(cache, slots.cuda()), (k, v)):
        assert torch.equal(got.cpu().double(), fp4.values(*fp4.quantise(x)))
    # one sequence whose pages lie at both ends
    table = torch.tensor([[0, pages - 1]], dtype=torch.int32).cuda()
    q = torch.randn(1, 2, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    lengths = torch.tensor([2 * page], dtype=torch.int32).cuda()
    got = paged_attention(q, cache, table, lengths)
    n = 2 * page - 2  # all other keys and values are zeros: score 0
    kv = [fp4.values(*fp4.quantise(x))[:2, 0] for x in (k, v)]
    s = q[0].cpu().double() @ kv[0].T * dim ** -0.5
    w = torch.exp(s) / (torch.exp(s).sum(-1, keepdim=True) + n)
    want = w @ kv[1]
    assert ((got[0].cpu().double() - want).abs() <= 1e-5 * (w @ kv[1].abs()) + 1e-9).all()


# ---------------------------------------------------------------- attention

class Setup:
    """Sequences in a 4-bit cache whose every other slot, and every table entry that is
    not needed, holds rubbish (scales of NaN)."""

    def __init__(self, q_type, q_heads, heads, dim, page, lengths, *, window=0, seed=1):
        g = torch.Generator().manual_seed(seed)
        batch, columns = len(lengths), max(1, -(-max([0, *lengths]) // page)) + 2
        pages = batch * columns + 2
        self.window, self.max_length, self.scale = window, columns * page, dim ** -0.5
        self.cache = PagedCache.allocate(pages, heads, page, dim, dtype=FP4)
        for t in (self.cache.k, self.cache.v, self.cache.k_scale, self.cache.v_scale):
            raw(t).fill_(255)
        order = torch.randperm(pages, generator=g)
        table = torch.full((batch, columns), -7, dtype=torch.int32)
        table[:, 1::2] = 2 ** 31 - 1
        self.slots, at = [], 0
        for b, n in enumerate(lengths):
            first = max(0, n - window) if window else 0
            for c in range(first // page, -(-n // page)):
                table[b, c] = order[at]
                at += 1
            j = torch.arange(first, n)
            self.slots.append(table[b, j // page].long() * page + j % page)
        flat = torch.cat(self.slots)
        kv = torch.randn(2, len(flat), heads, dim, generator=g)
        kv *= torch.exp(0.5 * torch.randn(2, len(flat), heads, 1, generator=g))
        cache_write(self.cache, kv[0].cuda(), kv[1].cuda(), flat.cuda())
        self.q = (2 * torch.randn(batch, q_heads, dim, generator=g)).to(q_type).cuda()
        self.table, self.lengths = table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()

    def call(self, **kw):
        kw = {"window": self.window, "max_length": self.max_length, "return_lse": True, **kw}
        return paged_attention(kw.pop("q", self.q), self.cache, kw.pop("table", self.table),
                               kw.pop("lengths", self.lengths), **kw)

    def check(self, got, only=None):
        out, lse = (t.cpu().double() for t in got)
        heads, d = self.cache.heads, self.cache.head_dim
        q = self.q.cpu().double().unflatten(1, (heads, -1))
        # (a subnormal's half step is that of the smallest normal number: FP16 outputs of
        # 1e-6 lie 2^-24 apart, 2^-25 from the nearest, not 2^-11 of themselves)
        info = torch.finfo(self.q.dtype)
        for b, slots in enumerate(self.slots):
            if only is not None and b not in only:
                continue
            n = len(slots)
            if n == 0:
                assert (out[b] == 0).all() and (lse[b] == float("-inf")).all()
                continue
            k, v = (held(t, s, slots).transpose(0, 1)
                    for t, s in ((self.cache.k, self.cache.k_scale),
                                 (self.cache.v, self.cache.v_scale)))
            s = self.scale * q[b] @ k.transpose(1, 2)
            size = self.scale * q[b].abs() @ k.abs().transpose(1, 2)
            w = torch.softmax(s, -1)
            want, a, total = w @ v, w @ v.abs(), torch.logsumexp(s, -1)
            relative = ((d + 8) * 2.0 ** -23 * size.amax(-1) + 2.0 ** -22 * s.abs().amax(-1)
                        + 2.0 ** -23 + (2 * n / 128 + 300) * 2.0 ** -23)
            tol = (2 * a * relative[..., None] + a * 2.0 ** -17
                   + info.eps / 2 * want.abs().clamp(min=info.tiny))
            gap = (out[b].view_as(want) - want).abs()
            assert (gap <= tol).all(), (b, n, (gap / tol).max().item())
            gap = (lse[b].view_as(total) - total).abs()
            assert (gap <= 2 * relative + 2.0 ** -22 * total.abs()).all(), (b, n)


RAGGED = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 640, 1025]


@pytest.mark.parametrize("q_type", ROWS)
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_ragged_lengths(q_type, dim):
    print(f"fp4 attention {q_type} dim {dim}", flush=True)
    s = Setup(q_type, 8, 2, dim, 16, RAGGED)
    s.check(s.call())


@pytest.mark.parametrize("q_type", ROWS)
@pytest.mark.parametrize("q_heads,heads,dim,page", [
    (1, 1, 32, 16), (3, 3, 64, 32), (5, 1, 128, 64), (16, 1, 128, 4096), (17, 1, 64, 16),
    (48, 2, 128, 128), (32, 1, 256, 32), (66, 2, 32, 16), (71, 1, 128, 16)])
def test_heads_and_pages(q_type, q_heads, heads, dim, page):
    print(f"fp4 attention {q_type} {q_heads, heads, dim, page}", flush=True)
    s = Setup(q_type, q_heads, heads, dim, page, [77, 300, 0, 513], seed=3)
    s.check(s.call())


@pytest.mark.parametrize("q_type", ROWS)
@pytest.mark.parametrize("window", [1, 5, 16, 100, 333, 5000])
def test_windows(q_type, window):
    s = Setup(q_type, 6, 3, 64, 32, [0, 1, 4, 16, 37, 100, 101, 500, 1999], window=window, seed=5)
    s.check(s.call())


@pytest.mark.parametrize("q_type", ROWS)
@pytest.mark.parametrize("dim", [32, 128])
def test_long_rows_and_full_cards(q_type, dim):
    s = Setup(q_type, 8, 2, dim, 64, [20011, 6001, 0, 300], seed=7)
    assert workspace_bytes(s.q, s.cache, s.max_length) > 256
    first = s.call()
    s.check(first)
    for a, b in zip(first, s.call()):
        assert torch.equal(a, b)
    s.check(s.call(max_length=20011))
    g = torch.Generator().manual_seed(8)
    lengths = torch.randint(0, 700, (1500,), generator=g)
    wide = Setup(q_type, 24, 2, dim, 16, lengths.tolist(), seed=8)
    wide.check(wide.call(), only=set(range(0, 1500, 41)))


def test_shares_of_long_sequences():
    """Enough to read that the work goes by equal shares."""
    s = Setup(BF16, 16, 8, 256, 64, [40001, 0, 30000, 1, 50123, 20000], seed=10)
    s.check(s.call(), only={0, 1, 3})


def test_what_cannot_be_read_gives_nan():
    s = Setup(F32, 4, 2, 64, 16, [100, 64, 300, 17], seed=9)
    want = s.call()
    table, lengths = s.table.clone(), s.lengths.clone()
    table[1, 2], lengths[2] = s.cache.pages, -3
    out, lse = s.call(table=table, lengths=lengths)
    for b, bad in enumerate([False, True, True, False]):
        assert torch.isnan(out[b]).all() == bad and torch.isnan(lse[b]).all() == bad
        if not bad:
            assert torch.equal(out[b], want[0][b])
    # a value's block of NaN is that of its channels, a key's of the whole head
    page, slot = divmod(int(s.slots[0][40]), 16)
    raw(s.cache.v_scale)[page, 1, slot, 1] = 255
    out, lse = s.call()
    bad = torch.isnan(out)
    assert bad[0, 2:, 32:].all() and bad.sum() == 2 * 32 and torch.isfinite(lse).all()
    raw(s.cache.k_scale)[page, 0, slot, 0] = 255
    out, lse = s.call()
    assert torch.isnan(out[0, :2]).all() and torch.isnan(lse[0, :2]).all()
    assert torch.isfinite(lse[0, 2:]).all()
