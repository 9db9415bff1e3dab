"""Attention over the paged cache on the GPU against softmax in 64 bits.

Tolerance, derived.  With a = sum_j w_j |v_j| (w the softmax weights):
* a score sums D products in FP32 (its queries split exactly), is scaled by at
  most two factors and taken to a power: at most (D + 8) 2^-23 of
  scale sum_d |q_d k_jd| in the exponent, plus 2^-22 of the score itself and one
  unit 2^-23 of the power; the maximum m enters weight and sum alike, m's own
  rounding with them;
* a weight times a value enters as two 16-bit terms: 2^-17 (BF16; FP16 2^-21);
* an accumulator takes at most n/128 + 1 tiles of 32 products and as many
  changes of reference, then joins of 4 waves and of at most 256 chunks: at
  most (2 n/128 + 300) roundings of 2^-23, those of the sum likewise.
Errors of weights and of their sum count once each, so
  |out - o| <= 2 a (delta + (2 n/128 + 300) 2^-23) + a 2^-17 + eps/2 |o|
with delta the bound on the exponent's error over the row's keys (a bound of
e^delta - 1 <= 2 delta holds where delta < 1).  The sum's logarithm is off by
twice the same relative error, plus 2^-22 of its value.
"""
from __future__ import annotations

import pytest
import torch

from fireprot_amd import kv_cache
from fireprot_amd.kv_cache import PagedCache
from fireprot_amd.paged_attention import paged_attention, workspace_bytes

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
FP8, INT8 = torch.float8_e4m3fn, torch.int8
PAIRS = [(F32, F32), (BF16, BF16), (F16, F16), (F32, FP8), (BF16, FP8), (F16, FP8), (F32, INT8),
         (BF16, INT8), (F16, INT8)]


class Setup:
    """Sequences of the given lengths in a cache whose every other slot, and
    every table entry that is not needed, holds rubbish."""

    def __init__(self, q_type, cache_type, q_heads, heads, dim, page, lengths, *, window=0,
                 spread=2.0, seed=1, max_length=None, rubbish=True):
        g = torch.Generator().manual_seed(seed)
        batch = len(lengths)
        self.window, self.lengths_list = window, list(lengths)
        longest = max([0, *lengths])
        columns = max(1, -(-longest // page)) + 2
        pages = batch * columns + 2
        self.cache = PagedCache.allocate(pages, heads, page, dim, dtype=cache_type)
        order = torch.randperm(pages, generator=g)
        table = torch.full((batch, columns), -7, dtype=torch.int32)
        table[:, 1::2] = 2 ** 31 - 1
        slots, at = [], 0
        for b, n in enumerate(lengths):
            first = max(0, n - window) if window else 0
            for c in range(first // page, -(-n // page)):
                table[b, c] = order[at]
                at += 1
            j = torch.arange(first, n)
            slots.append(table[b, j // page].long() * page + j % page)
        self.first = [max(0, n - window) if window else 0 for n in lengths]
        self.slots = slots
        flat = torch.cat(slots)
        gain = torch.exp(0.5 * torch.randn(2, len(flat), heads, 1, generator=g))
        kv = torch.randn(2, len(flat), heads, dim, generator=g) * gain
        if rubbish:
            for t in (self.cache.k, self.cache.v):
                t.view(torch.uint8).fill_(0x7F)  # NaN as float8 and, on the next line, all types
                if cache_type not in (FP8, INT8):
                    t.fill_(float("nan"))
            for t in (self.cache.k_scale, self.cache.v_scale):
                if t is not None:
                    t.fill_(float("nan"))
        kv = kv.to(q_type if cache_type in (FP8, INT8) else cache_type)
        kv_cache.cache_write(self.cache, kv[0].cuda(), kv[1].cuda(), flat.cuda())
        self.q = (torch.randn(batch, q_heads, dim, generator=g) * spread).to(q_type).cuda()
        self.table = table.cuda()
        self.lengths = torch.tensor(lengths, dtype=torch.int32).cuda()
        self.scale = dim ** -0.5
        self.max_length = columns * page if max_length is None else max_length

    def call(self, **kw):
        kw = {"window": self.window, "max_length": self.max_length, "return_lse": True, **kw}
        return paged_attention(kw.pop("q", self.q), self.cache, kw.pop("table", self.table),
                               kw.pop("lengths", self.lengths), **kw)

    def reference(self, scale=None, only=None):
        """(o, lse, tolerance of o, tolerance of lse), float64 on the CPU, of the
        sequences ``only`` (all)."""
        scale = self.scale if scale is None else scale
        b, hq, d = self.q.shape
        heads, page = self.cache.heads, self.cache.page_size
        out = torch.zeros(b, hq, d, dtype=torch.float64)
        lse = torch.full((b, hq), float("-inf"), dtype=torch.float64)
        tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
        q = self.q.cpu().double().view(b, heads, hq // heads, d)
        data = []
        for t, s in ((self.cache.k, self.cache.k_scale), (self.cache.v, self.cache.v_scale)):
            t = t.view(torch.uint8).cpu().view(t.dtype) if t.element_size() == 1 else t.cpu()
            data.append((t, None if s is None else s.cpu()))
        for i, slots in enumerate(self.slots):
            n = len(slots)
            if n == 0 or (only is not None and i not in only):
                continue
            kv = []
            for t, s in data:
                raw = t.view(torch.uint8) if t.element_size() == 1 else t
                x = raw[slots // page, :, slots % page]
                x = x.view(t.dtype).double()
                if s is not None:
                    x = x * s[slots // page, :, slots % page][..., None].double()
                kv.append(x.transpose(0, 1))  # [heads, n, d]
            k, v = kv
            s = scale * q[i] @ k.transpose(1, 2)
            size = abs(scale) * q[i].abs() @ k.abs().transpose(1, 2)
            w = torch.softmax(s, -1)
            o = w @ v
            total = torch.logsumexp(s, -1)
            delta = ((d + 8) * 2.0 ** -23 * size.amax(-1) + 2.0 ** -22 * s.abs().amax(-1)
                     + 2.0 ** -23)
            relative = delta + (2 * n / 128 + 300) * 2.0 ** -23
            a = w @ v.abs()
            out[i], lse[i] = o.reshape(hq, d), total.reshape(hq)
            info = torch.finfo(self.q.dtype)
            tol[i] = (2 * a * relative[..., None] + a * 2.0 ** -17
                      + info.eps / 2 * o.abs().clamp(min=info.tiny)).reshape(hq, d)
            ltol[i] = (2 * relative + 2.0 ** -22 * total.abs()).reshape(hq)
        return out, lse, tol, ltol

    def check(self, got, scale=None, only=None):
        out, lse = got
        want, want_lse, tol, ltol = self.reference(scale, only)
        if only is not None:
            out, lse, want, want_lse, tol, ltol = (
                t[sorted(only)] for t in (out, lse, want, want_lse, tol, ltol))
        gap = (out.cpu().double() - want).abs()
        assert not torch.isnan(gap).any()
        assert (gap <= tol).all(), f"out {(gap / tol.clamp(min=1e-300)).max().item()} of the bound"
        lse = lse.cpu().double()
        empty = torch.isinf(want_lse)
        assert torch.equal(lse[empty], want_lse[empty])
        lgap = (lse[~empty] - want_lse[~empty]).abs()
        assert (lgap <= ltol[~empty]).all()


RAGGED = [0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 256, 257, 640, 1025]


@pytest.mark.parametrize("q_type,cache_type", PAIRS)
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_ragged_lengths(q_type, cache_type, dim):
    print(f"paged {q_type} {cache_type} dim {dim}", flush=True)
    s = Setup(q_type, cache_type, 8, 2, dim, 16, RAGGED)
    s.check(s.call())


@pytest.mark.parametrize("q_type,cache_type", PAIRS)
@pytest.mark.parametrize("q_heads,heads,dim,page", [
    (1, 1, 32, 16), (3, 3, 64, 32), (5, 1, 128, 64), (16, 1, 128, 4096), (17, 1, 64, 16),
    (48, 2, 128, 128), (32, 1, 256, 32), (66, 2, 32, 16), (71, 1, 128, 16)])
def test_heads_and_pages(q_type, cache_type, q_heads, heads, dim, page):
    print(f"paged {q_type} {cache_type} {q_heads, heads, dim, page}", flush=True)
    s = Setup(q_type, cache_type, q_heads, heads, dim, page, [77, 300, 0, 513], seed=3)
    s.check(s.call())


@pytest.mark.parametrize("q_type,cache_type", [(F32, F32), (BF16, BF16), (F16, INT8), (BF16, FP8)])
@pytest.mark.parametrize("window", [1, 5, 16, 100, 333, 5000])
def test_windows(q_type, cache_type, window):
    s = Setup(q_type, cache_type, 6, 3, 64, 32, [0, 1, 4, 16, 37, 100, 101, 500, 1999],
              window=window, seed=5)
    s.check(s.call())


@pytest.mark.parametrize("q_type,cache_type", PAIRS)
def test_many_chunks(q_type, cache_type):
    s = Setup(q_type, cache_type, 8, 2, 128, 64, [20011, 6001, 0, 300], seed=7)
    assert workspace_bytes(s.q, s.cache, s.max_length) > 4 * 8 * 8 * 130 * 4  # several chunks
    s.check(s.call())
    # the bound of the lengths changes the cut, not the result
    s.check(s.call(max_length=20011))
    # one chunk a sequence, by a batch that fills the card without cutting
    wide = Setup(q_type, cache_type, 64, 64, 32, 32, [900] * 40, seed=8)
    assert workspace_bytes(wide.q, wide.cache, wide.max_length) >= 256
    wide.check(wide.call())


@pytest.mark.parametrize("q_type,cache_type", PAIRS)
@pytest.mark.parametrize("batch,q_heads,heads,dim,longest,window", [
    (700, 4, 2, 32, 600, 0), (300, 24, 1, 64, 1500, 0), (257, 40, 1, 128, 700, 300),
    (1025, 3, 1, 256, 300, 0), (5000, 2, 2, 32, 130, 50)])
def test_shares_of_many_sequences(q_type, cache_type, batch, q_heads, heads, dim, longest, window):
    """More rows than work-groups: shares begin and end inside rows, span several
    and start anywhere in the batch (empty sequences among them)."""
    print(f"paged {q_type} {cache_type} {batch, q_heads, heads, dim, longest, window}", flush=True)
    g = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, longest + 1, (batch,), generator=g)
    lengths[torch.rand(batch, generator=g) < 0.2] = 0
    lengths[-1] = longest
    s = Setup(q_type, cache_type, q_heads, heads, dim, 16, lengths.tolist(), window=window, seed=6)
    got = s.call()
    only = set(torch.randint(0, batch, (60,), generator=g).tolist()) | {0, batch - 1}
    s.check(got, only=only)
    assert (got[0][lengths == 0] == 0).all() and torch.isfinite(got[0]).all()
    # bad pages and lengths of some leave the others alone
    table, n = s.table.clone(), s.lengths.clone()
    bad = [i for i in range(batch) if i % 7 == 3 and lengths[i] > 0]
    for i in bad[::2]:
        table[i, (int(lengths[i]) - 1) // 16] = s.cache.pages
    n[bad[1::2]] = -5
    again = s.call(table=table, lengths=n)
    rest = torch.ones(batch, dtype=torch.bool)
    rest[bad] = False
    assert torch.isnan(again[0][bad]).all() and torch.isnan(again[1][bad]).all()
    # (a length left out moves the shares, and with them the sums' order)
    s.check(again, only={i for i in only if rest[i]})


@pytest.mark.parametrize("q_type,dim", [(F32, 256), (F32, 128), (BF16, 256)])
@pytest.mark.parametrize("window", [0, 200])
def test_short_rows_of_wide_heads_in_parts(q_type, dim, window):
    """Few rows of 512 keys or fewer, and of more bytes than one work-group reads."""
    s = Setup(q_type, q_type, 6, 3, dim, 16, [500, 0, 1, 130, 64, 257], seed=21,
              window=window)
    s.check(s.call())


@pytest.mark.parametrize("q_type,cache_type", [(BF16, BF16), (F16, INT8)])
def test_a_row_of_more_units_than_can_be_joined(q_type, cache_type):
    """One row of 564 000 keys: more units of a small call's size than the join has
    places for."""
    s = Setup(q_type, cache_type, 2, 1, 32, 16, [564_000], seed=18)
    s.check(s.call())


def test_more_sequences_than_a_grid_axis_has_places():
    g = torch.Generator().manual_seed(19)
    lengths = torch.randint(0, 40, (66_000,), generator=g)
    s = Setup(BF16, BF16, 2, 1, 32, 16, lengths.tolist(), seed=19)
    got = s.call()
    s.check(got, only=set(range(0, 66_000, 997)) | {65_535, 65_536, 65_999})
    assert (got[0][lengths == 0] == 0).all() and torch.isfinite(got[0]).all()


def test_queries_near_the_limit_over_codes():
    """Products with 8-bit codes are formed before their scale: a row's largest code
    is at least 224 (FP8) and 127 (INT8), 448 at most, so queries of 2^118 and more
    overflow FP32 whatever the keys.  The documented limit is 2^110."""
    for cache_type in (FP8, INT8):
        s = Setup(F32, cache_type, 2, 1, 32, 16, [100], seed=20, spread=0.0)
        s.q[0, 0, 3], s.q[0, 1, 5] = 2.0 ** 110, -(2.0 ** 110)
        s.check(s.call(scale=2.0 ** -110), 2.0 ** -110)
        s.q[0, 0, 3] = float("inf")
        out, _ = s.call()
        assert torch.isnan(out[0, 0]).all()


@pytest.mark.parametrize("q_type,cache_type", [(BF16, BF16), (BF16, FP8), (F32, F32)])
def test_long_shares(q_type, cache_type):
    """Shares of more keys than one look-up of pages serves."""
    lengths = [9000 - 101 * i for i in range(40)]
    s = Setup(q_type, cache_type, 32, 32, 32, 16, lengths, seed=16)
    s.check(s.call(), only={0, 1, 17, 38, 39})


@pytest.mark.parametrize("q_type,cache_type", PAIRS)
def test_large_and_small_scores(q_type, cache_type):
    for scale, spread in ((1.0, 4.0), (1e-3, 1.0), (-0.3, 3.0), (0.0, 1.0)):
        s = Setup(q_type, cache_type, 4, 2, 64, 16, [1, 50, 700], spread=spread, seed=9)
        s.check(s.call(scale=scale), scale)


def test_unlike_value_scales():
    """Rows of an 8-bit cache whose scales are far apart: their products with
    the weights keep their digits."""
    for cache_type in (FP8, INT8):
        s = Setup(F32, cache_type, 4, 2, 64, 16, [300], seed=10)
        g = torch.Generator().manual_seed(1)
        v = torch.randn(300, 2, 64, generator=g) * 10.0 ** torch.randint(-12, 13, (300, 2, 1),
                                                                         generator=g).float()
        k = torch.randn(300, 2, 64, generator=g)
        kv_cache.cache_write(s.cache, k.cuda(), v.cuda(), s.slots[0].cuda())
        s.check(s.call())


@pytest.mark.parametrize("q_type,cache_type", PAIRS)
def test_bad_pages_and_lengths_give_nan(q_type, cache_type):
    s = Setup(q_type, cache_type, 8, 2, 64, 16, [40, 200, 3000, 17, 64, 0], seed=11)
    good, good_lse = s.call()
    pages = s.cache.pages
    for b, column, page in ((0, 2, -1), (1, 0, pages), (2, 187, 2 ** 31 - 1), (3, 1, -2 ** 31)):
        table = s.table.clone()
        table[b, column] = page
        out, lse = s.call(table=table)
        assert torch.isnan(out[b]).all() and torch.isnan(lse[b]).all()
        rest = [i for i in range(6) if i != b]
        assert torch.equal(out[rest], good[rest]) and torch.equal(lse[rest], good_lse[rest])
    lengths = s.lengths.clone()
    lengths[0], lengths[4], lengths[5] = -1, s.max_length + 1, -2 ** 31
    out, lse = s.call(lengths=lengths)
    assert torch.isnan(out[[0, 4, 5]]).all() and torch.isnan(lse[[0, 4, 5]]).all()
    assert torch.equal(out[1:4], good[1:4])
    out, _ = s.call(max_length=199)
    assert torch.isnan(out[1:3]).all() and torch.isfinite(out[[0, 3, 4, 5]]).all()


@pytest.mark.parametrize("q_type,cache_type", [(F32, F32), (BF16, BF16), (F16, F16)])
def test_nonfinite_keys_and_values(q_type, cache_type):
    s = Setup(q_type, cache_type, 4, 1, 64, 16, [100, 100, 100, 100], seed=12)
    good, _ = s.call()
    p = [int(x[50]) for x in s.slots]
    s.cache.k[p[0] // 16, 0, p[0] % 16, 3] = float("nan")
    s.cache.v[p[1] // 16, 0, p[1] % 16, 5] = float("inf")
    s.cache.v[p[2] // 16, 0, p[2] % 16, 7] = float("nan")
    out, lse = s.call()
    assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all()
    assert (out[1, :, 5] == float("inf")).all() and torch.isnan(out[2, :, 7]).all()
    keep = torch.arange(64) != 5
    assert torch.equal(out[1][:, keep], good[1][:, keep])
    assert torch.equal(out[3], good[3])
    # all scores -inf: 0 / 0, as softmax gives
    s.cache.k[:] = float("-inf")
    out, _ = s.call(q=torch.ones_like(s.q))
    assert torch.isnan(out).all()


def test_offsets_past_32_bits():
    page, dim = 4096, 256
    for cache_type in (INT8, BF16):
        pages = 2 ** 31 // (page * dim) + 4
        cache = PagedCache.allocate(pages, 1, page, dim, dtype=cache_type)
        s = Setup(BF16, cache_type, 4, 1, dim, 16, [700], seed=13)
        j = torch.arange(700)
        k, v = kv_cache.cache_read(s.cache, s.slots[0].cuda(), dtype=F32)
        kv_cache.cache_write(cache, k, v, ((pages - 1) * page + j).cuda())
        table = torch.tensor([[pages - 1]], dtype=torch.int32).cuda()
        out, lse = paged_attention(s.q, cache, table, s.lengths, max_length=s.max_length,
                                   return_lse=True)
        want, want_lse = s.call()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("q_type,cache_type", [(F32, F32), (BF16, FP8), (F16, F16)])
def test_strides_and_given_outputs(q_type, cache_type):
    s = Setup(q_type, cache_type, 6, 2, 64, 16, [5, 90, 1200], seed=14)
    want, want_lse = s.call()
    b, h, d = s.q.shape
    wide = torch.zeros(b, h, d + 32, dtype=q_type, device="cuda")
    wide[..., 16:16 + d] = s.q
    odd = torch.zeros(b * h * d + 1, dtype=q_type, device="cuda")
    odd[1:] = s.q.flatten()
    swapped = s.q.transpose(0, 1).contiguous().transpose(0, 1)
    tall = torch.zeros(b, h, d, 2, dtype=q_type, device="cuda")
    tall[..., 1] = s.q
    for q in (wide[..., 16:16 + d], odd[1:].view(b, h, d), swapped, tall[..., 1]):
        out, lse = s.call(q=q)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    buffer = torch.full((b, h + 1, d + 16), 7.0, dtype=q_type, device="cuda")
    got, _ = s.call(out=buffer[:, :h, :d])
    assert got.data_ptr() == buffer.data_ptr() and torch.equal(buffer[:, :h, :d], want)
    buffer[:, :h, :d] = 7.0
    assert (buffer == 7.0).all()
    same = s.q.clone()
    s.call(q=same, out=same)
    assert torch.equal(same, want)
    table = torch.zeros(b, s.table.shape[1], 2, dtype=torch.int32, device="cuda")
    table[..., 0] = s.table
    lengths = torch.stack([s.lengths, s.lengths * 0], 1)[:, 0]
    assert torch.equal(s.call(table=table[..., 0], lengths=lengths)[0], want)
    assert torch.equal(s.call(table=s.table[:, :76], max_length=76 * 16)[0], want)


@pytest.mark.parametrize("longest", [150, 3000])
def test_sequences_that_share_their_pages(longest):
    """One row of the table, and one query, for every sequence (zero strides)."""
    s = Setup(BF16, FP8, 8, 2, 64, 16, [longest] * 3, seed=22)
    s.table[1:], s.q[1:] = s.table[:1], s.q[:1]
    lengths = torch.tensor([longest, 0, longest - 41], dtype=torch.int32, device="cuda")
    want, want_lse = s.call(lengths=lengths)
    got, got_lse = s.call(q=s.q[:1].expand_as(s.q), table=s.table[:1].expand_as(s.table),
                          lengths=lengths)
    assert torch.equal(got, want) and torch.equal(got_lse, want_lse)
    first, _ = s.call(lengths=lengths[:1].expand(3))
    assert torch.equal(first, want[:1].expand_as(first))


def test_poisoned_workspace_and_repeats():
    s = Setup(BF16, BF16, 32, 8, 128, 16, [1, 3000, 12000, 0], seed=15)
    want, want_lse = s.call()
    size = workspace_bytes(s.q, s.cache, s.max_length)
    for fill in (0xFF, 0x00, 0x7F):
        ws = torch.full((size + 64,), fill, dtype=torch.uint8, device="cuda")
        out, lse = s.call(workspace=ws[:size])
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        assert (ws[size:] == fill).all()
    with pytest.raises(ValueError, match="workspace"):
        s.call(workspace=ws[:size - 1])


def test_two_streams_and_two_graphs():
    a = Setup(BF16, BF16, 16, 4, 128, 16, [9000, 100], seed=16)
    b = Setup(BF16, BF16, 16, 4, 128, 16, [7000, 4100], seed=17)
    want = [a.call()[0], b.call()[0]]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s, stream in zip((a, b), streams):
        with torch.cuda.stream(stream):
            got.append(s.call()[0])
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # two graphs captured one after the other, replayed side by side
    graphs, outs = [], []
    for s in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(s.call()[0])
        graphs.append(graph)
    for rep in range(4):
        for s in (a, b):
            s.lengths.copy_(torch.tensor([s.lengths_list[0] - 100 * rep, 50 + rep]))
            s.q.copy_(torch.randn(s.q.shape, generator=torch.Generator().manual_seed(rep)))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for s, out in zip((a, b), outs):
            assert torch.equal(out, s.call()[0])


def test_refusals_on_the_device():
    s = Setup(BF16, BF16, 4, 2, 64, 16, [20, 30])
    q, cache, table, n = s.q, s.cache, s.table, s.lengths
    for args, kw in (((q.float(), cache, table, n), {}), ((q[0], cache, table, n), {}),
                     ((q[..., :32], cache, table, n), {}), ((q[:, :3], cache, table, n), {}),
                     ((q, cache, table.long(), n), {}), ((q, cache, table[:1], n), {}),
                     ((q, cache, table, n.long()), {}), ((q, cache, table, n[:1]), {}),
                     ((q, cache, table.cpu(), n), {}), ((q, cache, table, n), dict(window=-1)),
                     ((q, cache, table, n), dict(max_length=table.shape[1] * 16 + 1)),
                     ((q, cache, table, n), dict(max_length=-1)),
                     ((q, cache, table, n), dict(out=q[:1])),
                     ((q, cache, table, n), dict(out=q.float())),
                     ((q, cache, table, n), dict(out=q[:, :1].expand_as(q))),
                     ((q.clone().requires_grad_(), cache, table, n), {})):
        with pytest.raises(ValueError):
            paged_attention(*args, **kw)
    with pytest.raises(RuntimeError, match="status 2"):
        paged_attention(q, cache, table, n, scale=float("nan"))


def test_no_sequences_and_no_tokens():
    s = Setup(F16, F16, 4, 2, 64, 16, [20, 30])
    out, lse = s.call(q=s.q[:0], table=s.table[:0], lengths=s.lengths[:0])
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    out, lse = s.call(table=s.table[:, :0], lengths=s.lengths * 0, max_length=0)
    assert (out == 0).all() and (lse == float("-inf")).all()
