"""Errors of the attention over the paged cache beside those of a plain form in
32 bits, row by row: bounds that lost bits show up against, at lengths from a
single key on.

Tolerances, derived.  The plain form rounds every product, sum, power and
quotient to FP32 and its output to q's type.  The kernel takes the same steps, in
other orders, with up to three roundings more on the way to an exponent (log2 e
times the scale, times the key's own scale, their product with the sum) and one
for each wave and share that is joined.  Independent roundings add up in squares,
so for FP32 outputs the root of the mean square error stays within a small factor
of the plain form's: 4 are allowed, and one unit, 2^-23, for rows that the plain
form gets exactly.  16-bit outputs have the last rounding in common, which is all
but the whole of either error; the weights' own 16 bits, 2^-16 of each, are added
outright, and a tenth for outputs that fall on the other side of a tie.

With queries of zero every weight is 1 and its sum n, exactly, and a row of n <= 4
keys lies in one wave's tile: an output is the sum of n products (three each where
weights are split in three; all exact, 8 bits by 8) over n, the reciprocal's, its
product's and the sums' roundings no more than 3n + 4, each 2^-23 of sum |v| / n.
"""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_paged_attention import BF16, F16, F32, FP8, INT8, PAIRS, Setup

pytestmark = pytest.mark.gpu


def rows(s, i, dtype):
    """Keys and values [heads, n, D] of sequence i, as the cache holds them."""
    out, slots, page = [], s.slots[i], s.cache.page_size
    for t, scale in ((s.cache.k, s.cache.k_scale), (s.cache.v, s.cache.v_scale)):
        raw = t.view(torch.uint8).cpu() if t.element_size() == 1 else t.cpu()
        x = raw[slots // page, :, slots % page]
        x = (x.view(t.dtype) if t.element_size() == 1 else x).to(dtype)
        if scale is not None:
            x = x * scale.cpu()[slots // page, :, slots % page][..., None].to(dtype)
        out.append(x.transpose(0, 1).contiguous())
    return out


def attend(s, i, dtype):
    """(o [q_heads, D], lse [q_heads]) of sequence i, every step in ``dtype``."""
    k, v = rows(s, i, dtype)
    q = s.q[i].cpu().to(dtype).view(s.cache.heads, -1, s.cache.head_dim)
    x = torch.bmm(q, k.transpose(1, 2).contiguous()) * s.scale
    top = x.amax(-1, keepdim=True)
    w = torch.exp(x - top)
    total = w.sum(-1, keepdim=True)
    return ((torch.bmm(w, v) / total).reshape(s.q.shape[1:]),
            (top + torch.log(total)).reshape(s.q.shape[1]))


def rms(x):
    return x.double().square().mean().sqrt().item()


LENGTHS = [1, 2, 3, 4, 17, 130, 700, 4097]


@pytest.mark.parametrize("q_type,cache_type", PAIRS)
@pytest.mark.parametrize("q_heads,heads,dim", [(8, 2, 64), (8, 8, 32), (20, 1, 128), (8, 2, 256)])
def test_errors_are_of_the_plain_form_s_size(q_type, cache_type, q_heads, heads, dim):
    print(f"precision {q_type} {cache_type} {q_heads, heads, dim}", flush=True)
    s = Setup(q_type, cache_type, q_heads, heads, dim, 16, LENGTHS, seed=31)
    out, lse = (t.cpu() for t in s.call())
    for i, n in enumerate(LENGTHS):
        want, want_lse = attend(s, i, torch.float64)
        plain, plain_lse = attend(s, i, torch.float32)
        size = rms(want)
        here = rms(out[i].double() - want) / size
        there = rms(plain.to(q_type).double() - want) / size
        most = 4.0 * there + 2.0 ** -23 if q_type == F32 else 1.1 * there + 2.0 ** -16
        assert here <= most, f"{n} keys: {here:.3e}, the plain form {there:.3e}"
        gap = rms(lse[i].double() - want_lse)
        most = 4.0 * rms(plain_lse.double() - want_lse) + 2.0 ** -22 * (1 + rms(want_lse))
        assert gap <= most, f"{n} keys, lse: {gap:.3e}"


@pytest.mark.parametrize("cache_type", [F32, FP8, INT8])
@pytest.mark.parametrize("q_heads,heads,dim", [(2, 2, 32), (5, 1, 64), (24, 1, 128), (3, 1, 256)])
def test_weights_of_fp32_outputs_are_whole(cache_type, q_heads, heads, dim):
    lengths = [1, 2, 3, 4]
    s = Setup(F32, cache_type, q_heads, heads, dim, 16, lengths, seed=32, spread=0.0)
    out, _ = s.call()
    for i, n in enumerate(lengths):
        _, v = rows(s, i, torch.float64)
        v = v.repeat_interleave(q_heads // heads, 0)
        gap = (out[i].cpu().double() - v.mean(1)).abs()
        tol = (3 * n + 4) * 2.0 ** -23 * v.abs().mean(1)
        assert (gap <= tol).all(), f"{n} keys: {(gap / tol.clamp(min=1e-300)).max().item()}"


@pytest.mark.parametrize("q_type,cache_type", [(F32, F32), (BF16, BF16), (F16, INT8), (F32, FP8)])
def test_rows_that_are_not_cut(q_type, cache_type):
    """More rows than work-groups fit the card, each in one unit and without a join."""
    from fireprot_amd.paged_attention import NO_WORKSPACE, workspace_bytes

    lengths = [400 - 9 * i for i in range(40)]
    s = Setup(q_type, cache_type, 64, 64, 32, 32, lengths, seed=33)
    assert workspace_bytes(s.q, s.cache, s.max_length) == NO_WORKSPACE
    s.check(s.call(), only={0, 1, 20, 38, 39})


@pytest.mark.parametrize("q_type,cache_type", PAIRS)
@pytest.mark.parametrize("batch,q_heads,heads,dim,longest", [
    (3, 8, 2, 64, 300), (90, 24, 1, 128, 700), (300, 4, 2, 32, 130), (70, 12, 4, 256, 40)])
def test_shares_by_a_loose_bound(q_type, cache_type, batch, q_heads, heads, dim, longest):
    """A bound far above the lengths, as a captured graph is given: by it the call may
    read so much that it goes by shares, of sequences that are short, and empty."""
    from fireprot_amd.paged_attention import workspace_bytes

    print(f"loose bound {q_type} {cache_type} {batch, q_heads, heads, dim, longest}", flush=True)
    g = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, longest + 1, (batch,), generator=g)
    lengths[torch.rand(batch, generator=g) < 0.2] = 0
    lengths[-1] = longest
    bound = 1 << 20
    s = Setup(q_type, cache_type, q_heads, heads, dim, 4096, lengths.tolist(), seed=34,
              max_length=bound)
    wide = torch.full((batch, bound // 4096), -9, dtype=torch.int32, device="cuda")
    wide[:, :s.table.shape[1]] = s.table
    # (the size goes by the number of shares, not by the bound)
    assert workspace_bytes(s.q, s.cache, bound) == workspace_bytes(s.q, s.cache, bound // 2) > 256
    got = s.call(table=wide)
    s.check(got, only=set(range(0, batch, max(1, batch // 40))) | {batch - 1})
    assert (got[0][lengths == 0] == 0).all() and torch.isfinite(got[0]).all()
    again = s.call(table=wide)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("batch", [80, 150])
def test_calls_of_many_units(batch):
    """More work-groups of one unit each than the card holds at once, and joined: 2560
    of them for 80 sequences (two units to a row).  150 may read 221 MB and go by
    shares."""
    from fireprot_amd.paged_attention import workspace_bytes

    lengths = [(37 * i) % 701 for i in range(batch)]
    s = Setup(F16, INT8, 16, 16, 64, 16, lengths, seed=35)
    size, units = workspace_bytes(s.q, s.cache, s.max_length), 2 * 16 * batch
    assert (size > units * 2 * 64 * 4) == (batch == 80)
    s.check(s.call(), only=set(range(0, batch, 7)) | {batch - 1})
