"""The decoding operators as they are used together: a batch of sequences with
prompts of unlike lengths is prefilled into the paged cache and then extended
token by token (rotary positions in place, the rows written at their slots,
attention over the sequence's pages), against attention over the whole sequence
in 64 bits.

Tolerance, derived.  The reference rotates the raw keys and queries in 64 bits;
here each is rounded to its type once, eps/2 of its size, after errors below
2^-21 of |x1| + |x2| <= sqrt(2) |(x1, x2)|.  A score moves by at most scale *
sum_d |q_d| |k_d| taken over rotated pairs' lengths, times (eps + 2^-19); so do
the exponents, and an output by twice that times a = sum_j w_j |v_j|.  The
attention itself adds what its own test allows: (D + 8) 2^-23 of the same sum,
2^-17 a, (2 n / 128 + 300) 2^-23 twice, and eps/2 of the output.  In an 8-bit
cache the reference takes the rows that are read back, so only the queries'
rounding counts.
"""
from __future__ import annotations

import pytest
import torch

from fireprot_amd import kv_cache, rotary
from fireprot_amd.kv_cache import PagedCache
from fireprot_amd.paged_attention import paged_attention

pytestmark = pytest.mark.gpu

Q_HEADS, HEADS, DIM, PAGE, ROTARY = 8, 2, 64, 16, 32


def turn(x, positions, f, layout):
    """Rotated rows [n, h, D] in float64, and each channel's pair length."""
    x = x.double()
    angle = (positions.double()[:, None] * f.inv_freq.cpu())[:, None]
    cos, sin = torch.cos(angle) * f.scale, torch.sin(angle) * f.scale
    r = f.rotary_dim
    a, b = ((slice(0, r // 2), slice(r // 2, r)) if layout == "half"
            else (slice(0, r, 2), slice(1, r, 2)))
    y, size = x.clone(), x.abs()
    y[..., a], y[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., b] * cos + x[..., a] * sin
    size[..., a] = size[..., b] = f.scale * torch.sqrt(x[..., a] ** 2 + x[..., b] ** 2)
    return y, size


class Sequences:
    """The raw rows of every token so far, on the CPU."""

    def __init__(self, lengths, dtype, seed):
        self.g = torch.Generator().manual_seed(seed)
        self.dtype = dtype
        self.k = [self.rows(n, HEADS) for n in lengths]
        self.v = [self.rows(n, HEADS) for n in lengths]

    def rows(self, n, heads):
        return torch.randn(n, heads, DIM, generator=self.g).to(self.dtype)

    def lengths(self):
        return [len(k) for k in self.k]


def expect(seqs, b, q, f, layout, window, cache=None, slots=None):
    """(output, tolerance) [Q_HEADS, DIM] of sequence b's newest token."""
    n = len(seqs.k[b])
    lo = max(0, n - window) if window else 0
    eps = torch.finfo(seqs.dtype).eps
    qr, q_size = turn(q[None], torch.tensor([n - 1]), f, layout)
    if cache is None:
        k, k_size = turn(seqs.k[b], torch.arange(n), f, layout)
        v, moved = seqs.v[b].double(), eps + 2.0 ** -19
    else:
        k, v = (t.cpu().double() for t in kv_cache.cache_read(cache, slots, dtype=torch.float32))
        k_size, moved = k.abs(), eps / 2 + 2.0 ** -19
    k, k_size, v = (t[lo:].transpose(0, 1) for t in (k, k_size, v))
    qr, q_size = (t[0].view(HEADS, -1, DIM) for t in (qr, q_size))
    s = qr @ k.transpose(1, 2) * DIM ** -0.5
    size = (q_size @ k_size.transpose(1, 2) * DIM ** -0.5).amax(-1, keepdim=True)
    w = torch.softmax(s, -1)
    o, a = w @ v, w @ v.abs()
    delta = size * (moved + (DIM + 8) * 2.0 ** -23) + 2.0 ** -22 * s.abs().amax(-1, keepdim=True)
    tol = 2 * a * (delta + (2 * n / 128 + 300) * 2.0 ** -23) + a * 2.0 ** -17 + eps / 2 * o.abs()
    return o.reshape(Q_HEADS, DIM), tol.reshape(Q_HEADS, DIM)


@pytest.mark.parametrize("dtype,cache_type", [
    (torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
    (torch.float16, torch.float16), (torch.bfloat16, torch.float8_e4m3fn),
    (torch.float16, torch.int8), (torch.float32, torch.int8)])
@pytest.mark.parametrize("layout,window", [("half", 0), ("interleaved", 24)])
def test_prefill_and_steps(dtype, cache_type, layout, window):
    prompts = [5, 33, 1, 160]
    seqs = Sequences(prompts, dtype, 21)
    f = rotary.rotary_frequencies(ROTARY, scaling="by_parts", factor=4.0, original_length=32,
                                  device="cuda")
    columns = 13
    cache = PagedCache.allocate(4 * columns + 1, HEADS, PAGE, DIM, dtype=cache_type)
    order = torch.randperm(4 * columns + 1, generator=torch.Generator().manual_seed(2))
    table = order[:4 * columns].view(4, columns).int().cuda()
    # prefill: one padded batch, the padding without slots
    longest = max(prompts)
    k, v = (torch.zeros(4, longest, HEADS, DIM, dtype=dtype) for _ in range(2))
    positions = torch.full((4, longest), -1)
    for b, n in enumerate(prompts):
        k[b, :n], v[b, :n], positions[b, :n] = seqs.k[b], seqs.v[b], torch.arange(n)
    positions = positions.cuda()
    k = rotary.apply_rotary(k.cuda(), None, positions, f, layout=layout)
    slots = kv_cache.cache_slots(table, positions, PAGE)
    kv_cache.cache_write(cache, k.flatten(0, 1), v.cuda().flatten(0, 1), slots.flatten())
    coded = cache_type in kv_cache.CODED_DTYPES
    for step in range(20):
        new = [(seqs.rows(1, Q_HEADS), seqs.rows(1, HEADS), seqs.rows(1, HEADS)) for _ in prompts]
        at = torch.tensor(seqs.lengths())
        q, k, v = (torch.stack([x[i] for x in new]).cuda() for i in range(3))
        for b, (_, kb, vb) in enumerate(new):
            seqs.k[b], seqs.v[b] = torch.cat([seqs.k[b], kb]), torch.cat([seqs.v[b], vb])
        position = at[:, None].cuda()
        rotary.apply_rotary(q, k, position, f, layout=layout, q_out=q, k_out=k)
        slots = kv_cache.cache_slots(table, position, PAGE).flatten()
        kv_cache.cache_write(cache, k[:, 0], v[:, 0], slots)
        lengths = (at + 1).int().cuda()
        out = paged_attention(q[:, 0], cache, table, lengths, window=window)
        if step % 5 in (0, 4):
            for b, n in enumerate(seqs.lengths()):
                all_slots = kv_cache.cache_slots(table[b:b + 1], torch.arange(n)[None].cuda(), PAGE)
                want, tol = expect(seqs, b, new[b][0][0], f, layout, window,
                                   cache if coded else None, all_slots[0])
                gap = (out[b].cpu().double() - want).abs()
                assert (gap <= tol).all(), (step, b, (gap / tol).max().item())


def test_a_captured_step_follows_the_eager_one():
    """One graph of a whole step, replayed as the sequences grow, beside eager
    steps on a cache of its own: every output and the caches equal bit for bit."""
    batch, columns = 5, 40
    f = rotary.rotary_frequencies(DIM, device="cuda")
    table = torch.randperm(batch * columns, generator=torch.Generator().manual_seed(3))
    table = table.view(batch, columns).int().cuda()
    make = lambda: PagedCache.allocate(batch * columns, HEADS, PAGE, DIM,  # noqa: E731
                                       dtype=torch.float8_e4m3fn)
    one, two = make(), make()
    q = torch.zeros(batch, 1, Q_HEADS, DIM, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(batch, 1, HEADS, DIM, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    position = torch.zeros(batch, 1, dtype=torch.int64, device="cuda")

    def step(cache):
        qr, kr = rotary.apply_rotary(q, k, position, f)
        slots = kv_cache.cache_slots(table, position, PAGE).flatten()
        kv_cache.cache_write(cache, kr[:, 0], v[:, 0], slots)
        return paged_attention(qr[:, 0], cache, table, (position[:, 0] + 1).int())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(two)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(one)
    g = torch.Generator(device="cuda").manual_seed(4)
    for rep in range(12):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, device="cuda", generator=g))
        position.copy_(torch.tensor([[37 * rep + b] for b in range(batch)]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step(two)), f"replay {rep}"
    for a, b in ((one.k, two.k), (one.v, two.v)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(one.k_scale, two.k_scale) and torch.equal(one.v_scale, two.v_scale)
