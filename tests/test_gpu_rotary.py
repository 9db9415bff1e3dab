"""Rotary positions on the GPU against the formula in 64 bits.

Tolerance, derived: cos and sin come out within 2^-23 (two units of 2^-24);
the factor, the two products and the sum round once each, 2^-24 of at most
scale (|x1| + |x2|) apiece; together below 2^-21 scale (|x1| + |x2|).  Then one
rounding to the output type, half a step: finfo.eps / 2 of the value (of the
smallest normal number below it).
"""
from __future__ import annotations

import pytest
import torch

from fireprot_amd import rotary

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def reference(x, positions, f, layout, inverse=False):
    """(outputs, |x1| + |x2| of each rotated channel) in float64 on the CPU."""
    return _formula(x.detach().cpu().double(), positions, f, layout, inverse)


def _formula(x, positions, f, layout, inverse=False):
    r = f.rotary_dim
    pos = positions.cpu().double()
    angle = (pos[..., None] * f.inv_freq.cpu())  # [(b,) n, r/2]
    if x.dim() == 4 and angle.dim() == 2:
        angle = angle[None]
    angle = angle.unsqueeze(-2)
    cos, sin = torch.cos(angle) * f.scale, torch.sin(angle) * f.scale
    sin = -sin if inverse else sin
    a, b = ((slice(0, r // 2), slice(r // 2, r)) if layout == "half"
            else (slice(0, r, 2), slice(1, r, 2)))
    y, size = x.clone(), torch.zeros_like(x)
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, size * f.scale


def check(actual, x, positions, f, layout, inverse=False):
    want, size = reference(x, positions, f, layout, inverse)
    info = torch.finfo(actual.dtype)
    got = actual.detach().cpu().double()
    tol = 2.0 ** -21 * size + info.eps / 2 * want.abs().clamp(min=info.tiny)
    worst = ((got - want).abs() - tol).max().item() if got.numel() else 0.0
    assert worst <= 0.0, f"{worst} past the tolerance"
    rest = x[..., f.rotary_dim:]
    assert torch.equal(actual[..., f.rotary_dim:], rest), "the rest of the head is copied"


def randn(shape, dtype, seed=11):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("batch,tokens,q_heads,k_heads,head_dim,rotary_dim", [
    (1, 1, 1, 1, 2, 2), (2, 3, 4, 1, 128, 128), (3, 17, 5, 5, 80, 32), (1, 5, 3, 1, 80, 78),
    (2, 7, 8, 2, 33, 30), (1, 2, 2, 2, 512, 512), (1, 3, 2, 1, 512, 2), (5, 1, 71, 1, 64, 32),
    (1, 4099, 2, 1, 64, 64), (2, 1300, 1, 0, 32, 16)])
def test_against_the_formula(dtype, layout, batch, tokens, q_heads, k_heads, head_dim, rotary_dim):
    print(f"rotary {dtype} {layout} {batch, tokens, q_heads, k_heads, head_dim, rotary_dim}",
          flush=True)
    f = rotary.rotary_frequencies(rotary_dim, scaling="by_parts", factor=4.0,
                                  original_length=64, device="cuda")
    q = randn((batch, tokens, q_heads, head_dim), dtype)
    k = randn((batch, tokens, k_heads, head_dim), dtype, 12) if k_heads else None
    positions = torch.randint(-50, 5000, (batch, tokens),
                              generator=torch.Generator().manual_seed(5)).cuda()
    saved = q.clone()
    out = rotary.apply_rotary(q, k, positions, f, layout=layout)
    torch.cuda.synchronize()
    assert torch.equal(q, saved)
    for x, y in zip((q, k), out if k_heads else (out,)):
        assert y.is_contiguous()
        check(y, x, positions, f, layout)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("positions", [
    torch.tensor([0, 1, 2, 131071, 131072, 1048575], dtype=torch.int32),
    torch.tensor([-1, -131072, 2 ** 31 - 1, 2 ** 31, 2 ** 40 + 1, 7], dtype=torch.int64)])
def test_far_positions(dtype, positions):
    f = rotary.rotary_frequencies(128, device="cuda")
    q = randn((2, 6, 4, 128), dtype)
    out = rotary.apply_rotary(q, None, positions.cuda(), f)
    # the 64-bit angle itself is off by 2^-53 of its size on either side
    far = positions.double().abs().max().item() * 2.0 ** -52
    if far < 2.0 ** -24:
        check(out, q, positions, f, "half")
    else:
        keep = positions.abs() < 2 ** 32
        check(out[:, keep.cuda()], q[:, keep.cuda()], positions[keep], f, "half")
        assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("view", ["fused", "head_first", "channels", "offset1", "broadcast",
                                  "channel_stride"])
def test_strided_inputs(dtype, layout, view):
    b, n, h, d = 2, 9, 4, 64
    if view == "fused":
        x = randn((b, n, 3 * h * d), dtype)[..., h * d:2 * h * d].view(b, n, h, d)
    elif view == "head_first":
        x = randn((b, h, n, d), dtype).transpose(1, 2)
    elif view == "channels":
        x = randn((b, n, h, d + 24), dtype)[..., 24:]
    elif view == "offset1":
        x = randn((b * n * h * d + 1,), dtype)[1:].view(b, n, h, d)
    elif view == "broadcast":
        x = randn((b, n, 1, d), dtype).expand(b, n, h, d)
    else:
        x = randn((b, n, h, d, 2), dtype)[..., 1]
    f = rotary.rotary_frequencies(48, device="cuda")
    positions = torch.arange(n).cuda() * 3  # one vector for every sequence
    q, k = rotary.apply_rotary(x, x[:, :, :3], positions, f, layout=layout)
    torch.cuda.synchronize()
    check(q, x, positions, f, layout)
    check(k, x[:, :, :3], positions, f, layout)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_in_place_and_given_outputs(dtype, layout):
    f = rotary.rotary_frequencies(32, device="cuda")
    buffer = randn((3, 6, 10, 72), dtype)
    saved = buffer.clone()
    q, k = buffer[:, :, 1:5, :64], buffer[:, :, 5:7, :64]
    positions = torch.arange(18, dtype=torch.int32).view(3, 6).cuda()
    want_q, want_k = rotary.apply_rotary(q, k, positions, f, layout=layout)
    wide_q, wide_k = torch.full_like(buffer, 7.0), torch.full_like(buffer, 7.0)
    rotary.apply_rotary(q, k, positions, f, layout=layout, q_out=wide_q[:, :, 1:5, :64],
                        k_out=wide_k[:, :, 5:7, :64])
    got = rotary.apply_rotary(q, k, positions, f, layout=layout, q_out=q, k_out=k)
    torch.cuda.synchronize()
    assert got[0] is q and got[1] is k
    for y, w, want, lo, hi in ((q, wide_q, want_q, 1, 5), (k, wide_k, want_k, 5, 7)):
        assert torch.equal(y, want) and torch.equal(w[:, :, lo:hi, :64], want)
        w[:, :, lo:hi, :64] = 7.0
        assert (w == 7.0).all(), "nothing beside the given outputs is written"
    buffer[:, :, 1:7, :64] = saved[:, :, 1:7, :64]
    assert torch.equal(buffer, saved)


def test_offsets_past_32_bits():
    pitch = 2 ** 31 + 64  # elements between two tokens
    buffer = torch.empty(pitch + 256, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(buffer, (1, 2, 2, 128), (0, pitch, 128, 1))
    x.copy_(randn((1, 2, 2, 128), torch.bfloat16))
    f = rotary.rotary_frequencies(128, device="cuda")
    positions = torch.tensor([3, 9]).cuda()
    saved = x.clone()
    out = rotary.apply_rotary(x, None, positions, f)
    check(out, saved, positions, f, "half")
    rotary.apply_rotary(x, None, positions, f, q_out=x)
    torch.cuda.synchronize()
    assert torch.equal(x, out)


def test_empty_calls():
    f = rotary.rotary_frequencies(32, device="cuda")
    q, k = rotary.apply_rotary(randn((2, 0, 4, 32), torch.float32),
                               randn((2, 0, 1, 32), torch.float32),
                               torch.zeros(2, 0, dtype=torch.int64).cuda(), f)
    assert q.shape == (2, 0, 4, 32) and k.shape == (2, 0, 1, 32)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_nonfinite_values_stay_in_their_pairs(layout):
    f = rotary.rotary_frequencies(64, device="cuda")
    q = randn((1, 4, 2, 80), torch.float32)
    q[0, 1, 0, 3], q[0, 2, 1, 70] = float("nan"), float("inf")
    out = rotary.apply_rotary(q, None, torch.arange(4).cuda(), f, layout=layout)
    bad = ~torch.isfinite(out.cpu())
    want = torch.zeros_like(bad)
    want[0, 1, 0, 3] = want[0, 1, 0, 35 if layout == "half" else 2] = want[0, 2, 1, 70] = True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradients(dtype, layout):
    f = rotary.rotary_frequencies(48, scaling="by_parts", factor=8.0, original_length=32,
                                  device="cuda")
    positions = (torch.arange(15).view(3, 5) * 17).cuda()
    gq = randn((3, 5, 6, 64), dtype, 4)
    gk = randn((3, 5, 1, 64), dtype, 5).expand(3, 5, 2, 64)  # the gradient of a sum, say
    dq, dk = rotary.rotary_backward(gq, gk, positions, f, layout=layout)
    check(dq, gq, positions, f, layout, inverse=True)
    check(dk, gk, positions, f, layout, inverse=True)
    # the formula's gradient by autograd in 64 bits, shared by the heads of a
    # broadcast input
    x = torch.randn(3, 5, 1, 64, dtype=torch.float64, requires_grad=True)
    y, _ = _formula(x.expand(3, 5, 6, 64), positions, f, layout)
    (want,) = torch.autograd.grad(y, x, gq.cpu().double())
    got = dq.cpu().double().sum(2, keepdim=True)
    size = reference(gq, positions, f, layout, True)[1].sum(2, keepdim=True)
    tol = 6 * 2.0 ** -21 * size + torch.finfo(dtype).eps / 2 * dq.cpu().double().abs().sum(
        2, keepdim=True) + 1e-12
    assert ((got - want).abs() <= tol).all()


def test_gradient_against_differences():
    f = rotary.rotary_frequencies(32, device="cuda")
    positions = torch.tensor([5, 900, 70000]).cuda()
    q, g, d = (randn((1, 3, 2, 40), torch.float32, seed) for seed in (1, 2, 3))
    dq = rotary.rotary_backward(g, None, positions, f)
    h = 0.5  # the map is linear: any step is exact but for rounding
    up = rotary.apply_rotary(q + h * d, None, positions, f).double()
    down = rotary.apply_rotary(q - h * d, None, positions, f).double()
    slope = ((up - down) * g.double()).sum() / (2 * h)
    # each output is off by at most 2^-21 (|x1| + |x2|) + 2^-24 |y| (inputs q +- h d
    # rounded once more, 2^-24), on both sides of the quotient and in dq
    size = (q.abs() + d.abs()).double().flatten()
    bound = 4 * 2.0 ** -20 * size.sum() * g.abs().max().double()
    assert abs(slope - (dq.double() * d.double()).sum()) <= bound


def test_refusals_on_the_device():
    f = rotary.rotary_frequencies(32, device="cuda")
    q = randn((2, 3, 4, 32), torch.float32)
    p = torch.arange(3).cuda()
    for bad in (lambda: rotary.apply_rotary(q.double(), None, p, f),
                lambda: rotary.apply_rotary(q, q.half(), p, f),
                lambda: rotary.apply_rotary(q, q[:1], p, f),
                lambda: rotary.apply_rotary(q, None, p.float(), f),
                lambda: rotary.apply_rotary(q, None, p[:2], f),
                lambda: rotary.apply_rotary(q, None, p.cpu(), f),
                lambda: rotary.apply_rotary(q[..., :16], None, p, f),
                lambda: rotary.apply_rotary(q[0, 0], None, p, f),
                lambda: rotary.apply_rotary(q, None, p, f.to("cpu")),
                lambda: rotary.apply_rotary(q, None, p, f, q_out=q[:1]),
                lambda: rotary.apply_rotary(q, None, p, f, q_out=q[:, :, :1].expand_as(q)),
                lambda: rotary.apply_rotary(q.clone().requires_grad_(), None, p, f),
                lambda: rotary.apply_rotary(q, None, p, f, q_out=q.clone().requires_grad_()),
                lambda: rotary.apply_rotary(q, q, p, f, q_out=q, k_out=q),
                lambda: rotary.rotary_backward(q, q.clone().requires_grad_(), p, f)):
        with pytest.raises(ValueError):
            bad()
    with torch.no_grad():
        rotary.apply_rotary(q.clone().requires_grad_(), None, p, f)


def test_other_stream_and_graph():
    f = rotary.rotary_frequencies(64, device="cuda")
    q, k = randn((4, 8, 6, 64), torch.bfloat16), randn((4, 8, 2, 64), torch.bfloat16, 2)
    positions = torch.arange(32).view(4, 8).cuda()
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rotary.apply_rotary(q, k, positions, f, q_out=qo, k_out=ko)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    want = rotary.apply_rotary(q, k, positions, f)
    assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rotary.apply_rotary(q, k, positions, f, q_out=qo, k_out=ko)
        back = rotary.rotary_backward(qo, ko, positions, f)
    for rep in range(4):
        q.copy_(randn(q.shape, torch.bfloat16, 50 + rep))
        positions += 11
        graph.replay()
        torch.cuda.synchronize()
        want = rotary.apply_rotary(q, k, positions, f)
        wback = rotary.rotary_backward(*want, positions, f)
        assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])
        assert torch.equal(back[0], wback[0]) and torch.equal(back[1], wback[1])


@pytest.mark.parametrize("dtype,layout", [(torch.bfloat16, "half"), (torch.float32, "interleaved")])
def test_large_calls_equal_small_ones(dtype, layout):
    """Rows of 64 MB and more are loaded past the caches, several tokens to a
    work-group: the same bits as call by call."""
    tokens, heads, dim = (64 << 20) // (20 * 128 * dtype.itemsize) + 7, 16, 128
    f = rotary.rotary_frequencies(96, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(8)
    q = torch.randn(tokens, heads, dim, device="cuda", generator=g).to(dtype)
    k = torch.randn(tokens, 4, dim, device="cuda", generator=g).to(dtype)
    positions = torch.arange(tokens, device="cuda") * 3
    whole = rotary.apply_rotary(q, k, positions, f, layout=layout)
    for lo in (0, 1000, tokens - 300):
        part = slice(lo, lo + 300)
        small = rotary.apply_rotary(q[part], k[part], positions[part], f, layout=layout)
        assert torch.equal(whole[0][part], small[0]) and torch.equal(whole[1][part], small[1])
    check(whole[0][-5:], q[-5:], positions[-5:], f, layout)


def test_many_heads_and_units():
    """The most heads, and rows of more vectors than a work-group has threads."""
    f = rotary.rotary_frequencies(2, device="cuda")
    q, k = randn((1, 2, 8191, 6), torch.bfloat16), randn((1, 2, 1, 6), torch.bfloat16, 2)
    positions = torch.tensor([1, 77]).cuda()
    out = rotary.apply_rotary(q, k, positions, f)
    check(out[0], q, positions, f, "half")
    check(out[1], k, positions, f, "half")
    wide = randn((1, 3, 8, 513), torch.float16)[..., 1:]  # 512 channels, one element a vector
    out = rotary.apply_rotary(wide, None, positions.new_tensor([0, 5, 9]), f)
    check(out, wide, positions.new_tensor([0, 5, 9]), f, "half")


def test_more_tokens_than_one_launch():
    """2^22 groups of 16 tokens and more: a second launch."""
    tokens = 2 ** 26 + 35
    f = rotary.rotary_frequencies(2, device="cuda")
    q = torch.ones(tokens, 1, 2, device="cuda", dtype=torch.bfloat16)
    positions = torch.arange(tokens, device="cuda", dtype=torch.int32) % 1000
    out = rotary.apply_rotary(q, None, positions, f)
    for part in (slice(0, 2000), slice(2 ** 26 - 1000, tokens)):
        assert torch.equal(out[part], rotary.apply_rotary(q[part], None, positions[part], f))
    check(out[-300:], q[-300:], positions[-300:], f, "half")
