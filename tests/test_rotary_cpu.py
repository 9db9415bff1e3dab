"""Rotary positions without a GPU: the frequencies' formulas and the refusals
of the C entry and of the Python one (nothing here reaches a launch)."""
from __future__ import annotations

import math

import pytest
import torch

from fireprot_amd import _native, rotary


@pytest.fixture(scope="module")
def lib():
    if not _native.LIB_PATH.exists():
        from fireprot_amd import build
        build.build()
    return _native.library()


def _args(**override):
    args = dict(dtype=0, layout=0, q=256, q_sb=1024, q_sn=128, q_sh=32, q_out=512, qo_sb=1024,
                qo_sn=128, qo_sh=32, q_heads=4, k=256, k_sb=1024, k_sn=128, k_sh=32, k_out=512,
                ko_sb=1024, ko_sn=128, ko_sh=32, k_heads=4, positions=256, positions_64=1, p_sb=8,
                p_sn=1, inv_freq=256, scale=1.0, inverse=0, batch=2, tokens=8, head_dim=32,
                rotary_dim=32, stream=None)
    assert set(override) <= set(args)
    args.update(override)
    return list(args.values())


@pytest.mark.parametrize("bad", [
    dict(dtype=3), dict(dtype=-1), dict(layout=2), dict(positions_64=2), dict(inverse=2),
    dict(head_dim=0), dict(head_dim=513), dict(rotary_dim=0), dict(rotary_dim=33),
    dict(rotary_dim=34), dict(q_heads=0), dict(k_heads=-1), dict(q_heads=8000, k_heads=193),
    dict(batch=-1), dict(tokens=-1), dict(batch=1 << 16, tokens=1 << 15),
    dict(batch=1 << 40, tokens=1 << 40), dict(q_sn=-128), dict(qo_sh=-32), dict(k_sb=-1),
    dict(ko_sn=-1), dict(p_sn=-1), dict(q_out=256, qo_sn=64), dict(k_out=256, ko_sn=64),
])
def test_sizes_are_refused(lib, bad):
    assert lib.fpx_rotary(*_args(**bad)) == _native.FPX_ERR_DIMS


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(q_out=None), dict(k=None), dict(k_out=None), dict(positions=None),
    dict(inv_freq=None), dict(q=258), dict(q_out=514), dict(positions=260), dict(inv_freq=260),
    dict(dtype=2, k=257), dict(positions_64=0, positions=258),
])
def test_pointers_are_refused(lib, bad):
    assert lib.fpx_rotary(*_args(**bad)) == _native.FPX_ERR_POINTER


def test_empty_calls_launch_nothing(lib):
    assert lib.fpx_rotary(*_args(batch=0)) == 0
    assert lib.fpx_rotary(*_args(tokens=0, q=None)) == 0


def test_frequencies_follow_their_formulas():
    r, base, factor, trained = 64, 10000.0, 8.0, 2048
    plain = [base ** (-2 * i / r) for i in range(r // 2)]

    def check(f, want, scale=1.0):
        assert f.inv_freq.dtype == torch.float64 and f.rotary_dim == r
        assert f.scale == pytest.approx(scale, rel=1e-15)
        torch.testing.assert_close(f.inv_freq, torch.tensor(want, dtype=torch.float64),
                                   rtol=1e-13, atol=0.0)

    check(rotary.rotary_frequencies(r), plain)
    check(rotary.rotary_frequencies(r, scaling="linear", factor=factor),
          [f / factor for f in plain])
    ntk = rotary.rotary_frequencies(r, scaling="ntk", factor=factor)
    check(ntk, [(base * factor ** (r / (r - 2))) ** (-2 * i / r) for i in range(r // 2)])
    # the slowest pair is interpolated by the factor, the fastest is kept
    assert ntk.inv_freq[0] == 1.0
    assert ntk.inv_freq[-1].item() == pytest.approx(plain[-1] / factor, rel=1e-12)
    parts = []
    for f in plain:
        turns = trained * f / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - 1.0) / 31.0))
        parts.append(f * keep + f / factor * (1 - keep))
    check(rotary.rotary_frequencies(r, scaling="by_parts", factor=factor, original_length=trained),
          parts, scale=0.1 * math.log(factor) + 1.0)
    assert rotary.rotary_frequencies(r, scaling="by_parts", factor=factor, scale=1.0,
                                     original_length=trained).scale == 1.0
    assert rotary.rotary_frequencies(2, scaling="ntk", factor=4.0).inv_freq.tolist() == [1.0]


@pytest.mark.parametrize("bad", [
    dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=8, scaling="cubic"),
    dict(rotary_dim=8, base=0.0), dict(rotary_dim=8, scaling="linear", factor=0.5),
    dict(rotary_dim=8, factor=2.0), dict(rotary_dim=8, scaling="by_parts", factor=2.0),
    dict(rotary_dim=8, scaling="by_parts", factor=2.0, original_length=64, slow=4.0, fast=4.0),
    dict(rotary_dim=8, scaling="linear", factor=float("nan")),
])
def test_frequencies_refuse(bad):
    with pytest.raises(ValueError):
        rotary.rotary_frequencies(**bad)


@pytest.mark.parametrize("inv_freq", [
    torch.ones(4), torch.ones(2, 2, dtype=torch.float64), torch.ones(0, dtype=torch.float64),
    torch.ones(8, dtype=torch.float64)[::2],
    torch.ones(8, dtype=torch.float64, requires_grad=True)])
def test_given_frequencies_are_checked(inv_freq):
    with pytest.raises(ValueError, match="inv_freq"):
        rotary.RotaryFrequencies(inv_freq)


def test_cpu_tensors_are_refused(lib):
    q = torch.zeros(1, 2, 4, 32)
    with pytest.raises(ValueError, match="HIP device"):
        rotary.apply_rotary(q, None, torch.arange(2), rotary.rotary_frequencies(32))
    with pytest.raises(ValueError, match="layout"):
        rotary.apply_rotary(q, None, torch.arange(2), rotary.rotary_frequencies(32), layout="x")
