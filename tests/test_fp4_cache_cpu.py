"""The 4-bit cache without a GPU: its shapes, its refusals, the entries' checks."""
from __future__ import annotations

import pytest
import torch

from tests import fp4
from fireprot_amd import _native, kv_cache
from fireprot_amd.kv_cache import FP4, PagedCache
from tests.test_kv_cache_cpu import _args, lib  # noqa: F401

E8M0 = torch.float8_e8m0fnu
FOUR = dict(cache_dtype=_native.FPX_F4E2M1)


def test_the_definition_used_by_the_tests():
    x = torch.zeros(3, 32)
    x[0, :4] = torch.tensor([7.0, -0.75, 0.25, 2.5])
    x[1, 0], x[1, 1] = 7.0001, -7.0001
    x[2, 5] = float("nan")
    codes, scales = fp4.quantise(x)
    assert scales.flatten().tolist() == [127, 128, 255]
    assert codes[0, :2].tolist() == [0x7 | 0xA << 4, 0x0 | 0x4 << 4]
    got = fp4.values(codes, scales)
    assert got[0, :4].tolist() == [6.0, -1.0, 0.0, 2.0]
    assert got[1, :2].tolist() == [8.0, -8.0]
    assert torch.isnan(got[2]).all()


@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_shapes(dim):
    cache = PagedCache.allocate(5, 3, 16, dim, dtype=FP4, device="cpu")
    assert (cache.pages, cache.heads, cache.page_size, cache.head_dim) == (5, 3, 16, dim)
    assert cache.dtype == FP4 and cache.k.shape == (5, 3, 16, dim // 2)
    assert cache.k_scale.shape == (5, 3, 16, dim // 32) and cache.k_scale.dtype == E8M0


def test_tensors_are_checked():
    good = PagedCache.allocate(2, 3, 16, 64, dtype=FP4, device="cpu")
    bytes_ = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    scale = bytes_(2, 3, 16, 2).view(E8M0)
    for k_scale in (None, torch.zeros(2, 3, 16), bytes_(2, 3, 16, 2), bytes_(2, 3, 16, 4).view(E8M0),
                    bytes_(2, 3, 16).view(E8M0)):
        with pytest.raises(ValueError):
            PagedCache(good.k, good.v, k_scale, scale)
    with pytest.raises(ValueError):  # bytes are no codes
        PagedCache(good.k.view(torch.uint8), good.v.view(torch.uint8), good.k_scale, good.v_scale)
    with pytest.raises(ValueError):  # 48 channels
        k = bytes_(2, 3, 16, 24).view(FP4)
        PagedCache(k, k.clone(), scale, good.v_scale)
    with pytest.raises(ValueError):
        PagedCache(good.k, good.v, good.k_scale, good.k_scale)
    with pytest.raises(ValueError):
        PagedCache.allocate(1, 1, 16, 16, dtype=FP4, device="cpu")
    with pytest.raises(ValueError):  # an 8-bit cache's scales
        PagedCache(*(torch.zeros(2, 3, 16, 64, dtype=torch.int8) for _ in range(2)), scale, scale)


@pytest.mark.parametrize("entry", ["fpx_cache_write", "fpx_cache_read"])
def test_entries_check_a_cache_in_4_bits(lib, entry):  # noqa: F811
    call = getattr(lib, entry)
    for bad in (dict(k_scale=None), dict(v_scale=None), dict(k_scale=260), dict(cache_k=520),
                dict(cache_v=None)):
        assert call(*_args(**FOUR, **bad)) == _native.FPX_ERR_POINTER
    for bad in (dict(head_dim=16), dict(head_dim=80), dict(page_size=8), dict(row_dtype=6)):
        assert call(*_args(**FOUR, **bad)) == _native.FPX_ERR_DIMS
    # 4 pages of 4 heads of 16 rows: 64 bytes of codes, 4 of scales each
    mb = 1 << 20
    apart = dict(k=mb, v=2 * mb, slots=3 * mb, cache_k=4 * mb, cache_v=5 * mb, k_scale=6 * mb,
                 v_scale=7 * mb, tokens=8)
    for meets in (dict(k=4 * mb + 256 * 64 - 16), dict(k_scale=2 * mb + 16), dict(v=7 * mb + 1008)):
        assert call(*_args(**FOUR, **{**apart, **meets})) == _native.FPX_ERR_DIMS
    if entry == "fpx_cache_write":
        for meets in (dict(cache_v=4 * mb + 256 * 64 - 16), dict(v_scale=6 * mb + 1008),
                      dict(slots=6 * mb + 1016)):
            assert call(*_args(**FOUR, **{**apart, **meets})) == _native.FPX_ERR_DIMS


def test_attention_over_4_bits_is_planned(lib):  # noqa: F811
    size = lib.fpx_paged_attention_workspace_bytes
    assert size(_native.FPX_F4E2M1, 2, 8, 2, 128, 100, 0) == 256  # no parts
    assert size(_native.FPX_F4E2M1, 2, 8, 2, 128, 5000, 0) > 256
    assert size(_native.FPX_F4E2M1, 2, 8, 2, 48, 100, 0) == 0
    assert size(5, 2, 8, 2, 128, 100, 0) == 0
