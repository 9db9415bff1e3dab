"""The paged cache without a GPU: the refusals of its C entries and of its
Python side, and the slots of positions (nothing here reaches a launch)."""
from __future__ import annotations

import pytest
import torch

from fireprot_amd import _native, kv_cache


@pytest.fixture(scope="module")
def lib():
    if not _native.LIB_PATH.exists():
        from fireprot_amd import build
        build.build()
    return _native.library()


def _args(**override):
    args = dict(row_dtype=1, cache_dtype=3, k=256, k_st=512, k_sh=128, v=256, v_st=512, v_sh=128,
                slots=256, tokens=8, cache_k=512, cache_v=1024, k_scale=256, v_scale=256, pages=4,
                heads=4, page_size=16, head_dim=128, stream=None)
    assert set(override) <= set(args)
    args.update(override)
    return list(args.values())


@pytest.mark.parametrize("entry", ["fpx_cache_write", "fpx_cache_read"])
@pytest.mark.parametrize("bad", [
    dict(row_dtype=3), dict(row_dtype=-1), dict(cache_dtype=5), dict(cache_dtype=-1),
    dict(head_dim=80), dict(head_dim=0), dict(head_dim=512), dict(page_size=8),
    dict(page_size=24), dict(page_size=8192), dict(page_size=0), dict(heads=0), dict(heads=-4),
    dict(pages=0), dict(pages=1 << 31), dict(tokens=-1), dict(tokens=1 << 29, heads=4),
    dict(tokens=1 << 62), dict(k_st=-1), dict(k_sh=-1), dict(v_st=-1), dict(v_sh=-1)])
def test_sizes_are_refused(lib, entry, bad):
    assert getattr(lib, entry)(*_args(**bad)) == _native.FPX_ERR_DIMS


@pytest.mark.parametrize("entry", ["fpx_cache_write", "fpx_cache_read"])
@pytest.mark.parametrize("bad", [
    dict(k=None), dict(v=None), dict(slots=None), dict(cache_k=None), dict(cache_v=None),
    dict(k_scale=None), dict(v_scale=None), dict(k=257), dict(row_dtype=0, v=258),
    dict(slots=260), dict(cache_k=520), dict(cache_v=1025), dict(k_scale=260)])
def test_pointers_are_refused(lib, entry, bad):
    assert getattr(lib, entry)(*_args(**bad)) == _native.FPX_ERR_POINTER


def test_empty_calls_launch_nothing(lib):
    assert lib.fpx_cache_write(*_args(tokens=0, k=None)) == 0
    assert lib.fpx_cache_read(*_args(tokens=0, k=None)) == 0


def test_cache_tensors_are_checked():
    def make(shape=(2, 3, 16, 64), dtype=torch.float16, **kw):
        return kv_cache.PagedCache.allocate(*shape, dtype=dtype, device="cpu", **kw)

    cache = make()
    assert (cache.pages, cache.heads, cache.page_size, cache.head_dim) == (2, 3, 16, 64)
    assert cache.k_scale is None
    coded = make(dtype=torch.int8)
    assert coded.k_scale.shape == (2, 3, 16)
    for bad in (dict(shape=(0, 3, 16, 64)), dict(shape=(2, 0, 16, 64)), dict(shape=(2, 3, 8, 64)),
                dict(shape=(2, 3, 48, 64)), dict(shape=(2, 3, 16, 48)),
                dict(dtype=torch.float64)):
        with pytest.raises(ValueError):
            make(**bad)
    k, s = cache.k, coded.k_scale
    for args in ((k, k[:1]), (k, k.float()), (k[0], k[0]), (k, cache.v, s, s), (k, k),
                 (k, k.view(2, 3, 16, 64)), (k.clone().requires_grad_(), cache.v),
                 (k, cache.v.clone().requires_grad_()), (coded.k, coded.v),
                 (coded.k, coded.v, s, None), (coded.k, coded.v, s, s.double()),
                 (coded.k, coded.v, s, s[:1]), (k.transpose(0, 1), k.transpose(0, 1)),
                 (torch.zeros(2 * 3 * 16 * 64 + 1, dtype=torch.float16)[1:].view(2, 3, 16, 64),
                  k)):
        with pytest.raises(ValueError):
            kv_cache.PagedCache(*args)


def test_calls_on_the_cpu_are_refused(lib):
    cache = kv_cache.PagedCache.allocate(2, 3, 16, 64, dtype=torch.float16, device="cpu")
    rows = torch.zeros(4, 3, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="HIP device"):
        kv_cache.cache_write(cache, rows, rows, torch.arange(4))
    with pytest.raises(ValueError, match="HIP device"):
        kv_cache.cache_read(cache, torch.arange(4))


def test_slots_of_positions():
    table = torch.tensor([[3, 1], [0, 2]], dtype=torch.int32)
    positions = torch.tensor([[0, 15, 16, 31], [-1, 17, 32, 5]])
    top = torch.iinfo(torch.int64).max
    assert kv_cache.cache_slots(table, positions, 16).tolist() == [
        [48, 63, 16, 31], [-1, 33, top, 5]]
    assert kv_cache.cache_slots(table[:, :0], positions, 16).tolist() == [
        [top] * 4, [-1, top, top, top]]
    for bad in ((table[0], positions, 16), (table, positions[0], 16), (table, positions[:1], 16),
                (table, positions, 10)):
        with pytest.raises(ValueError):
            kv_cache.cache_slots(*bad)
