"""Attention over the paged cache without a GPU: the refusals of its C entry and
its workspace's size (nothing here reaches a launch)."""
from __future__ import annotations

import pytest
import torch

from fireprot_amd import _native, kv_cache, paged_attention


@pytest.fixture(scope="module")
def lib():
    if not _native.LIB_PATH.exists():
        from fireprot_amd import build
        build.build()
    return _native.library()


def _args(**override):
    args = dict(dtype=1, cache_dtype=1, q=256, q_sb=1024, q_sh=128, cache_k=512, cache_v=1024,
                k_scale=None, v_scale=None, pages=64, heads=2, page_size=16, head_dim=128,
                block_table=256, table_sb=8, table_pages=8, lengths=256, batch=3, q_heads=8,
                max_length=128, window=0, scale=0.1, out=2048, o_sb=1024, o_sh=128, lse=None,
                workspace=256, workspace_bytes=1 << 30, stream=None)
    assert set(override) <= set(args)
    args.update(override)
    return list(args.values())


@pytest.mark.parametrize("bad", [
    dict(dtype=3), dict(dtype=0), dict(cache_dtype=0), dict(cache_dtype=7), dict(head_dim=96),
    dict(page_size=8), dict(page_size=20), dict(heads=0), dict(q_heads=7), dict(q_heads=1),
    dict(pages=0), dict(batch=-1), dict(batch=1 << 23), dict(batch=1 << 20), dict(max_length=-1),
    dict(max_length=1 << 30, table_pages=1 << 40), dict(window=-1), dict(q_sb=-8), dict(q_sh=124),
    dict(o_sb=1020), dict(o_sh=-128), dict(table_sb=-1), dict(table_pages=7),
    dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=3e38), dict(out=256, o_sh=256)])
def test_sizes_are_refused(lib, bad):
    assert lib.fpx_paged_attention(*_args(**bad)) == _native.FPX_ERR_DIMS


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(q=264), dict(out=None), dict(out=2056), dict(cache_k=None),
    dict(cache_v=520), dict(block_table=None), dict(block_table=258), dict(lengths=None),
    dict(lengths=257), dict(lse=258), dict(workspace=None, max_length=4096, table_pages=256),
    dict(workspace=128, max_length=4096, table_pages=256),
    dict(cache_dtype=3), dict(cache_dtype=4, k_scale=256, v_scale=264)])
def test_pointers_are_refused(lib, bad):
    assert lib.fpx_paged_attention(*_args(**bad)) == _native.FPX_ERR_POINTER


def test_workspace(lib):
    size = lib.fpx_paged_attention_workspace_bytes
    long = dict(max_length=1 << 16, table_pages=1 << 12)
    need = size(1, 3, 8, 2, 128, 1 << 16, 0)
    assert need > 3 * 8 * 2 * (128 + 2) * 4  # at least two shares a row
    assert lib.fpx_paged_attention(*_args(workspace_bytes=need - 1, **long)) \
        == _native.FPX_ERR_WORKSPACE
    assert size(1, 3, 8, 2, 128, 128, 0) == 256
    # a window bounds the work as a length does
    assert size(1, 3, 8, 2, 128, 1 << 16, 64) == 256
    assert size(1, 3, 8, 2, 128, 1 << 16, 1 << 40) == need
    # two places a work-group, whatever the length
    assert size(1, 3, 8, 2, 128, 1 << 24, 0) == size(1, 3, 8, 2, 128, 1 << 20, 0)
    for bad in ((5, 3, 8, 2, 128, 128, 0), (1, -1, 8, 2, 128, 128, 0), (1, 3, 7, 2, 128, 128, 0),
                (1, 3, 8, 2, 100, 128, 0), (1, 3, 8, 2, 128, -1, 0),
                (1, 3, 8, 2, 128, 1 << 30, 0), (1, 3, 8, 2, 128, 128, -1),
                (1, 1 << 18, 8, 2, 128, 128, 0), (1, 3, 0, 0, 128, 128, 0),
                (1, 1 << 17, 8, 8, 128, 1 << 20, 0)):
        assert size(*bad) == 0


def test_empty_batch_launches_nothing(lib):
    assert lib.fpx_paged_attention(*_args(batch=0, q=None)) == 0


def test_cpu_tensors_are_refused(lib):
    cache = kv_cache.PagedCache.allocate(2, 2, 16, 64, dtype=torch.float16, device="cpu")
    with pytest.raises(ValueError, match="HIP device"):
        paged_attention.paged_attention(
            torch.zeros(1, 4, 64, dtype=torch.float16), cache,
            torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32))
