"""Page bounds and their selection without a GPU: what the entries refuse, and the
checks of the Python side."""
from __future__ import annotations

import pytest
import torch

from fireprot_amd import _native
from fireprot_amd.kv_cache import FP4, PagedCache
from fireprot_amd.page_selection import PageBounds
from tests.test_kv_cache_cpu import lib  # noqa: F401

MB = 1 << 20


def _bounds_args(**override):
    args = dict(cache_dtype=3, cache_k=MB, k_scale=2 * MB, pages=40, heads=2, page_size=16,
                head_dim=128, block_table=3 * MB, table_sb=9, table_pages=9, lengths=4 * MB, batch=3,
                max_length=144, fresh=1, bounds=5 * MB, stream=None)
    assert set(override) <= set(args)
    args.update(override)
    return list(args.values())


def _select_args(**override):
    args = dict(dtype=1, bounds_dtype=1, q=MB, q_sb=1024, q_sh=128, q_heads=8, bounds=2 * MB,
                pages=40, heads=2, page_size=16, head_dim=128, block_table=3 * MB,
                table_sb=300, table_pages=300, lengths=4 * MB, batch=3, max_length=4800, count=4, sinks=1, recent=1,
                index=5 * MB, table_out=6 * MB, lengths_out=7 * MB, workspace=8 * MB,
                workspace_bytes=1 << 16, stream=None)
    assert set(override) <= set(args)
    args.update(override)
    return list(args.values())


@pytest.mark.parametrize("bad", [
    dict(cache_dtype=5), dict(pages=0), dict(heads=0), dict(page_size=20), dict(head_dim=96),
    dict(batch=-1), dict(batch=(1 << 20) + 1), dict(max_length=-1), dict(max_length=1 << 30),
    dict(max_length=145), dict(table_sb=-1), dict(fresh=0),
    dict(batch=1 << 20, heads=4096, fresh=1 << 30),
    dict(bounds=MB), dict(bounds=2 * MB + 16), dict(bounds=3 * MB), dict(bounds=4 * MB - 64)])
def test_bounds_sizes_are_refused(lib, bad):  # noqa: F811
    assert lib.fpx_page_bounds(*_bounds_args(**bad)) == _native.FPX_ERR_DIMS


@pytest.mark.parametrize("bad", [
    dict(cache_k=None), dict(cache_k=MB + 8), dict(k_scale=None), dict(block_table=None),
    dict(lengths=4 * MB + 2), dict(bounds=None), dict(bounds=5 * MB + 8)])
def test_bounds_pointers_are_refused(lib, bad):  # noqa: F811
    assert lib.fpx_page_bounds(*_bounds_args(**bad)) == _native.FPX_ERR_POINTER


@pytest.mark.parametrize("bad", [
    dict(dtype=3), dict(bounds_dtype=4), dict(bounds_dtype=6), dict(q_heads=7), dict(q_heads=0),
    dict(q_sb=-8), dict(q_sh=132), dict(heads=0), dict(page_size=20), dict(head_dim=96),
    dict(batch=-1), dict(batch=1 << 18), dict(max_length=4801), dict(max_length=1 << 30),
    dict(count=0), dict(count=1), dict(sinks=-1), dict(recent=0), dict(sinks=3, recent=2),
    dict(count=1 << 26), dict(table_sb=-1), dict(table_pages=299),
    dict(index=MB), dict(index=2 * MB), dict(table_out=3 * MB), dict(lengths_out=4 * MB),
    dict(table_out=5 * MB + 92), dict(lengths_out=6 * MB), dict(workspace=MB + 1024),
    dict(workspace=7 * MB), dict(index=8 * MB + 212)])
def test_selection_sizes_are_refused(lib, bad):  # noqa: F811
    assert lib.fpx_select_pages(*_select_args(**bad)) == _native.FPX_ERR_DIMS


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(q=MB + 8), dict(bounds=None), dict(block_table=None), dict(lengths=None),
    dict(index=None), dict(table_out=5 * MB + 2), dict(lengths_out=None), dict(workspace=None),
    dict(workspace=8 * MB + 128)])
def test_selection_pointers_are_refused(lib, bad):  # noqa: F811
    assert lib.fpx_select_pages(*_select_args(**bad)) == _native.FPX_ERR_POINTER


def test_workspaces(lib):  # noqa: F811
    size = lib.fpx_select_pages_workspace_bytes
    assert size(1, 1, 16, 129 * 16, 4) == 1024  # 129 ranks, rounded up
    assert size(3, 2, 16, 128 * 16, 4) == 256   # few pages: none
    assert size(100, 2, 16, 4800, 300) == 256 and size(100, 2, 16, 4801, 301) == 256
    assert size(100, 2, 16, 4801, 300) == -(-200 * 301 * 4 // 512) * 512
    for bad in ((-1, 2, 16, 144, 4), (3, 0, 16, 144, 4), (3, 2, 24, 144, 4), (3, 2, 16, -1, 4),
                (3, 2, 16, 1 << 30, 4), (3, 2, 16, 144, 0)):
        assert size(*bad) == 0
    short = dict(batch=100, index=5 * MB, count=4, workspace_bytes=200 * 300 * 4 - 1)
    assert lib.fpx_select_pages(*_select_args(**short)) == _native.FPX_ERR_WORKSPACE


def test_empty_calls_launch_nothing(lib):  # noqa: F811
    assert lib.fpx_page_bounds(*_bounds_args(batch=0, bounds=None)) == 0
    assert lib.fpx_page_bounds(*_bounds_args(max_length=0, bounds=None)) == 0
    assert lib.fpx_select_pages(*_select_args(batch=0, q=None)) == 0


def test_lists_for_each_head_are_checked(lib):  # noqa: F811
    args = dict(dtype=1, cache_dtype=1, q=MB, q_sb=1024, q_sh=128, cache_k=2 * MB, cache_v=4 * MB,
                k_scale=None, v_scale=None, pages=40, heads=2, page_size=16, head_dim=128,
                block_table=6 * MB, table_sb=18, table_sh=9, table_pages=9, lengths=7 * MB, batch=3,
                q_heads=8, max_length=144, scale=1.0, out=8 * MB, o_sb=1024, o_sh=128, lse=9 * MB,
                workspace=None, workspace_bytes=0, stream=None)

    def call(**override):
        return lib.fpx_paged_attention_lists(*{**args, **override}.values())

    for bad in (dict(table_sh=-1), dict(table_pages=8), dict(q_heads=7), dict(dtype=0),
                dict(out=6 * MB - 6000), dict(lse=6 * MB + 4 * 50)):
        assert call(**bad) == _native.FPX_ERR_DIMS
    assert call(lse=6 * MB + 4 * 54, block_table=None) == _native.FPX_ERR_POINTER
    assert call(batch=0) == 0


def test_bounds_are_checked():
    cache = PagedCache.allocate(3, 2, 16, 64, dtype=FP4, device="cpu")
    bounds = PageBounds.allocate(cache)
    assert bounds.values.shape == (3, 2, 2, 64) and bounds.values.dtype == torch.bfloat16
    assert bounds.page_size == 16
    plain = PageBounds.allocate(PagedCache.allocate(3, 2, 16, 64, dtype=torch.float16, device="cpu"))
    assert plain.values.dtype == torch.float16
    t = torch.zeros(3, 2, 2, 64)
    for bad in ((t[:, :, :1], 16), (t[..., :48], 16), (t.double(), 16), (t, 24), (t[0], 16),
                (t[:, :, :, :32], 16), (t.clone().requires_grad_(), 16), (t[:0], 16),
                (torch.zeros(3 * 2 * 2 * 64 + 1)[1:].view(3, 2, 2, 64), 16)):
        with pytest.raises(ValueError):
            PageBounds(*bad)
