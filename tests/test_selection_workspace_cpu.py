"""Sizes that fpx_select_pages refuses have no workspace, and those that it takes have one."""
from __future__ import annotations

import pytest

from fireprot_amd import _native
from tests.test_kv_cache_cpu import lib  # noqa: F401
from tests.test_page_selection_cpu import _select_args

ROWS = 1 << 20  # (sequence, query head) of a call, at most


@pytest.mark.parametrize("batch,heads,page_size,max_length,count", [
    (ROWS, 64, 16, 1024, 4), (2, ROWS // 2 + 1, 16, 1024, 4), (ROWS, ROWS, 16, 129 * 16, 1),
    (ROWS, ROWS, 16, (1 << 30) - 1, 1),       # (its bytes pass 2^63)
    (1, 65536, 16, 1024, 4), (0, 65536, 16, 1024, 4),  # more heads than a cache has
    (ROWS, 1, 16, (1 << 30) - 1, 1),          # more tiles of pages than a launch has work-groups
    (1, 1, 16, 1024, 1 << 26), (1, 1, 4096, 1024, 1 << 18)])  # 2^30 keys chosen
def test_sizes_that_are_refused_have_none(lib, batch, heads, page_size, max_length,  # noqa: F811
                                          count):
    assert lib.fpx_select_pages_workspace_bytes(batch, heads, page_size, max_length, count) == 0
    columns = -(-max_length // page_size)
    args = dict(batch=batch, heads=heads, q_heads=heads, page_size=page_size,
                max_length=max_length, count=count, sinks=0, table_sb=columns,
                table_pages=columns, workspace_bytes=0)
    assert lib.fpx_select_pages(*_select_args(**args)) == _native.FPX_ERR_DIMS


@pytest.mark.parametrize("batch,heads,page_size,max_length,count,size", [
    (ROWS, 1, 16, 128 * 16, 4, 256), (1 << 14, 64, 16, 129 * 16, 4, (ROWS * 129 * 4)),
    (1, 65535, 16, 64, 4, 256), (1, 1, 16, 1024, (1 << 26) - 1, 256),
    (1, 1, 4096, 1024, (1 << 18) - 1, 256), (1, 1, 16, (1 << 30) - 1, 1, 1 << 28),
    (1 << 10, 1, 16, (1 << 30) - 1, 1, 1 << 38)])
def test_largest_sizes_have_one(lib, batch, heads, page_size, max_length, count,  # noqa: F811
                                size):
    assert lib.fpx_select_pages_workspace_bytes(batch, heads, page_size, max_length, count) == size
