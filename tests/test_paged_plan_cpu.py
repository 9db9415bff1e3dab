"""How the attention over the paged cache cuts its work, seen through the size of
its workspace (host arithmetic only): NO_WORKSPACE where every row is one unit of
one work-group, places for two shares a work-group otherwise."""
from __future__ import annotations

import pytest

from fireprot_amd import _native
from fireprot_amd.paged_attention import NO_WORKSPACE


@pytest.fixture(scope="module")
def size():
    if not _native.LIB_PATH.exists():
        from fireprot_amd import build
        build.build()
    entry = _native.library().fpx_paged_attention_workspace_bytes

    def workspace(cache_dtype, batch, q_heads, heads, head_dim, max_length, window=0):
        return entry(cache_dtype, batch, q_heads, heads, head_dim, max_length, window)
    return workspace


@pytest.mark.parametrize("cache_dtype", [_native.FPX_F32, _native.FPX_BF16, _native.FPX_F16,
                                         _native.FPX_F8E4M3, _native.FPX_I8])
def test_rows_of_one_unit_need_no_workspace(size, cache_dtype):
    # 2560 rows of at most a unit's 512 keys, and one key more
    assert size(cache_dtype, 40, 64, 64, 32, 512) == NO_WORKSPACE
    assert size(cache_dtype, 40, 64, 64, 32, 513) > NO_WORKSPACE
    # a window of w keys spans w + 31 of those that begin at a multiple of 32
    assert size(cache_dtype, 40, 64, 64, 32, 1 << 20, 481) == NO_WORKSPACE
    assert size(cache_dtype, 40, 64, 64, 32, 1 << 20, 482) > NO_WORKSPACE
