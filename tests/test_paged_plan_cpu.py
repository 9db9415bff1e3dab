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


@pytest.mark.parametrize("cache_dtype,q_heads,heads,head_dim,max_length,window", [
    (_native.FPX_I8, 16, 16, 64, 9001, 1000), (_native.FPX_I8, 16, 16, 64, 9001, 900),
    (_native.FPX_I8, 16, 16, 64, 9001, 1200), (_native.FPX_F8E4M3, 32, 16, 32, 2000, 0),
    (_native.FPX_BF16, 16, 8, 64, 600, 0), (_native.FPX_F32, 8, 8, 32, 700, 0)])
def test_the_cut_does_not_go_by_the_number_of_work_groups(size, cache_dtype, q_heads, heads,
                                                          head_dim, max_length, window):
    """While a call may read at most 128 MB each further sequence adds its own units'
    places, and nothing else; beyond, no length and no sequence changes what the fixed
    number of shares takes but the rows' places in a list (8 bytes each)."""
    element = {_native.FPX_F32: 4, _native.FPX_BF16: 2}.get(cache_dtype, 1)
    span = min(max_length, window + 31) if window else max_length
    most = (128 << 20) // (heads * span * 2 * head_dim * element)
    first = -(-192 // heads)  # from here on a unit has 512 keys
    assert most > first + 8
    each = size(cache_dtype, first, q_heads, heads, head_dim, max_length, window) / first
    for batch in range(first, most + 1):
        got = size(cache_dtype, batch, q_heads, heads, head_dim, max_length, window)
        assert abs(got - each * batch) <= 1024, batch
    beyond = [size(cache_dtype, batch, q_heads, heads, head_dim, max_length, window)
              for batch in (most + 1, 2 * most, 4 * most)]
    assert beyond[0] - beyond[1] == heads * 8 * (most + 1 - 2 * most)
    assert beyond[2] - beyond[1] == heads * 8 * 2 * most
