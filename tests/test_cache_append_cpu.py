"""fpx_cache_append without a GPU: what the entry and its Python side refuse."""
from __future__ import annotations

import pytest
import torch

from fireprot_amd import _native, cache_append, rotary
from fireprot_amd.kv_cache import PagedCache
from tests.test_kv_cache_cpu import lib  # noqa: F401

MB = 1 << 20


def _args(**override):
    args = dict(dtype=1, cache_dtype=3, layout=0, q=MB, q_sb=1024, q_sn=512, q_sh=128, q_out=2 * MB,
                qo_sb=1024, qo_sn=512, qo_sh=128, q_heads=4, k=3 * MB, k_sb=512, k_sn=256, k_sh=128,
                v=4 * MB, v_sb=512, v_sn=256, v_sh=128, positions=5 * MB, positions_64=1, p_sb=2,
                p_sn=1, inv_freq=6 * MB, scale=1.0, rotary_dim=128, slots=None, block_table=7 * MB,
                table_sb=3, table_pages=3, batch=8, tokens=2, cache_k=8 * MB, cache_v=9 * MB,
                k_scale=10 * MB, v_scale=11 * MB, pages=4, heads=2, page_size=16, head_dim=128,
                stream=None)
    assert set(override) <= set(args)
    args.update(override)
    return list(args.values())


@pytest.mark.parametrize("bad", [
    dict(dtype=3), dict(dtype=-1), dict(cache_dtype=5), dict(layout=2), dict(positions_64=2),
    dict(rotary_dim=0), dict(rotary_dim=3), dict(rotary_dim=130), dict(head_dim=80),
    dict(page_size=24), dict(pages=0), dict(heads=0), dict(q_heads=-1), dict(q_heads=8190),
    dict(heads=4097), dict(batch=-1), dict(tokens=-1), dict(batch=1 << 20, tokens=1 << 12),
    dict(q_sb=-1), dict(qo_sh=-1), dict(k_sn=-1), dict(v_sb=-1), dict(p_sb=-1), dict(table_sb=-1),
    dict(table_pages=-1), dict(q_out=MB, qo_sn=640), dict(slots=12 * MB), dict(block_table=None)])
def test_sizes_are_refused(lib, bad):  # noqa: F811
    assert lib.fpx_cache_append(*_args(**bad)) == _native.FPX_ERR_DIMS


@pytest.mark.parametrize("bad", [
    dict(k=None), dict(v=None), dict(q=None), dict(q_out=None), dict(positions=None),
    dict(inv_freq=None), dict(cache_k=None), dict(cache_v=8 * MB + 8), dict(k_scale=None),
    dict(v_scale=11 * MB + 4), dict(q=MB + 1), dict(dtype=0, v=4 * MB + 2),
    dict(positions=5 * MB + 4), dict(inv_freq=6 * MB + 4), dict(block_table=7 * MB + 2),
    dict(block_table=None, slots=12 * MB + 4)])
def test_pointers_are_refused(lib, bad):  # noqa: F811
    assert lib.fpx_cache_append(*_args(**bad)) == _native.FPX_ERR_POINTER


@pytest.mark.parametrize("bad", [
    dict(q_out=MB + 256), dict(q_out=3 * MB), dict(q_out=4 * MB + 64), dict(q_out=5 * MB),
    dict(q_out=6 * MB), dict(q_out=7 * MB), dict(q_out=8 * MB), dict(q_out=10 * MB),
    dict(qo_sh=64), dict(qo_sb=0), dict(cache_k=MB), dict(cache_v=3 * MB), dict(cache_k=4 * MB),
    dict(k_scale=5 * MB), dict(v_scale=6 * MB), dict(cache_v=7 * MB), dict(cache_v=8 * MB + 4096),
    dict(k_scale=9 * MB), dict(v_scale=10 * MB + 496),
    dict(block_table=None, slots=8 * MB)])
def test_overlaps_are_refused(lib, bad):  # noqa: F811
    assert lib.fpx_cache_append(*_args(**bad)) == _native.FPX_ERR_DIMS


def test_empty_calls_launch_nothing(lib):  # noqa: F811
    assert lib.fpx_cache_append(*_args(batch=0, k=None)) == 0
    assert lib.fpx_cache_append(*_args(tokens=0, q=None)) == 0


def test_tensors_are_checked():
    cache = PagedCache.allocate(4, 2, 16, 32, dtype=torch.float16, device="cpu")
    f = rotary.rotary_frequencies(32)
    k = torch.zeros(3, 5, 2, 32, dtype=torch.float16)
    positions = torch.zeros(3, 5, dtype=torch.int64)
    with pytest.raises(ValueError):  # not on a HIP device
        cache_append.cache_append(cache, None, k, k, positions, f,
                                  block_table=torch.zeros(3, 1, dtype=torch.int32))
    with pytest.raises(ValueError):
        cache_append.cache_append(cache, None, k, k, positions, f, layout="other")
