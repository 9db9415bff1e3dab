"""Tensors that share memory: the search (csrc/overlap.hpp, compiled for the host)
against sets of addresses, and the refusals of the C entries and of PagedCache
(nothing here reaches a launch)."""
from __future__ import annotations

import ctypes
import itertools
import pathlib
import random
import shutil
import subprocess

import pytest
import torch

from fireprot_amd import _native, kv_cache

CSRC = pathlib.Path(__file__).resolve().parents[1] / "fireprot_amd" / "csrc"

SHIM = r"""
#include "overlap.hpp"
using namespace fpx;
static MemoryBlock block(const int64_t* x) {  // base, element, 4 x (count, stride)
  return MemoryBlock(reinterpret_cast<const void*>(x[0]), x[1], MemoryAxis{x[2], x[3]},
                     MemoryAxis{x[4], x[5]}, MemoryAxis{x[6], x[7]}, MemoryAxis{x[8], x[9]});
}
extern "C" int t_meet(const int64_t* a, const int64_t* b) { return blocks_meet(block(a), block(b)); }
extern "C" int t_self(const int64_t* a) { return block_meets_itself(block(a)); }
"""


@pytest.fixture(scope="module")
def search(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    work = tmp_path_factory.mktemp("overlap")
    (work / "shim.cpp").write_text(SHIM)
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I",
                    str(CSRC), str(work / "shim.cpp"), "-o", str(work / "shim.so")], check=True)
    lib = ctypes.CDLL(str(work / "shim.so"))

    def numbers(b):
        base, element, axes = b
        axes = list(axes) + [(1, 0)] * (4 - len(axes))
        return (ctypes.c_int64 * 10)(base, element, *itertools.chain(*axes))

    return (lambda a, b: bool(lib.t_meet(numbers(a), numbers(b))),
            lambda a: bool(lib.t_self(numbers(a))))


def places(b):
    """First byte of each element of a block."""
    base, element, axes = b
    return [base + element * sum(i * s for i, (_, s) in zip(index, axes))
            for index in itertools.product(*(range(n) for n, _ in axes))]


def test_search_against_sets_of_addresses(search):
    meet, itself = search
    rng = random.Random(1)
    seen = {True: 0, False: 0}
    for _ in range(6000):
        element = rng.choice([1, 2, 4])
        blocks = []
        for _ in range(2):
            kind = rng.random()
            counts = [rng.randint(1, 5) for _ in range(4)]
            if kind < 0.5:  # a view of a tensor: strides that contain each other
                strides, s = [], 1
                for n in reversed(counts):
                    strides.insert(0, s)
                    s *= n + rng.randint(0, 3)
                if rng.random() < 0.5:
                    pairs = list(zip(counts, strides))
                    rng.shuffle(pairs)
                    counts, strides = zip(*pairs)
            else:  # any strides, broadcasts among them
                strides = [rng.choice([0, 1, 2, 3, 5, 7, 12, 30]) for _ in range(4)]
            blocks.append((4096 + element * rng.randint(0, 80), element,
                           list(zip(counts, strides))))
        a, b = blocks
        want = bool(set(places(a)) & set(places(b)))
        assert meet(a, b) == meet(b, a) == want, (a, b)
        seen[want] += 1
        where = places(a)
        assert itself(a) == (len(set(where)) < len(where)), a
    assert min(seen.values()) > 500


def test_views_of_one_tensor_that_interleave(search):
    meet, itself = search
    width = 48 * 128
    for tokens in (1, 7, 1 << 20):
        q = (1 << 30, 2, [(3, tokens * width), (tokens, width), (32, 128), (128, 1)])
        k = ((1 << 30) + 2 * 32 * 128, 2, [(3, tokens * width), (tokens, width), (8, 128), (128, 1)])
        assert not meet(q, k) and not itself(q)
        # one channel further to the left and the last head's last is the first's
        assert meet(q, (k[0] - 2, *k[1:]))
        # heads first
        h = ((1 << 30), 2, [(3, 40 * tokens * 128), (tokens, 128), (32, tokens * 128), (128, 1)])
        assert not meet(h, ((1 << 30) + 2 * 32 * tokens * 128, *h[1:])[:2]
                        + ([(3, 40 * tokens * 128), (tokens, 128), (8, tokens * 128), (128, 1)],))
    # past 32 bits, and strides no memory has
    assert meet((4096, 4, [(2, 1 << 40)]), (4096 + (4 << 40), 4, [(1, 0)]))
    assert not meet((4096, 4, [(2, 1 << 40)]), (4096 + (2 << 40), 4, [(1, 0)]))
    assert not itself((4096, 4, [(1 << 31, 1 << 62), (9, 1)]))
    # nothing has no place
    assert not meet((4096, 4, [(0, 1), (9, 1)]), (4096, 4, [(9, 1)]))


@pytest.fixture(scope="module")
def lib():
    if not _native.LIB_PATH.exists():
        from fireprot_amd import build
        build.build()
    return _native.library()


MB = 1 << 20


def rotary(**override):
    args = dict(dtype=1, layout=0, q=MB, q_sb=1024, q_sn=128, q_sh=32, q_out=2 * MB, qo_sb=1024,
                qo_sn=128, qo_sh=32, q_heads=4, k=3 * MB, k_sb=1024, k_sn=128, k_sh=32,
                k_out=4 * MB, ko_sb=1024, ko_sn=128, ko_sh=32, k_heads=4, positions=5 * MB,
                positions_64=1, p_sb=8, p_sn=1, inv_freq=6 * MB, scale=1.0, inverse=0, batch=2,
                tokens=8, head_dim=32, rotary_dim=32, stream=None)
    assert set(override) <= set(args)
    return list({**args, **override}.values())


@pytest.mark.parametrize("bad", [
    dict(q_out=MB + 2), dict(q_out=MB - 4094), dict(q_out=3 * MB), dict(q_out=3 * MB + 2048),
    dict(k_out=2 * MB), dict(k_out=2 * MB + 64), dict(k_out=MB), dict(k_out=3 * MB + 64),
    dict(q_out=5 * MB), dict(k_out=5 * MB + 64), dict(q_out=6 * MB - 4094), dict(k_out=6 * MB),
    dict(q_out=MB, k=MB), dict(qo_sn=64), dict(qo_sb=0), dict(ko_sh=16), dict(ko_sb=896),
    dict(q_out=2 * MB, qo_sn=160, qo_sb=1280, k_out=2 * MB + 254, ko_sn=160, ko_sb=1280,
         k_heads=1)])
def test_rotary_refuses(lib, bad):
    assert lib.fpx_rotary(*rotary(**bad)) == _native.FPX_ERR_DIMS


def cache(**override):
    args = dict(row_dtype=1, cache_dtype=3, k=MB, k_st=512, k_sh=128, v=2 * MB, v_st=512, v_sh=128,
                slots=3 * MB, tokens=8, cache_k=4 * MB, cache_v=5 * MB, k_scale=6 * MB,
                v_scale=7 * MB, pages=4, heads=4, page_size=16, head_dim=128, stream=None)
    assert set(override) <= set(args)
    return list({**args, **override}.values())


SIZE = 4 * 4 * 16 * 128  # bytes of one of the cache's tensors


@pytest.mark.parametrize("entry", ["fpx_cache_write", "fpx_cache_read"])
@pytest.mark.parametrize("bad", [
    dict(k=4 * MB), dict(v=4 * MB + SIZE - 2), dict(k=5 * MB + 64), dict(v=6 * MB),
    dict(k=7 * MB + 4 * 4 * 4 * 16 - 2)])
def test_rows_of_the_cache_are_refused(lib, entry, bad):
    assert getattr(lib, entry)(*cache(**bad)) == _native.FPX_ERR_DIMS


@pytest.mark.parametrize("entry", ["fpx_cache_write", "fpx_cache_read"])
def test_rows_inside_a_cache_of_more_bytes_than_63_bits_count(lib, entry):
    most = dict(cache_dtype=1, pages=2 ** 29, heads=2 ** 15, page_size=4096, head_dim=256,
                k_st=2 ** 23, k_sh=256, v_st=2 ** 23, v_sh=256, cache_k=1 << 40, cache_v=1 << 41,
                k=1 << 42, v=1 << 50)
    assert getattr(lib, entry)(*cache(**most)) == _native.FPX_ERR_DIMS


@pytest.mark.parametrize("bad", [
    dict(cache_v=4 * MB), dict(cache_v=4 * MB + SIZE - 16), dict(v_scale=6 * MB),
    dict(v_scale=6 * MB + 4 * 4 * 4 * 16 - 16), dict(k_scale=5 * MB), dict(slots=4 * MB),
    dict(slots=7 * MB)])
def test_writes_refuse_a_cache_that_overlaps(lib, bad):
    assert lib.fpx_cache_write(*cache(**bad)) == _native.FPX_ERR_DIMS


@pytest.mark.parametrize("bad", [
    dict(v=MB), dict(v=MB + 2), dict(v=MB + 256 * 3), dict(k_st=384), dict(v_sh=64), dict(k_sh=0),
    dict(k=3 * MB), dict(k_st=640, v=MB + 2 * 512 - 2, v_st=640)])
def test_reads_refuse_outputs_that_overlap(lib, bad):
    assert lib.fpx_cache_read(*cache(**bad)) == _native.FPX_ERR_DIMS


def attention(**override):
    args = dict(dtype=1, cache_dtype=1, q=MB, q_sb=1024, q_sh=128, cache_k=2 * MB, cache_v=4 * MB,
                k_scale=None, v_scale=None, pages=64, heads=2, page_size=16, head_dim=128,
                block_table=6 * MB, table_sb=256, table_pages=256, lengths=7 * MB, batch=3,
                q_heads=8, max_length=4096, window=0, scale=0.1, out=8 * MB, o_sb=1024, o_sh=128,
                lse=9 * MB, workspace=16 * MB, workspace_bytes=1 << 30, stream=None)
    assert set(override) <= set(args)
    return list({**args, **override}.values())


@pytest.mark.parametrize("bad", [
    dict(out=MB + 16), dict(out=MB - 16), dict(out=MB + 5 * 1024), dict(out=2 * MB),
    dict(out=4 * MB + 64 * 2 * 16 * 256 - 16), dict(out=6 * MB), dict(out=7 * MB), dict(out=9 * MB),
    dict(o_sh=64), dict(o_sb=0), dict(lse=MB), dict(lse=6 * MB + 64), dict(lse=7 * MB + 8),
    dict(lse=2 * MB), dict(workspace=MB), dict(workspace=2 * MB), dict(workspace=7 * MB),
    dict(workspace=8 * MB), dict(workspace=9 * MB)])
def test_attention_refuses(lib, bad):
    assert lib.fpx_paged_attention(*attention(**bad)) == _native.FPX_ERR_DIMS


def test_caches_whose_tensors_overlap_are_refused():
    buffer = torch.zeros(3, 3, 16, 64, dtype=torch.int8)
    other, scales = torch.zeros(2, 3, 16, 64, dtype=torch.int8), torch.zeros(3, 3, 16)
    s, t = scales[:2], torch.zeros(2, 3, 16)
    kv_cache.PagedCache(buffer[:2], other, s, t)
    for args in ((buffer[:2], other, s, s), (buffer[:2], other, s, scales[1:]),
                 (buffer[:2], buffer[1:], s, t), (buffer[:2], buffer[:2], s, t),
                 (buffer[:2], other, buffer.view(torch.float32).flatten()[:96].view(2, 3, 16), t)):
        with pytest.raises(ValueError, match="share memory"):
            kv_cache.PagedCache(*args)
    # side by side in one buffer
    both = torch.zeros(4, 3, 16, 64, dtype=torch.float16)
    kv_cache.PagedCache(both[:2], both[2:])
    kv_cache.PagedCache(both[2:], both[:2])
