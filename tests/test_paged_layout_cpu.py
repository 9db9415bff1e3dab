"""The paged cache's index rules (csrc/paged_layout.hpp) compiled for the host:
bad slots, bad pages, lengths and windows are decided here, before a kernel
with the same header runs them."""
from __future__ import annotations

import ctypes
import pathlib
import random
import shutil
import subprocess

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "fireprot_amd" / "csrc"

SHIM = r"""
#include "paged_layout.hpp"
using namespace fpx;
extern "C" {
int64_t t_row(int64_t slot, int head, int64_t pages, int heads, int shift) {
  return cache_row(slot, head, pages, heads, shift);
}
int t_range(int length, int max_length, int window, int* first, int* end) {
  KeyRange r = key_range(length, max_length, window);
  *first = r.first; *end = r.end;
  return r.valid;
}
int t_units(int first, int end, int unit) { return unit_count({first, end, true}, unit); }
int64_t t_limit(int64_t max_length, int64_t window, int unit) { return unit_limit(max_length, window, unit); }
int t_start(int total, int groups, int group) { return share_start(make_shares(total, groups), group); }
int t_share(int total, int groups, int unit) { return share_of(make_shares(total, groups), unit); }
int t_entry(int key, int first, int end, int shift) { return table_entry(key, {first, end, true}, shift); }
int t_page(int page, int64_t pages) { return page_valid(page, pages); }
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    work = tmp_path_factory.mktemp("paged_layout")
    (work / "shim.cpp").write_text(SHIM)
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", str(CSRC),
                    str(work / "shim.cpp"), "-o", str(work / "shim.so")], check=True)
    lib = ctypes.CDLL(str(work / "shim.so"))
    lib.t_row.restype = ctypes.c_int64
    lib.t_row.argtypes = [ctypes.c_int64, ctypes.c_int, ctypes.c_int64, ctypes.c_int, ctypes.c_int]
    lib.t_page.argtypes = [ctypes.c_int, ctypes.c_int64]
    lib.t_limit.restype = ctypes.c_int64
    lib.t_limit.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int]
    return lib


def test_rows(rules):
    for pages, heads, shift in ((1, 1, 4), (7, 3, 5), (2 ** 31 - 1, 65535, 4)):
        size = 1 << shift
        rng = random.Random(pages)
        for slot in [0, pages * size - 1] + [rng.randrange(pages * size) for _ in range(50)]:
            for head in (0, heads - 1):
                want = ((slot // size) * heads + head) * size + slot % size
                assert rules.t_row(slot, head, pages, heads, shift) == want
                assert want < pages * heads * size
        for slot in (-1, -5, -2 ** 63):
            assert rules.t_row(slot, 0, pages, heads, shift) == -1
        for slot in (pages * size, pages * size + 1, 2 ** 63 - 1):
            assert rules.t_row(slot, 0, pages, heads, shift) == -2


def test_ranges(rules):
    first, end = ctypes.c_int(), ctypes.c_int()
    for length in (-2 ** 31, -1, 0, 1, 15, 16, 100, 101, 2 ** 31 - 1):
        for window in (0, 1, 7, 100, 2 ** 31 - 1):
            ok = rules.t_range(length, 100, window, ctypes.byref(first), ctypes.byref(end))
            assert ok == (0 <= length <= 100)
            if ok:
                assert end.value == length
                assert first.value == (max(0, length - window) if window else 0)
            else:
                assert first.value == end.value == 0


def test_units_cover_a_range_and_never_pass_their_limit(rules):
    rng = random.Random(3)
    for _ in range(4000):
        unit = rng.choice([64, 128])
        max_length = rng.choice([0, 1, 31, 32, 33, rng.randrange(1, 20000), 2 ** 30 - 1])
        window = rng.choice([0, 1, rng.randrange(1, 5000), 2 ** 30 - 1])
        length = rng.randint(0, min(max_length, 40000))
        if rng.random() < 0.3:
            length = max_length
        first = max(0, length - window) if window else 0
        n = rules.t_units(first, length, unit)
        assert 1 <= n <= rules.t_limit(max_length, window, unit)
        start = first // 32 * 32
        if length > first:  # the last unit holds the last key
            assert start + (n - 1) * unit < length <= start + n * unit
        else:
            assert n == 1
    # the limit is reached
    assert rules.t_limit(1000, 0, 128) == 8 and rules.t_units(0, 1000, 128) == 8
    assert rules.t_limit(1000, 98, 128) == 2 and rules.t_units(31, 129, 128) == 2


def test_shares_are_equal_and_cover_all_units(rules):
    rng = random.Random(4)
    for _ in range(300):
        groups = rng.choice([1, 2, 255, 256, 512, 1024])
        total = rng.choice([1, groups - 1, groups, groups + 1, rng.randrange(1, 5000),
                            2 ** 31 - 1 - rng.randrange(1000)])
        total = max(1, total)
        starts = [rules.t_start(total, groups, i) for i in range(groups + 1)]
        assert starts[0] == 0 and starts[-1] == total
        sizes = [b - a for a, b in zip(starts, starts[1:])]
        assert max(sizes) - min(sizes) <= 1
        for i in range(groups):
            for unit in {starts[i], starts[i + 1] - 1}:
                if starts[i] <= unit < starts[i + 1]:
                    assert rules.t_share(total, groups, unit) == i


def test_table_entries_stay_in_the_range(rules):
    for first, end in ((0, 1), (0, 100), (37, 100), (63, 64), (95, 96)):
        for key in range(0, 200):
            for shift in (4, 5, 7):
                want = min(max(key, first), end - 1) >> shift
                assert rules.t_entry(key, first, end, shift) == want


def test_bad_pages(rules):
    for page in (-2 ** 31, -1, 5, 6, 2 ** 31 - 1):
        assert not rules.t_page(page, 5)
    for page in range(5):
        assert rules.t_page(page, 5)
