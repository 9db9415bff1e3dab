"""Slots of positions whose table entry names no page: past every cache, where a
write leaves the token out and a read gives NaN, and not the padding's -1, which
reads as zeros."""
from __future__ import annotations

import pytest
import torch

from fireprot_amd import kv_cache

PAST = torch.iinfo(torch.int64).max


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_negative_pages(kind):
    table = torch.tensor([[-1, 2], [3, -(2 ** 31)], [-7, -1]], dtype=kind)
    positions = torch.tensor([[0, 15, 16, -3], [0, 16, 31, 32], [3, 20, -1, 99]])
    assert kv_cache.cache_slots(table, positions, 16).tolist() == [
        [PAST, PAST, 32, -1], [48, PAST, PAST, PAST], [PAST, PAST, -1, PAST]]


def test_pages_past_every_cache_stay_slots():
    table = torch.tensor([[2 ** 31 - 1]], dtype=torch.int32)
    assert kv_cache.cache_slots(table, torch.tensor([[0, 4095]]), 4096).tolist() == [
        [(2 ** 31 - 1) * 4096, 2 ** 43 - 1]]
