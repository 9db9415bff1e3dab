"""Selection of pages whose bounds are infinite, against the definition of a score:

  max over the head's queries of sum_c max(q_c lo_c, q_c hi_c)

term by term in 64 bits, with NaN for zero times infinity and for a sum of both infinities,
so that a page is NaN (and taken before all others) only where a product or a sum is.  An
FP64 sum rounded to FP32 is the same in any order but for one in some 10^7."""
from __future__ import annotations

import pytest
import torch

from fireprot_amd.page_selection import PageBounds, select_pages
from tests.test_gpu_page_selection import check_selection

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = float("inf")


def by_definition(q, values, table, lengths, page, count, recent=1):
    """(index, lengths) of sequences whose pages all lie in the cache, on the CPU."""
    q, values, table = q.cpu().double(), values.cpu().double(), table.cpu().long()
    heads = values.shape[1]
    index = torch.full((len(q), heads, count), -1, dtype=torch.int32)
    kept = torch.zeros(len(q), dtype=torch.int32)
    for b, n in enumerate(lengths.tolist()):
        total = -(-n // page)
        m = min(total, count)
        kept[b] = n - (total - m) * page
        for h in range(heads):
            lo, hi = values[table[b, :total], h].unbind(1)
            score = torch.stack([torch.maximum(x * lo, x * hi).sum(-1)
                                 for x in q[b].unflatten(0, (heads, -1))[h]]).amax(0).float()
            nan = torch.isnan(score).tolist()
            score = torch.nan_to_num(score, nan=INF, posinf=INF, neginf=-INF).tolist()
            rank = sorted(range(total),
                          key=lambda i: (i < total - recent, not nan[i], -score[i], i))
            index[b, h, :m] = torch.tensor(sorted(rank[:m]), dtype=torch.int32)
    return index, kept


@pytest.mark.parametrize("q_type,kind", [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16)])
@pytest.mark.parametrize("group,heads,dim", [(1, 2, 32), (5, 1, 64), (8, 2, 128), (19, 1, 256)])
@pytest.mark.parametrize("total", [100, 700])
def test_infinite_bounds(q_type, kind, group, heads, dim, total):
    print(f"infinite bounds {q_type} {kind} {group, heads, dim, total}", flush=True)
    g = torch.Generator().manual_seed(dim + total)
    values = torch.randn(total, heads, 2, dim, generator=g).sort(dim=2)[0]
    # a channel of some pages infinite above, below, on both sides, wholly so, and a NaN
    for first, edges in ((3, (None, INF)), (4, (-INF, None)), (5, (-INF, INF)), (6, (INF, INF)),
                         (7, (-INF, -INF)), (8, (None, float("nan")))):
        at = torch.arange(first, total, 13)
        channel = torch.randint(0, dim, (len(at),), generator=g)
        for side, x in enumerate(edges):
            if x is not None:
                values[at, :, side, channel] = x
    values[9::26, :, 1, 0], values[9::26, :, 0, 1] = INF, -INF  # two channels
    values = values.to(kind)
    q = torch.randn(3, heads * group, dim, generator=g)
    # one sequence of queries that all point away from what is infinite above, one with zeros
    q[1] = -q[1].abs()
    q[2, :, ::5] = 0.0
    q = q.to(q_type)
    table = torch.stack([torch.randperm(total, generator=g) for _ in range(3)]).int()
    lengths = torch.tensor([total * 16, total * 16 - 5, (total - 30) * 16 + 1], dtype=torch.int32)
    for count in (2, 20, total // 2, total - 40):
        got = select_pages(q.cuda(), PageBounds(values.cuda(), 16), table.cuda(), lengths.cuda(),
                           count)
        check_selection(got, by_definition(q, values, table, lengths, 16, count), table)


def test_an_overflowed_channel_is_not_always_chosen():
    """One channel of a page overflowed: queries that do not ask for it pass the page by."""
    values = torch.zeros(200, 1, 2, 64, dtype=F16)
    values[:, 0, 1, 0] = torch.arange(200)
    values[17, 0, 1, 5] = INF
    table = torch.arange(200).int()[None].cuda()
    lengths = torch.tensor([3200], dtype=torch.int32).cuda()
    q = torch.ones(1, 1, 64, dtype=F16)
    for x, first in ((1.0, 17), (-1.0, 198)):
        q[0, 0, 5] = x
        got = select_pages(q.cuda(), PageBounds(values.cuda(), 16), table, lengths, 2)
        assert got.index[0, 0].tolist() == [first, 199]
