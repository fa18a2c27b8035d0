"""The paged context operators at the edges of what their documentation allows: rows that are taken whole, scores that are not numbers,
lengths far outside the table, launch forms of large calls (against the 64-bit restatement of paged_reference)."""
import math

import pytest
import torch

import paged_reference as R
from nvblox_mindmap_amd.diffuser_actor import paged_context as P

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def summaries(low, high, hd, page=16):
    """Pages [n, kv_heads, 16] that only a selection reads: their summaries, and keys / values that may be any."""
    n, heads, w = low.shape
    empty = torch.zeros((n, heads, page, w), dtype=low.dtype, device="cuda")
    return P.ContextPages(empty, torch.zeros((n, heads, w, page), dtype=low.dtype, device="cuda"), low.cuda(), high.cuda(), hd)


# slots of the table, pages that a context holds, count: every launch form of the selection (four waves, sixteen, segments, a row of any
# length), each with more entries than threads and a count that takes them all
@pytest.mark.parametrize("slots,held,count", [(1536, 257, 512), (1536, 400, 400), (700, 700, 701), (1536, 1536, 1536), (8192, 1100, 1100), (5000, 4999, 6000), (8192, 8192, 8192),
                                              (40000, 100, 128), (8193, 1365, 1365), (40000, 409, 409), (40000, 5000, 5000), (40000, 40000, 40000)])
def test_a_row_that_is_taken_whole(slots, held, count):
    """As many pages as the context holds, or more: all of them in order, then -1, whatever the signs of their scores."""
    H, T, hd, pool = 4, 2, 16, 64
    g = torch.Generator().manual_seed(slots + held)
    low = -torch.rand(pool, H, 16, generator=g) - 1.0
    q = torch.rand(2, T, H * hd, generator=g) + 0.1  # scores of -1.6 to -36
    q[1, 1] *= torch.where(torch.rand(H * hd, generator=g) < 0.5, 1.0, -1.0)  # ... and of both signs
    table = torch.randint(0, pool, (2, slots), generator=g).to(torch.int32)
    table[1, ::5] = -1
    lengths = i32([16 * held - 15, 16 * held])
    got = P.select_pages(q.cuda(), summaries(low, low * 0.9, hd), table.cuda(), lengths.cuda(), H, count).cpu()
    for b in range(2):
        there = (table[b, :held] >= 0).nonzero().flatten().to(torch.int32)
        want = torch.cat([there, torch.full((count - len(there),), -1, dtype=torch.int32)])
        assert torch.equal(got[b], want.expand(T, H, count)), b
