"""Attention over 4-bit pools for more requests than a wave has lanes, whose schedule is written out before:
two KV heads a unit and one, tables that KV heads share and tables of their own, with a window and without."""

import pytest
import torch

from mini_hisparse_amd.row_kernels import attend_pages

from page_cases import case, check

# two and four pairs of KV heads, and three (units that no four waves divide); more than 8 query heads a KV
# head and three KV heads, which are not paired
LAYOUTS = [(4, 2, 32), (14, 2, 64), (8, 8, 64), (6, 6, 64), (28, 4, 128), (20, 2, 64), (6, 3, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("batch,heads,kv,dim,per_head",
                         [(65, *shape, False) for shape in LAYOUTS] + [(200, *shape, False) for shape in LAYOUTS[:4]]
                         + [(65, 14, 2, 64, True), (65, 6, 3, 32, True)])
def test_many_requests(gpu, batch, heads, kv, dim, per_head):
    gen = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, 200, (batch,), generator=gen)
    lengths[::9] = 0
    lengths[batch // 2], lengths[-1] = 6000, 3000
    for dtype, window, sinks in (("bf16", None, 0), ("f16", 100, 4), ("bf16", 2500, 40)):
        args = case(batch, heads, kv, dim, 16, lengths.tolist(), "fp4", dtype, gpu, window=window, sinks=sinks,
                    per_head=per_head, wide=400)
        check(attend_pages(*args, window=window, sinks=sinks), args, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("page", [16, 12])
def test_more_than_a_turn_of_the_schedule(gpu, page, per_head):
    """1100 requests: two turns of the workgroup that writes the schedule."""
    gen = torch.Generator().manual_seed(page)
    lengths = torch.randint(0, 120, (1100,), generator=gen)
    lengths[::7] = 0
    lengths[3], lengths[1050] = 9000, 2000
    for window, sinks in ((None, 0), (1800, 40)):
        args = case(1100, 4, 2, 32, page, lengths.tolist(), "fp4", "bf16", gpu, window=window, sinks=sinks,
                    per_head=per_head, wide=400)
        check(attend_pages(*args, window=window, sinks=sinks), args, window, sinks)
