"""4-bit attention of KV heads in pairs and one by one in the launch for short histories, on both sides of
the rule that chooses: the tables' width and the number of requests."""

import pytest
import torch

from mini_hisparse_amd.row_kernels import attend_pages

from page_cases import case, check

DTYPES = ["bf16", "f16", "f32"]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 32), (14, 2, 64), (16, 2, 64), (12, 2, 128), (2, 2, 128)])
@pytest.mark.parametrize("page", [16, 12, 64])
def test_one_part_of_many_requests(gpu, page, heads, kv, dim, dtype):
    """128 requests of two KV heads have a workgroup for every CU one by one, 129 go in pairs."""
    for batch in (128, 129):
        gen = torch.Generator().manual_seed(batch)
        lengths = torch.randint(0, 150, (batch,), generator=gen)
        lengths[::9] = 0
        lengths[5] = 1000
        for window, sinks in ((None, 0), (40, 4)):
            args = case(batch, heads, kv, dim, page, lengths.tolist(), "fp4", dtype, gpu, window=window, sinks=sinks,
                        wide=0)
            check(attend_pages(*args, window=window, sinks=sinks), args, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,dim,batch", [(8, 8, 32, 16), (8, 8, 64, 16), (16, 8, 64, 16), (8, 4, 128, 32)])
@pytest.mark.parametrize("page", [16, 12])
def test_several_parts(gpu, page, heads, kv, dim, batch, dtype):
    """Tables of 4000 tokens, which pairs of these batches take in short parts and single heads in long
    ones; of 1900, which single heads take in short parts."""
    for top in (4000, 1900):
        lengths = [top, 0, 33, 1, 1025, 1024, top - 17] + [5, 64, 0] * batch
        for window, sinks in ((None, 0), (1500, 33)):
            args = case(batch, heads, kv, dim, page, lengths[:batch], "fp4", dtype, gpu, window=window, sinks=sinks,
                        wide=0)
            check(attend_pages(*args, window=window, sinks=sinks), args, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("code,dtype,dim,batch", [("fp4", "bf16", 64, 129), ("fp4", "f16", 128, 4), ("fp4", "f32", 64, 16)])
def test_replays(gpu, code, dtype, dim, batch):
    """Captured calls in pairs, in one part and in several, follow the lengths of the moment."""
    heads = 8 if batch == 16 else 2
    lengths = [4000 if batch == 16 else 900] + [300] * (batch - 1)
    query, pool, tables, at = case(batch, heads, heads, dim, 16, lengths, code, dtype, gpu, wide=0)
    graph = torch.cuda.CUDAGraph()
    attend_pages(query, pool, tables, at)
    with torch.cuda.graph(graph):
        out = attend_pages(query, pool, tables, at)
    for now in (lengths, [0] + [7] * (batch - 1), [lengths[0] - 1] + [299] * (batch - 1), [33] * batch):
        at.copy_(torch.tensor(now, dtype=torch.int32))
        out.fill_(7.0)
        graph.replay()
        assert torch.equal(out, attend_pages(query, pool, tables, at))
        check(out, (query, pool, tables, at))
