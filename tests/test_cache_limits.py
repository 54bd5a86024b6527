"""The cache operators at the ends of the sizes they take: the most requests, heads, rows and tokens,
pools past 2^32 rows, and captured calls that share their memory."""

import pytest
import torch

from mini_hisparse_amd.dense import norm_rotary_split
from mini_hisparse_amd.quantized import QuantizedPool, append_quantized, read_quantized
from mini_hisparse_amd.row_kernels import attend_pages

from test_attend_pages import case, check
from test_norm_rotary import check as check_norm, formula as norm_formula
from test_quantized import quantise


@pytest.fixture(autouse=True)
def give_back_memory():
    """Some of these hold tens of GB."""
    yield
    if torch.cuda.is_available():
        torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [2, 200])
def test_as_many_requests_as_a_call_takes(gpu, wide):
    """65535 requests of 0 .. 40 tokens, and one long one among them: of 7 kinds, compared with
    the kinds' formula."""
    batch, heads, kv, dim, page = 65_535, 4, 2, 32, 16
    kinds = case(7, heads, kv, dim, page, [40, 1, 0, 17, 33, 16, 32], "int8", "bf16", gpu, wide=wide)
    pick = torch.arange(batch, device=gpu) % 7
    query, tables, lengths = (t[pick].contiguous() for t in (kinds[0], kinds[2], kinds[3]))
    got = attend_pages(query, kinds[1], tables, lengths)
    check(got[:7], kinds)
    if wide == 2:  # every request in one part whatever the batch
        assert torch.equal(got, got[:7][pick])
    else:
        for first in (700, 32_767, batch - 7):
            rows = torch.arange(first, first + 7, device=gpu)
            check(got[rows], tuple(x if x is kinds[1] else x[pick[rows]] for x in kinds))
        assert (got[pick == 2] == 0).all() and got.isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim", [(65_535, 65_535, 32), (65_535, 1, 32), (65_535, 65_535, 5), (65_535, 1, 33)])
@pytest.mark.parametrize("wide", [2, 200])
def test_as_many_heads_as_a_call_takes(gpu, heads, kv, dim, wide):
    args = query, pool, tables, lengths = case(1, heads, kv, dim, 16, [37], "int8", "bf16", gpu, wide=wide, spare=1)
    got = attend_pages(*args)
    group = heads // kv
    for h in (0, 1, 15, 16, 4095, 32_767, 65_519, 65_520, 65_534):  # the formula over every head would take long
        k = h // group
        one = QuantizedPool(pool.codes[:, :, :, k : k + 1].contiguous(), pool.scales[:, :, :, k : k + 1].contiguous())
        check(got[:, h : h + 1], (query[:, h : h + 1], one, tables, lengths))


@pytest.mark.gpu
def test_table_of_as_many_tokens_as_it_may_name(gpu):
    """A table for 2^31 - 16 tokens of which few are there."""
    query, pool, tables, lengths = case(2, 4, 2, 64, 16, [100, 33], "int8", "bf16", gpu)
    wide = torch.full((1, 2**27 - 1), -1, dtype=torch.int32, device=gpu)
    for b in range(2):
        wide[0, : tables.shape[1]] = tables[b]
        args = (query[b : b + 1], pool, wide, lengths[b : b + 1])
        got = attend_pages(*args)
        check(got, (*args[:2], tables[b : b + 1], args[3]))


@pytest.mark.gpu
@pytest.mark.parametrize("dim,page", [(32, 2**18), (32, 2**18 - 1), (33, 2**18)])
def test_as_many_tokens_as_a_request_may_have(gpu, dim, page):
    """Nearly 2^31 tokens: a first and a last page of their own, and one read thousands of times between
    them, each with about a third of the weight, so that none can be lost."""
    pages = (2**31 - 1) // page
    gen = torch.Generator().manual_seed(dim)
    query = torch.randn(1, 1, dim, generator=gen).repeat(1, 2, 1).to(torch.bfloat16)
    codes = torch.randint(90, 128, (3, 2, page, 1, dim), generator=gen, dtype=torch.int8)
    codes[0, 0] *= -query[0, 0].sign().to(torch.int8)  # the middle's keys: scores near -9, the others' 0
    codes[0, 1] *= -1
    length = query[0, 0].double().abs().sum().item() * 109 * dim**-0.5  # of a score at scale 1
    scales = torch.tensor([[9.0 / length, 0.5 / 127], [0.0, 1.0 / 127], [0.0, 3.0 / 127]])
    scales = scales[:, :, None, None].repeat(1, 1, page, 1)
    pool = QuantizedPool(codes.to(gpu), scales.to(gpu))
    tables = torch.zeros(1, pages, dtype=torch.int32, device=gpu)
    tables[0, 0], tables[0, -1] = 1, 2
    lengths = torch.tensor([pages * page], dtype=torch.int32, device=gpu)
    got = attend_pages(query.to(gpu), pool, tables, lengths).double().cpu()
    values = codes.double() * scales.double()[..., None]
    q, total, want, weight = query[0, 0].double(), 0.0, 0.0, 0.0
    for block, times in ((0, pages - 2), (1, 1), (2, 1)):
        p = times * torch.exp(values[block, 0, :, 0] @ q * dim**-0.5)
        total, want, weight = total + p.sum(), want + p @ values[block, 1, :, 0], weight + p @ values[block, 1, :, 0].abs()
    want, weight = want / total, weight / total
    shares = [(pages - 2) * torch.exp(values[0, 0, :, 0] @ q * dim**-0.5).sum().item() / total.item(), page / total.item()]
    assert all(0.15 < x < 0.6 for x in shares)
    # a lane adds at most 2^19 products (2^31 tokens over 1024 splits of four waves) in fp32; beside that
    # test_attend_pages.check's terms, all below 2^-14 here
    tol = 2.0**-8 * want.abs() + 2 * (2**19 * 2.0**-24 + 2.0**-14) * weight
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max().item()


@pytest.mark.gpu
def test_pool_of_more_rows_than_32_bits_count(gpu):
    blocks, page = 2**28 + 1, 16
    pool = QuantizedPool.empty(blocks, page, 1, 1, torch.int8, gpu)
    rows = torch.tensor([2**32 + 15, 2**32 + 3, 2**32 - 1, 2**31 + 7, 5, blocks * page, -1], device=gpu)
    k = torch.tensor([1.0, -2.0, 3.0, -4.0, 5.0, 6.0, 7.0], device=gpu).view(7, 1, 1)
    append_quantized(k, -k, rows, pool)
    values, scales = quantise(k, torch.int8)
    want = torch.where((rows < blocks * page) & (rows >= 0), (values * scales[..., None]).view(7).to(gpu), 0.0)
    for got, sign in zip(read_quantized(pool, rows, torch.float32), (1, -1)):
        assert ((got.view(7).double() - sign * want).abs() <= 2.0**-24 * want.abs()).all()
    for i, r in enumerate(rows[:5].tolist()):
        assert pool.codes[r // page, 0, r % page, 0, 0].item() == values[i].item()
    assert pool.scales[2**28].count_nonzero().item() == 4 and pool.scales[0].count_nonzero().item() == 2
    tables = torch.tensor([[2**28, 0]], dtype=torch.int32, device=gpu)  # 16 rows past 2^32, two of them not zero
    query = torch.ones(1, 1, 1, device=gpu)
    small = QuantizedPool(*(t[tables[0].long()].contiguous() for t in (pool.codes, pool.scales)))
    lengths = torch.tensor([22], dtype=torch.int32, device=gpu)
    args = (query, small, torch.tensor([[0, 1]], dtype=torch.int32, device=gpu), lengths)
    check(attend_pages(query, pool, tables, lengths), args)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [8, 1])
def test_as_many_head_vectors_as_a_call_takes(gpu, dim):
    rows_n, page = 2**25, 16
    pool = QuantizedPool.empty(rows_n // page, page, 1, dim, torch.int8, gpu)
    gen = torch.Generator(device=gpu).manual_seed(dim)
    k = torch.randn(rows_n, 1, dim, generator=gen, device=gpu)
    rows = rows_n - 1 - torch.arange(rows_n, device=gpu)
    append_quantized(k, k, rows, pool)
    assert torch.equal(pool.scales[:, 0], pool.scales[:, 1]) and torch.equal(pool.codes[:, 0], pool.codes[:, 1])
    scale = (k.abs().amax(-1, keepdim=True).double() / 127).float()
    assert torch.equal(pool.scales[:, 0].reshape(-1).flip(0), scale.view(-1))
    for got in read_quantized(pool, rows, torch.float32):
        # half a code's step, and the scale's and the product's rounding
        assert ((got - k).abs() <= scale * 0.5 * (1 + 2.0**-16) + k.abs() * 2.0**-22).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,dim", [(2**24 + 3, 4), (2**24 - 1, 258)])
def test_prompt_of_many_rows(gpu, rows, dim):
    """Several rows to a workgroup, and as many workgroups as a launch has (one row each)."""
    heads = kv = 1
    qkv = torch.zeros(rows, 3 * dim, dtype=torch.bfloat16, device=gpu)
    picked = torch.tensor([0, 1, 127, 128, 2**23 + 1, rows - 129, rows - 2, rows - 1], device=gpu)
    gen = torch.Generator().manual_seed(dim)
    some = torch.randn(len(picked), 3 * dim, generator=gen).to(torch.bfloat16).to(gpu)
    qkv[picked] = some
    wq, wk = (torch.rand(dim, generator=gen).to(torch.bfloat16).to(gpu) for _ in range(2))
    positions = torch.arange(rows, device=gpu)
    q, k, v = norm_rotary_split(qkv, wq, wk, 1e-6, positions, heads, kv, dim, 1e6)
    (want_q, want_k), (size_q, size_k), want_v = norm_formula(some, wq, wk, 1e-6, picked, heads, kv, dim, 1e6)
    check_norm(q[picked], want_q, size_q, torch.bfloat16)
    check_norm(k[picked], want_k, size_k, torch.bfloat16)
    assert torch.equal(v[picked].double().cpu(), want_v)
    for x in (q, k, v):  # a row of zeros is one
        x[picked] = 0
        assert not x.any()


@pytest.mark.gpu
@pytest.mark.parametrize("code,dtype", [("int8", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("wide", [200, 20_000])
def test_graphs_that_share_their_memory(gpu, code, dtype, wide):
    """Two captured calls on one memory pool, whose workspaces lie in the same place: replayed in
    turn, with other lengths and eager calls between."""
    a = case(2, 14, 2, 64, 16, [1900, 700], code, dtype, gpu, wide=wide)
    b = case(3, 8, 4, 128, 16, [1500, 900, 31], code, dtype, gpu, wide=wide)
    graphs, outs = [], [torch.empty_like(a[0]), torch.empty_like(b[0])]
    for args, out in zip((a, b), outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            attend_pages(*args, out=out)
        graphs.append(graph)
    for step in range(4):
        wants = [attend_pages(*a), attend_pages(*b)]
        for out in outs:
            out.fill_(9.0)
        for i in (0, 1, 1, 0):
            graphs[i].replay()
            assert torch.equal(outs[i], wants[i])
        a[3][0] -= 401
        b[3][1] -= 290
        b[0].neg_()
