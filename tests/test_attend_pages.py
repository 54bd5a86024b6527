"""Attention over page tables (attend_pages) against softmax attention in 64 bits, with every
row it may not use filled with NaN, and the calls it refuses."""

import ctypes
import shutil
import subprocess

import pytest
import torch

from mini_hisparse_amd import _lib, build
from mini_hisparse_amd.quantized import QuantizedPool, append_quantized
from mini_hisparse_amd.row_kernels import attend_pages, attend_rows

PLAIN = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def rows_of(values, code):
    """(codes or plain values, scales or None) of random rows [blocks, 2, P, Hkv, D]."""
    if code in PLAIN:
        return values.to(PLAIN[code]), None
    top = 127.0 if code == "int8" else 448.0
    scales = values.abs().amax(-1) / top
    q = values / scales[..., None]
    return (q.round() if code == "int8" else q).clamp(-top, top).to(CODES[code]), scales


def case(batch, heads, kv, dim, page, lengths, code, dtype, device, seed=0, absent=0.0, per_head=False, spare=3,
         amplitude=1.0, wide=2):
    """A batch whose tables are scattered over the pool.  Rows no request may use -- past a
    length, of blocks in no table -- are NaN (for int8 codes: NaN scales and any codes)."""
    gen = torch.Generator().manual_seed(seed + dim + page + sum(lengths))
    lists = kv if per_head else 1
    pages = [-(-n // page) for n in lengths]
    width = max(1, max(pages)) + wide
    blocks = lists * sum(pages) + spare
    order = torch.randperm(blocks, generator=gen)
    tables = torch.randint(-3, blocks + 3, (batch, lists, width), generator=gen)  # past the pages: anything
    values = torch.randn(blocks, 2, page, kv, dim, generator=gen)
    values[..., : max(1, dim // 50)] *= 8
    values[:, 1] *= amplitude
    used = torch.zeros(blocks, page, kv, dtype=torch.bool)
    taken = 0
    for b, n in enumerate(lengths):
        for h in range(lists):
            mine = order[taken : taken + pages[b]]
            taken += pages[b]
            tables[b, h, : pages[b]] = mine
            for i, block in enumerate(mine.tolist()):
                gone = absent and torch.rand((), generator=gen).item() < absent
                if gone:
                    tables[b, h, i] = [-1, blocks, -(2**31), 2**31 - 1][i % 4]
                elif per_head:
                    used[block, : n - i * page, h] = True
                else:
                    used[block, : n - i * page] = True
    stored, scales = rows_of(values, code)
    junk = ~used[:, None].expand(-1, 2, -1, -1)
    if scales is None:
        stored[junk] = float("nan")
    else:
        scales[junk] = float("nan")
        raw = stored.view(torch.int8)
        raw[junk] = 0x7F  # e4m3's NaN, int8's 127
    query = torch.randn(batch, heads, dim, generator=gen).to(PLAIN[dtype])
    tables = tables.to(torch.int32) if per_head else tables[:, 0].to(torch.int32)
    pool = stored.to(device) if scales is None else QuantizedPool(stored.to(device), scales.to(device))
    return query.to(device), pool, tables.to(device), torch.tensor(lengths, dtype=torch.int32, device=device)


def store_of(pool):
    """The pool's values in 64 bits."""
    if not isinstance(pool, QuantizedPool):
        return pool.cpu().double()
    return pool.codes.cpu().float().double() * pool.scales.cpu().double()[..., None]


def formula(query, pool, tables, lengths):
    """(out, weighted sum of |V|, largest sum of |q K| D^-1/2, largest |score|, tokens) in 64 bits."""
    store = store_of(pool)
    query, tables, lengths = query.cpu().double(), tables.cpu().long(), lengths.cpu().tolist()
    blocks, _, page, kv, dim = store.shape
    batch, heads, _ = query.shape
    group = heads // kv
    out, weight, size, top, count = (torch.zeros(batch, heads, n, dtype=torch.float64) for n in (dim, dim, 1, 1, 1))
    for b, n in enumerate(lengths):
        n = max(0, min(n, tables.shape[-1] * page))
        token = torch.arange(n)
        for h in range(kv):
            table = tables[b, h] if tables.dim() == 3 else tables[b]
            block = table[token // page]
            keep = (block >= 0) & (block < blocks)
            if not keep.any():
                continue
            k, v = (store[block[keep], plane, (token % page)[keep], h] for plane in (0, 1))
            rows = slice(h * group, (h + 1) * group)
            q = query[b, rows]
            scores = q @ k.T * dim**-0.5
            p = torch.softmax(scores, -1)
            out[b, rows], weight[b, rows] = p @ v, p @ v.abs()
            size[b, rows] = (q.abs() @ k.abs().T).amax(-1, keepdim=True) * dim**-0.5
            top[b, rows] = scores.abs().amax(-1, keepdim=True)
            count[b, rows] = float(keep.sum())
    return out, weight, size, top, count


def check(got, args, held=None):
    """|error| <= half a step of the dtype, and before that rounding the weights' error times
    the weighted |V| twice (numerator and sum): with u = 2^-24, a score is off by at most
    D u of its sum of magnitudes, three roundings of the score and 4 u of its size again in
    the exponential's argument; the exponential by 4 u; the sums of n tokens and their
    rescalings by (n + 16) u; a weight held as the sum of two 16-bit parts by the product of
    their half steps (bfloat16 2^-8 2^-8, float16 2^-11 2^-11 and half a subnormal step,
    2^-25, of the largest weight), of three bfloat16 parts (float32 queries) by 2^-24."""
    query, pool = args[0], args[1]
    want, weight, size, top, count = formula(*args)
    u, dim = 2.0**-24, query.shape[-1]
    f16 = not isinstance(pool, QuantizedPool) and query.dtype == torch.float16
    if held is None:
        held = 2.0**-24 if query.dtype == torch.float32 else 2.0**-22 if f16 else 2.0**-16
    weights = (dim + 4) * u * size + 8 * u * top + 4 * u + (count + 16) * u + held
    tol = torch.finfo(query.dtype).eps / 2 * want.abs() + 2 * weights * weight
    # float32 has no normal value below 2^-126 and no value below 2^-149: a weight smaller
    # than 2^-126 of the largest may be held as 0, so each of the n tokens may miss 2^-126 of
    # the largest |V| (q of 1000 sigma: the true output is 1e-45 where the winner's V is 0)
    largest = (store_of(pool).nan_to_num(0.0).abs().amax()).item()
    tol = tol + count * 2.0**-126 * largest + (count * 2.0**-25 * largest if f16 else 0)
    if query.dtype == torch.float16:
        tol = tol + 2.0**-25
    error = (got.double().cpu() - want).abs()
    over = error > tol
    assert not over.any(), (error[over].max().item(), tol[over].max().item())


SHAPES = [(28, 4, 128), (14, 2, 64), (4, 2, 32), (8, 8, 128), (16, 1, 128), (20, 1, 64), (36, 1, 128), (12, 3, 96),
          (5, 5, 80), (3, 1, 256), (2, 2, 512), (2, 1, 20), (3, 3, 7), (1, 1, 1), (22, 11, 64), (2, 1, 511)]
POOLS = [("int8", "bf16"), ("e4m3", "bf16"), ("int8", "f16"), ("e4m3", "f16"), ("int8", "f32"), ("e4m3", "f32"),
         ("bf16", "bf16"), ("f16", "f16"), ("f32", "f32")]


# a table of this many columns more goes over the launch for long histories
WIDE = 20_000


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [2, WIDE])
@pytest.mark.parametrize("code,dtype", POOLS)
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
def test_matches_the_formula(gpu, heads, kv, dim, code, dtype, wide):
    args = case(3, heads, kv, dim, 16, [333, 1, 97], code, dtype, gpu, wide=wide)
    check(attend_pages(*args), args)


@pytest.mark.gpu
@pytest.mark.parametrize("code,dtype", [("int8", "bf16"), ("e4m3", "f32"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("page", [1, 3, 8, 12, 16, 32, 48, 64, 256])
@pytest.mark.parametrize("wide", [2, 300_000])
def test_page_sizes(gpu, page, code, dtype, wide):
    args = case(2, 14, 2, 64, page, [401, 256], code, dtype, gpu, wide=wide)
    check(attend_pages(*args), args)
    args = case(1, 8, 4, 128, page, [63], code, dtype, gpu, wide=wide)
    check(attend_pages(*args), args)


@pytest.mark.gpu
@pytest.mark.parametrize("code,dtype", [("int8", "bf16"), ("e4m3", "f16"), ("f16", "f16"), ("f32", "f32")])
def test_lengths_around_the_tiles(gpu, code, dtype):
    """Lengths on both sides of a page, a tile and a split, and none at all."""
    for wide in (2, WIDE):
        for lengths in ([0], [1], [2], [15, 16, 17], [31, 32, 33], [63, 64, 65, 0, 127, 128, 129],
                        [255, 0, 256, 257], [511, 512, 513], [2047, 2048, 2049], [4000, 3, 0]):
            args = case(len(lengths), 8, 2, 128, 16, lengths, code, dtype, gpu, wide=wide)
            got = attend_pages(*args)
            check(got, args)
            for b, n in enumerate(lengths):
                assert n or (got[b] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("code,dtype", [("int8", "bf16"), ("e4m3", "bf16"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("page", [16, 5])
def test_absent_pages_and_tables_per_head(gpu, page, code, dtype):
    for per_head in (False, True):
        for absent in (0.0, 0.4, 1.0):
            for wide in (2, WIDE):
                args = case(3, 14, 2, 64, page, [700, 33, 16], code, dtype, gpu, absent=absent, per_head=per_head,
                            wide=wide)
                got = attend_pages(*args)
                check(got, args)
                assert absent < 1.0 or (got == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "bf16"])
def test_uneven_batches(gpu, code):
    """One long history among many short ones, and the other way round."""
    for lengths in ([9000] + [5] * 20, [3000] * 5 + [0, 1], [40] * 70):
        args = case(len(lengths), 14, 2, 64, 16, lengths, code, "bf16", gpu)
        check(attend_pages(*args), args)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim,page", [(4, 2, 32, 16), (5, 1, 64, 5)])
@pytest.mark.parametrize("batch", [64, 65, 128, 1024, 1100, 2049])
def test_many_requests(gpu, batch, heads, kv, dim, page):
    """Batches on both sides of a wave's lanes and of the schedule's workgroup, with empty
    requests, long ones first, last and alone; captured, with other lengths per replay."""
    gen = torch.Generator().manual_seed(batch)
    short = torch.randint(0, 60, (batch,), generator=gen)
    short[::7] = 0
    longest = 4000
    first, last, none = short.clone(), short.clone(), torch.zeros_like(short)
    first[0], first[1] = longest, 1
    last[-1], last[batch // 2] = longest, 2500
    most = torch.stack([first, last, short]).amax(0)
    query, pool, tables, lengths = args = case(batch, heads, kv, dim, page, most.tolist(), "int8", "bf16", gpu, wide=200)
    assert tables.shape[-1] * page > 32 * 32
    check(attend_pages(*args), args)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(query)
    with torch.cuda.graph(graph):
        attend_pages(*args, out=out)
    for now in (first, none, last, short):
        lengths.copy_(now)
        out.fill_(7.0)
        graph.replay()
        assert out.isfinite().all() and torch.equal(out, attend_pages(*args))
        check(out, args)


@pytest.mark.gpu
@pytest.mark.parametrize("code,dtype", [("int8", "bf16"), ("int8", "f16"), ("e4m3", "f32"), ("f16", "f16"),
                                        ("bf16", "bf16")])
def test_small_and_large_values(gpu, code, dtype):
    """V rows of any size: the weights times a scale keep their precision (float16 queries too),
    and float16's subnormal values count (1e-6 is 17 of their steps)."""
    for amplitude in (1e-6, 1e-3, 2000.0):
        for wide in (2, WIDE):
            args = case(2, 8, 2, 128, 16, [300, 1], code, dtype, gpu, amplitude=amplitude, wide=wide)
            check(attend_pages(*args), args)


@pytest.mark.gpu
def test_sharp_and_flat_scores(gpu):
    for size in (0.0, 30.0, 1000.0):
        args = case(2, 28, 4, 128, 16, [500, 77], "int8", "f32", gpu)
        args = (args[0] * size, *args[1:])
        check(attend_pages(*args), args)


@pytest.mark.gpu
@pytest.mark.parametrize("code,dtype", POOLS)
def test_nan_in_a_used_row_reaches_its_heads_alone(gpu, code, dtype):
    for dim in (64, 96):
        query, pool, tables, lengths = case(2, 4, 2, dim, 16, [40, 40], code, dtype, gpu)
        block = tables[0, 1].item()
        (pool.scales if code in CODES else pool)[block, 0, 3, 1] = float("nan")  # a key of request 0, KV head 1
        got = attend_pages(query, pool, tables, lengths)
        assert got[0, 2:].isnan().all() and got[0, :2].isfinite().all() and got[1].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("code,dtype", POOLS)
@pytest.mark.parametrize("dim", [80, 96, 256])
def test_pages_masks_and_nan_at_other_head_dims(gpu, dim, code, dtype):
    """80 of the head dim run on the vector unit, 96 in two column parts of a V row, 256 in
    workgroups of half the waves (float32 on the vector unit)."""
    for page in (1, 12, 16, 48):
        for wide in (2, WIDE):
            args = case(3, 6, 3, dim, page, [401, 0, 63], code, dtype, gpu, absent=0.3, per_head=page > 1, wide=wide)
            check(attend_pages(*args), args)
    args = case(2, 40, 2, dim, 16, [2100, 700], code, dtype, gpu)  # several parts of a request, 16 heads and 4 of a unit
    check(attend_pages(*args), args)
    query, pool, tables, lengths = case(2, 4, 2, dim, 16, [40, 40], code, dtype, gpu)
    block = tables[0, 1].item()
    (pool.scales if code in CODES else pool)[block, 1, 3, 1] = float("nan")  # a value of request 0, KV head 1
    got = attend_pages(query, pool, tables, lengths)
    assert got[0, 2:].isnan().any() and got[0, :2].isfinite().all() and got[1].isfinite().all()


@pytest.mark.gpu
def test_lengths_past_the_tables_and_below_zero(gpu):
    query, pool, tables, lengths = case(2, 4, 2, 64, 16, [64, 48], "int8", "bf16", gpu, spare=1)
    tables = tables[:, :3].contiguous()  # 48 tokens at most
    want = attend_pages(query, pool, tables, torch.tensor([48, 48], dtype=torch.int32, device=gpu))
    got = attend_pages(query, pool, tables, torch.tensor([2**31 - 1, 49], dtype=torch.int32, device=gpu))
    assert torch.equal(got, want)
    none = attend_pages(query, pool, tables, torch.tensor([-1, -(2**31)], dtype=torch.int32, device=gpu))
    assert (none == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("code,dtype", [("int8", "bf16"), ("bf16", "bf16"), ("f32", "f32")])
def test_strides_outputs_and_misaligned_buffers(gpu, code, dtype):
    query, pool, tables, lengths = case(3, 8, 2, 64, 16, [100, 7, 50], code, dtype, gpu)
    want = attend_pages(query, pool, tables, lengths)
    wide = torch.zeros(3, 8, 100, dtype=query.dtype, device=gpu)
    wide[..., 3:67] = query
    assert torch.equal(attend_pages(wide[..., 3:67], pool, tables, lengths), want)
    turned = query.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(attend_pages(turned, pool, tables, lengths), want)
    assert torch.equal(attend_pages(query.repeat_interleave(2, 2)[..., ::2], pool, tables, lengths), want)
    spread = torch.full((3, 2 * tables.shape[1]), 7, dtype=torch.int32, device=gpu)
    spread[:, : tables.shape[1]] = tables
    assert torch.equal(attend_pages(query, pool, spread[:, : tables.shape[1]], lengths), want)
    shared = tables[:, None].expand(-1, 2, -1)  # the same list for both KV heads
    assert torch.equal(attend_pages(query, pool, shared, lengths), want)
    guarded = torch.full((5, 8, 64), 9.0, dtype=query.dtype, device=gpu)
    got = attend_pages(query, pool, tables, lengths, out=guarded[1:4])
    assert got.data_ptr() == guarded[1].data_ptr() and torch.equal(got, want)
    assert (guarded[0] == 9).all() and (guarded[4] == 9).all()
    # a pool that starts at an odd element: the element-wise kernel, on a workspace of any size
    store = pool.codes if code in CODES else pool
    room = torch.empty(store.numel() + 1, dtype=torch.int8 if code in CODES else store.dtype, device=gpu)
    moved = room[1:].view(store.shape)
    moved.copy_(store.view(room.dtype))
    moved = QuantizedPool(moved.view(store.dtype), pool.scales) if code in CODES else moved
    for columns in (tables.shape[1], 400, 30_000):  # one part, a few, the long launch
        padded = torch.full((3, columns), -1, dtype=torch.int32, device=gpu)
        padded[:, : tables.shape[1]] = tables
        args = (query, moved, padded, lengths)
        check(attend_pages(*args), args)


@pytest.mark.gpu
@pytest.mark.parametrize("code,dtype", [("int8", "bf16"), ("f32", "f32")])
def test_one_request_of_a_batch_does_not_change_another(gpu, code, dtype):
    """The same request gives the same bits twice, alone or beside others of its length."""
    args = case(4, 14, 2, 64, 16, [900, 900, 900, 900], code, dtype, gpu)
    first, again = attend_pages(*args), attend_pages(*args)
    assert torch.equal(first, again)


@pytest.mark.gpu
def test_pool_past_32_bit_offsets(gpu):
    blocks, page, kv, dim = 140_000, 16, 8, 128  # 4.6e9 codes
    pool = QuantizedPool.empty(blocks, page, kv, dim, torch.int8, gpu)
    tables = torch.tensor([[blocks - 1, 70_000], [65_537, 131_073]], dtype=torch.int32, device=gpu)
    lengths = torch.tensor([29, 32], dtype=torch.int32, device=gpu)
    rows = (tables.long()[:, :, None] * page + torch.arange(page, device=gpu)).flatten()
    k, v = (torch.randn(len(rows), kv, dim, device=gpu) for _ in range(2))
    append_quantized(k, v, rows, pool)
    query = torch.randn(2, 16, dim, device=gpu).to(torch.bfloat16)
    got = attend_pages(query, pool, tables, lengths)
    order = torch.tensor([[2, 1], [0, 3]], dtype=torch.int32, device=gpu)  # the same rows in a small pool
    small = QuantizedPool(*(t[tables.long()[[1, 0, 0, 1], [0, 1, 0, 1]]].contiguous()
                            for t in (pool.codes, pool.scales)))
    args = (query, small, order, lengths)
    check(got, args)


@pytest.mark.gpu
def test_agrees_with_attend_rows(gpu):
    """The same rows by page table and by row list, over one plain pool."""
    from mini_hisparse_amd.config import CacheConfig

    query, pool, tables, lengths = case(2, 28, 4, 128, 16, [320, 320], "bf16", "bf16", gpu)
    config = CacheConfig(gpu_pages=pool.shape[0], page_size=16, kv_heads=4, head_dim=128, device=gpu,
                         dtype=torch.bfloat16)
    rows = (tables.long()[:, :20, None] * 16 + torch.arange(16, device=gpu)).flatten(1)
    by_rows = attend_rows(query, pool, rows, config)
    args = (query, pool, tables, lengths)
    check(by_rows, args, held=2.0**-8)  # its weights are held in one bfloat16 part
    check(attend_pages(*args), args)


@pytest.mark.gpu
@pytest.mark.parametrize("code,dtype", [("int8", "bf16"), ("bf16", "bf16"), ("f32", "f32")])
def test_streams_and_captured_replays(gpu, code, dtype):
    """Calls at once on two streams, and captured calls replayed with other tables, lengths and
    queries, with eager calls between the replays; two graphs replayed at once."""
    a = case(3, 14, 2, 64, 16, [2000, 1300, 5], code, dtype, gpu)
    b = case(2, 14, 2, 64, 16, [1500, 900], code, dtype, gpu, seed=1)
    want_a, want_b = attend_pages(*a), attend_pages(*b)
    main = torch.cuda.current_stream(torch.device(gpu))
    streams = [torch.cuda.Stream(torch.device(gpu)) for _ in range(2)]
    for s in streams:
        s.wait_stream(main)
    results = []
    for _ in range(4):
        for s, args in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                results.append(attend_pages(*args))
    for s in streams:
        main.wait_stream(s)
    for i, r in enumerate(results):
        assert torch.equal(r, (want_a, want_b)[i % 2])
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph, args in zip(graphs, (a, b)):
        with torch.cuda.graph(graph):
            outs.append(attend_pages(*args))
    for step in range(4):
        a[3][0] -= 301 * step  # shorter histories
        b[0].normal_()
        want_a, want_b = attend_pages(*a), attend_pages(*b)
        for s in streams:
            s.wait_stream(main)
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        for s in streams:
            main.wait_stream(s)
        assert torch.equal(outs[0], want_a) and torch.equal(outs[1], want_b)


def behind_one_key(heads, kv, dim, page, lengths, nats, amplitude, device, wide):
    """float16 requests whose first key stands ``nats`` above every other and has the value 0; the
    others, with keys near 0, have values of one sign, so that nothing but their small weights is left."""
    query, pool, tables, lengths = case(len(lengths), heads, kv, dim, page, lengths, "f16", "f16", device, wide=wide)
    group = heads // kv
    query = query[:, ::group].repeat_interleave(group, 1).contiguous()  # one direction for the heads of a group
    pool[:, 0] *= 0.01
    pool[:, 1] = pool[:, 1].abs().clamp(max=1.0) * amplitude
    for b in range(len(query)):
        block = tables[b, 0].item()
        q = query[b, ::group].double()
        pool[block, 0, 0] = (q * (nats * dim**0.5 / q.square().sum(-1, keepdim=True))).half()
        pool[block, 1, 0] = 0
    return query, pool, tables, lengths


def check_float16(got, args):
    """As ``check``, but for what float16's range may cost a weight: its two parts hold it to 2^-22 of
    itself, and to 2^-45 of the largest (half a subnormal step, 2^-25, of weights held at 2^9, whose
    remainders are held at 2^11)."""
    query, pool = args[0], args[1]
    want, weight, size, top, count = formula(*args)
    u, dim = 2.0**-24, query.shape[-1]
    weights = (dim + 4) * u * size + 8 * u * top + 4 * u + (count + 16) * u + 2.0**-22
    largest = store_of(pool).nan_to_num(0.0).abs().amax().item()
    tol = 2.0**-11 * want.abs() + 2.0**-25 + 2 * weights * weight + count * 2.0**-45 * largest
    error = (got.double().cpu() - want).abs()
    over = error > tol
    assert not over.any(), (error[over].max().item(), tol[over].max().item())


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 32), (6, 2, 64), (3, 3, 96), (14, 2, 128), (2, 2, 256), (2, 1, 80)])
@pytest.mark.parametrize("nats", [10.0, 15.0, 16.0, 17.5, 20.0, 24.0])
def test_small_weights_of_float16_pools_count(gpu, heads, kv, dim, nats):
    """A first key that leads a history by far and has no value: the output is what the small weights
    of all other tokens leave, in a tile, in a wave's tiles and in the long launch's."""
    for page, lengths, wide in ((16, [32, 2], 2), (16, [700, 97], 2), (5, [300], 2), (16, [20_000, 33], WIDE)):
        for amplitude in (1.0, 60_000.0):
            args = behind_one_key(heads, kv, dim, page, lengths, nats, amplitude, gpu, wide)
            check_float16(attend_pages(*args), args)


@pytest.mark.gpu
def test_float16_scores_of_any_size(gpu):
    """Scores that float32 holds only to 2^-3 .. 2^8: the weights stay finite, the largest one wins."""
    for size in (1e3, 1e5, 6e6, 6e7):
        query, pool, tables, lengths = case(2, 8, 2, 128, 16, [300, 40], "f16", "f16", gpu)
        used = torch.where(pool.isnan(), pool, pool.sign() * pool.abs().clamp(0.25, 2.0))
        pool[:, 0] = used[:, 0] * size**0.5
        query = query.sign() * query.abs().clamp(0.25, 2.0) * size**0.5
        got = attend_pages(query, pool, tables, lengths)
        want, _, magnitude, _, _ = formula(query, pool, tables, lengths)
        assert got.isfinite().all()
        # a head whose best key leads by more than the scores' rounding has that key's value
        store, group = store_of(pool), 4
        for b, n in enumerate(lengths.tolist()):
            token = torch.arange(n)
            block = tables[b].cpu().long()[token // 16]
            for h in range(8):
                k, v = (store[block, plane, token % 16, h // group] for plane in (0, 1))
                scores = (k @ query[b, h].cpu().double()) * 128**-0.5
                first, second = scores.topk(2).values
                if first - second > 20 + 2 * 140 * 2.0**-24 * magnitude[b, h].item():
                    best = v[scores.argmax()]
                    assert ((got[b, h].cpu().double() - best).abs() <= 2.0**-11 * best.abs() + 1e-5).all()


def test_refusals_without_a_gpu():
    pool = QuantizedPool.empty(4, 16, 2, 8, torch.int8, "cpu")
    plain = torch.zeros(4, 2, 16, 2, 8)
    query = torch.zeros(3, 4, 8)
    tables, lengths = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    bad = [
        ("query", (query[0], pool, tables, lengths)),
        ("query", (query, pool.codes[0], tables, lengths)),
        ("head_dim", (query[..., :4], pool, tables, lengths)),
        ("multiple", (query[:, :3], pool, tables, lengths)),
        ("query", (query[:0], pool, tables[:0], lengths[:0])),
        ("dtype", (query.double(), pool, tables, lengths)),
        ("query dtype", (query.half(), plain, tables, lengths)),
        ("contiguous", (query, plain.transpose(2, 3).contiguous().transpose(2, 3), tables, lengths)),
        ("tables", (query, pool, tables.long(), lengths)),
        ("tables", (query, pool, tables[:2], lengths)),
        ("tables", (query, pool, tables[:, :0], lengths)),
        ("tables", (query, pool, tables.repeat(1, 2)[:, ::2], lengths)),
        ("tables", (query, pool, tables[:, None].expand(-1, 3, -1), lengths)),
        ("lengths", (query, pool, tables, lengths.long())),
        ("lengths", (query, pool, tables, lengths[:2])),
        ("lengths", (query, pool, tables, lengths.repeat(2)[::2])),
        ("ROCm", (query, pool, tables, lengths)),
    ]
    for match, args in bad:
        with pytest.raises(ValueError, match=match):
            attend_pages(*args)
    with pytest.raises(ValueError, match="out"):
        attend_pages(query, pool, tables, lengths, out=torch.zeros(3, 4, 16)[..., ::2])


def test_entry_point_refusals_without_a_gpu():
    lib = _lib.load()
    buffer = ctypes.create_string_buffer(256)
    at = ctypes.addressof(buffer)
    at += -at % 16

    def call(q=at, qd=2, pool=at, scales=at, code=3, blocks=4, page=16, kv=1, dim=64, tables=at, pages=1000,
             lengths=at, batch=1, heads=2, out=at, ws=at, nbytes=1 << 40):
        return lib.hs_attend_pages(q, heads * dim, dim, qd, pool, scales, code, blocks, page, kv, dim, tables, pages,
                                   0, pages, lengths, batch, heads, out, heads * dim, dim, ws, nbytes, None)

    for bad in (dict(q=None), dict(qd=3), dict(pool=None), dict(scales=None), dict(code=2), dict(code=5), dict(code=0),
                dict(blocks=0), dict(blocks=2**31), dict(page=0), dict(kv=0), dict(kv=3), dict(dim=0), dict(dim=513),
                dict(tables=None), dict(pages=0), dict(pages=2**31), dict(page=2**20, pages=2**12), dict(lengths=None),
                dict(batch=0), dict(batch=70_000), dict(heads=0), dict(out=None), dict(ws=None), dict(nbytes=16),
                dict(ws=at + 8)):
        assert call(**bad) == -1, bad
        assert lib.hs_last_error()
    size = lib.hs_attend_pages_workspace_bytes
    assert size(2, 3, 0, 1, 1, 64, 16, 1) == 256
    assert size(2, 3, 4, 14, 2, 64, 16, 10) == 0 and size(2, 3, 4, 14, 2, 64, 16, 1000) > 0  # one part, several


PARTS = r"""
#include "page_parts.h"
#include <vector>
using namespace hs;

// Parts of B requests of n tokens and, of the first, `first`, at the sure size: by the schedule
// written out (lanes <= 0) and by that of a wave's lanes (whose sum is held in fp32).
extern "C" int64_t parts_at_the_sure_size(int64_t B, int64_t n, int64_t first, int64_t target, int64_t min_tiles,
                                          int lanes) {
  const int64_t limit = 0x7fffffff;
  const int32_t rest = tiles_of(clamp_length(n, limit)), one = tiles_of(clamp_length(first, limit));
  const int64_t total = one + (B - 1) * static_cast<int64_t>(rest);
  const uint32_t room = sure_room(target, B);
  const uint32_t sure = lanes > 0 ? sure_size(static_cast<float>(total), room) : sure_size(total, room);
  const uint32_t per = tried_size(sure, sure, 0, static_cast<uint32_t>(min_tiles));
  if (B == 1 || lanes < 0) return parts_of(one, per);  // of the first request alone
  return parts_of(one, per) + (B - 1) * static_cast<int64_t>(parts_of(rest, per));
}
"""


@pytest.fixture(scope="module")
def part_arithmetic(tmp_path_factory):
    if shutil.which(build.HIPCC) is None:
        pytest.skip("hipcc is not installed")
    folder = tmp_path_factory.mktemp("parts")
    (folder / "parts.hip").write_text(PARTS)
    command = [build.HIPCC, "--offload-host-only", "-shared", "-fPIC", "-O1", f"-I{build.CSRC}",
               str(folder / "parts.hip"), "-o", str(folder / "parts.so")]
    subprocess.run(command, check=True, capture_output=True)
    count = ctypes.CDLL(str(folder / "parts.so")).parts_at_the_sure_size
    count.restype, count.argtypes = ctypes.c_int64, [ctypes.c_int64] * 5 + [ctypes.c_int]
    return count


def test_parts_stay_within_their_slots_at_any_length(part_arithmetic):
    """The sure size gives at most target + B parts, for which the workspace has slots, also where
    the tiles of all requests are more than 32 bits hold."""
    longest = 2**31 - 1
    for batch in (1, 2, 63, 64, 65, 66, 128, 512, 16_384, 16_385, 32_769, 65_535):
        for target in (1, 2, 3, 7, 64, 128, 256, 512):
            for n in (0, 1, 33, 4096, 10**6, 2**30, 2**30 + 2**25, longest):
                for first in (0, n, 2 * n // 3, longest):
                    for lanes in (0, 1) if batch <= 64 else (0,):
                        parts = part_arithmetic(batch, n, first, target, 1, lanes)
                        assert batch <= parts <= target + batch, (batch, target, n, first, lanes, parts)
                    # the merge holds the weights of one request's slots
                    assert part_arithmetic(batch, n, first, target, 1, -1) <= max(1, target)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim,code,dtype,lengths", [
    (1, 1, 80, "int8", "bf16", [262_139]),  # 1024 splits of the general kernel, by four columns and by one
    (2, 1, 81, "bf16", "bf16", [262_140]),
    (2, 1, 32, "int8", "bf16", [70_000]),  # 256 parts of the long launch
    (2, 1, 32, "f16", "f16", [140_000] + [0] * 60 + [17] * 10),  # nearly 512 of one request
])
def test_as_many_slots_as_a_request_can_have(gpu, heads, kv, dim, code, dtype, lengths):
    args = case(len(lengths), heads, kv, dim, 16, lengths, code, dtype, gpu)
    check(attend_pages(*args), args)


def formula_on_the_device(query, pool, tables, lengths):
    """``formula`` for histories of many tokens: the same sums in 64 bits, on the device; a table's pages
    may repeat."""
    codes, scales = (pool.codes, pool.scales) if isinstance(pool, QuantizedPool) else (pool, None)
    store = codes.float().double() if scales is None else codes.float().double() * scales.double()[..., None]
    store = store.nan_to_num(0.0)  # the rows that no request may use
    blocks, _, page, kv, dim = store.shape
    batch, heads, _ = query.shape
    parts = [torch.zeros(batch, heads, n, dtype=torch.float64, device=query.device) for n in (dim, dim, 1, 1, 1)]
    head = torch.arange(kv, device=query.device)[:, None]
    for b, n in enumerate(lengths.tolist()):
        token = torch.arange(n, device=query.device)
        block = tables[b].long().expand(kv, -1)[:, token // page]  # [kv, n]
        keep = ((block >= 0) & (block < blocks))[:, None]
        k, v = (store[block.clamp(0, blocks - 1), plane, token % page, head] * keep.transpose(1, 2) for plane in (0, 1))
        q = query[b].double().view(kv, -1, dim)
        scores = ((q @ k.transpose(1, 2)) * dim**-0.5).masked_fill(~keep, float("-inf"))
        p = torch.softmax(scores, -1).nan_to_num(0.0)  # no token at all
        size = (q.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True) * dim**-0.5
        top = scores.masked_fill(~keep, 0.0).abs().amax(-1, keepdim=True)
        count = keep.sum(-1, keepdim=True).double().expand(top.shape)
        for part, x in zip(parts, (p @ v, p @ v.abs(), size, top, count)):
            part[b] = x.reshape(heads, -1)
    return [x.cpu() for x in parts]


def long_waves(tiles, batch, kv, dim, page, code, dtype, device, per_head=False, holes=()):
    """A batch for which a wave of the long launch has about ``tiles`` tiles (one head a KV head; 128
    workgroups of two waves for each of four of them): equal parts, two requests' worth of parts at least.
    Pages repeat; those from ``holes`` are absent.  Blocks 0 and 1 are in no table and NaN."""
    gen = torch.Generator().manual_seed(tiles + batch + dim + page)
    tokens = tiles * 2 * 32 * 128 // batch
    lengths = [tokens - (7 * b) % 29 for b in range(batch)]  # the last tile and half of a page in part
    blocks, width, lists = 300, -(-tokens // page) + 3, kv if per_head else 1
    tables = torch.randint(2, blocks, (batch, lists, width), generator=gen)
    for first, last in holes:
        tables[:, :, first:last] = torch.tensor([-1, blocks, 2**31 - 1])[torch.arange(last - first) % 3]
    values = torch.randn(blocks, 2, page, kv, dim, generator=gen)
    stored, scales = rows_of(values, code)
    (stored if scales is None else scales)[:2] = float("nan")
    tables = (tables if per_head else tables[:, 0]).to(torch.int32).to(device)
    pool = stored.to(device) if scales is None else QuantizedPool(stored.to(device), scales.to(device))
    query = torch.randn(batch, kv, dim, generator=gen).to(PLAIN[dtype]).to(device)
    return query, pool, tables, torch.tensor(lengths, dtype=torch.int32, device=device)


def check_long(got, args):
    """``check``'s bound (float16 pools as in ``check_float16``) against the sums on the device."""
    query, pool = args[0], args[1]
    want, weight, size, top, count = formula_on_the_device(*args)
    u, dim, plain = 2.0**-24, query.shape[-1], not isinstance(pool, QuantizedPool)
    held = 2.0**-24 if query.dtype == torch.float32 else 2.0**-22 if plain and query.dtype == torch.float16 else 2.0**-16
    weights = (dim + 4) * u * size + 8 * u * top + 4 * u + (count + 16) * u + held
    tol = torch.finfo(query.dtype).eps / 2 * want.abs() + 2 * weights * weight
    if query.dtype == torch.float16:
        tol = tol + 2.0**-25 + count * 2.0**-45 * 9.0  # no |V| of these is above 9
    error = (got.double().cpu() - want).abs()
    over = error > tol
    assert not over.any(), (error[over].max().item(), tol[over].max().item())


@pytest.mark.gpu
@pytest.mark.parametrize("code,dtype", [("int8", "bf16"), ("e4m3", "f16"), ("bf16", "bf16"), ("f16", "f16"),
                                        ("f32", "f32")])
@pytest.mark.parametrize("tiles", [31, 32, 33, 64, 70])
def test_waves_of_more_tiles_than_a_batch_of_table_entries(gpu, tiles, code, dtype):
    """A wave reads the table for 32 of its tiles at a time: one batch, exactly and in part, two, and
    a third in part; absent pages in the middle of a batch, over a whole one, at the end."""
    pages = tiles * 2 * 32 * 128 // 64 // 16  # of a request of 64, whose two parts are tiles * 4 pages each
    half, third = pages // 2, pages // 3  # 128 pages are a wave's 32 tiles and its neighbour's
    for batch, holes in ((64, ()), (63, ()), (80, ()),
                         (64, ((5, 9), (third, third + 9), (pages - 20, pages))),
                         (64, ((0, half),)), (64, ((half, min(half + 128, pages)),)), (64, ((120, min(260, pages)),))):
        args = long_waves(tiles, batch, 8, 64, 16, code, dtype, gpu, holes=holes)
        check_long(attend_pages(*args), args)


@pytest.mark.gpu
@pytest.mark.parametrize("code,dtype", [("int8", "bf16"), ("bf16", "bf16")])
@pytest.mark.parametrize("dim,page", [(64, 48), (64, 12), (128, 16), (96, 32), (256, 16)])
def test_long_waves_at_other_pages_and_head_dims(gpu, dim, page, code, dtype):
    for per_head in (False, True):
        args = long_waves(40, 60, 4, dim, page, code, dtype, gpu, per_head=per_head, holes=((30, 90),))
        check_long(attend_pages(*args), args)


@pytest.mark.gpu
@pytest.mark.parametrize("code,dtype", [("int8", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("dim,wide", [(64, 2), (64, WIDE), (80, 2)])
def test_what_the_other_requests_hold_does_not_change_one(gpu, dim, wide, code, dtype):
    """A request's bits depend on the sizes and lengths of its batch, not on what the other requests'
    queries, tables and rows hold (NaN among them).  In a batch of its own it may be cut into other
    parts, so there it agrees with the formula."""
    lengths = [900, 1500, 900, 33]
    query, pool, tables, lengths = case(4, 14, 2, dim, 16, lengths, code, dtype, gpu, wide=wide)
    first = attend_pages(query, pool, tables, lengths)
    assert torch.equal(first, attend_pages(query, pool, tables, lengths))
    alone = [t[1:2].contiguous() for t in (query, tables, lengths)]
    alone = (alone[0], pool, *alone[1:])
    check(attend_pages(*alone), alone)
    check(first[1:2], alone)
    others = [0, 2, 3]
    query, tables = query.clone(), tables.clone()
    query[others] = -3 * query[others]
    tables[0] = tables[2].clone()
    tables[2, 3] = -1
    block = tables[3, 0].item()  # all of the last request's first page
    (pool.scales if code in CODES else pool)[block] = float("nan")
    again = attend_pages(query, pool, tables, lengths)
    assert torch.equal(again[1], first[1])
    assert again[3].isnan().all() and not torch.equal(again[0], first[0])


@pytest.mark.gpu
@pytest.mark.parametrize("code,dtype", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("e4m3", "bf16")])
@pytest.mark.parametrize("dim,wide", [(64, 2), (64, WIDE), (80, 2), (256, 2)])
def test_infinite_scores(gpu, dim, wide, code, dtype):
    """Tokens of score -inf have no weight, as in the formula; a head that has no others gives zeros (the
    formula has no value there); +inf gives NaN.  Other heads and requests are not touched."""
    query, pool, tables, lengths = case(2, 4, 2, dim, 16, [700, 700], code, dtype, gpu, wide=wide)
    plain = not isinstance(pool, QuantizedPool)
    query[:, :, 0] = query[:, :, 0].abs() + 1
    want = attend_pages(query, pool, tables, lengths)
    order = tables.long()[:, :44]

    def with_keys(first, last, value):  # of request 0, KV head 1: pages first .. last
        store = (pool if plain else pool.scales).clone()
        for block in order[0, first:last].tolist():
            if plain:
                store[block, 0, :, 1, 0] = value
            else:
                store[block, 0, :, 1] = value  # a scale: the sign of a score is its code's
        return store if plain else QuantizedPool(pool.codes, store)

    if plain:
        some = attend_pages(query, with_keys(3, 30, -float("inf")), tables, lengths)
        gone = tables[:1, None].repeat(1, 2, 1)
        gone[:, 1, 3:30] = -1  # the same tokens masked
        args = (query[:1], pool, gone, lengths[:1])
        check(some[:1], args)
        assert torch.equal(some[1], want[1])
        none = attend_pages(query, with_keys(0, 44, -float("inf")), tables, lengths)
        assert (none[0, 2:] == 0).all()
        assert torch.equal(none[0, :2], want[0, :2]) and torch.equal(none[1], want[1])
    lost = attend_pages(query, with_keys(5, 6, float("inf")), tables, lengths)
    assert lost[0, 2:].isnan().all()
    assert torch.equal(lost[0, :2], want[0, :2]) and torch.equal(lost[1], want[1])
