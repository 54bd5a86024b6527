"""4-bit K/V rows against their definition in 64 bits, bit for bit, and attention over them."""

import ctypes

import pytest
import torch

from mini_hisparse_amd import _lib
from mini_hisparse_amd.quantized import QuantizedPool, append_quantized, read_quantized
from mini_hisparse_amd.row_kernels import attend_pages

from page_cases import FP4, FP4_VALUES, case, check, pack_fp4, quantise_fp4, store_of, widen_fp4

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
E8M0 = torch.float8_e8m0fnu


def filled(blocks, page, kv, dim, device, seed=0):
    """A pool whose every byte is set: what must stay is seen to stay."""
    gen = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (blocks, 2, page, kv, dim // 2), generator=gen, dtype=torch.uint8)
    scales = torch.randint(0, 256, (blocks, 2, page, kv, dim // 32), generator=gen, dtype=torch.uint8)
    return QuantizedPool(codes.to(device).view(FP4), scales.to(device).view(E8M0))


def bytes_of(pool):
    return pool.codes.view(torch.uint8).cpu().clone(), pool.scales.view(torch.uint8).cpu().clone()


def some_rows(tokens, total, device, seed=0, skipped=0):
    gen = torch.Generator().manual_seed(seed)
    rows = torch.randperm(total, generator=gen)[:tokens]
    if skipped:
        bad = torch.randperm(tokens, generator=gen)[:skipped]
        rows[bad] = torch.tensor([-1, total, total + 5, -(2**40), 2**40])[torch.arange(skipped) % 5]
    return rows.to(device)


def check_append(k, v, rows, pool, before):
    blocks, _, page, _, _ = pool.codes.shape
    codes, scales = before
    for plane, x in enumerate((k, v)):
        c, s = quantise_fp4(x)
        c = pack_fp4(c)
        for i, r in enumerate(rows.tolist()):
            if 0 <= r < blocks * page:
                codes[r // page, plane, r % page], scales[r // page, plane, r % page] = c[i], s[i]
    got = bytes_of(pool)
    assert torch.equal(got[1], scales)
    assert torch.equal(got[0], codes)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv,dim,page", [(4, 128, 16), (2, 64, 16), (1, 32, 1), (3, 96, 12), (5, 160, 8), (1, 256, 64),
                                         (2, 512, 16), (1, 480, 3)])
def test_append_and_read_are_the_definition(gpu, dtype, kv, dim, page):
    gen = torch.Generator().manual_seed(dim)
    tokens, blocks = 37, -(-50 // page) + 1
    k, v = ((torch.randn(tokens, kv, dim, generator=gen) * torch.rand(tokens, kv, 1, generator=gen) * 9).to(dtype)
            .to(gpu) for _ in range(2))
    pool = filled(blocks, page, kv, dim, gpu)
    before = bytes_of(pool)
    rows = some_rows(tokens, blocks * page, gpu, skipped=5)
    append_quantized(k, v, rows, pool)
    check_append(k, v, rows, pool, before)
    store = store_of(pool)
    for out in DTYPES:
        for plane, x in enumerate(read_quantized(pool, rows, out)):
            assert x.shape == (tokens, kv, dim) and x.dtype == out
            for i, r in enumerate(rows.tolist()):
                want = store[r // page, plane, r % page] if 0 <= r < blocks * page else torch.zeros(kv, dim)
                assert torch.equal(x[i].cpu(), want.to(out))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_border_power_and_code(gpu, dtype):
    """Borders between two codes and their neighbours, largest magnitudes on both sides of a power's
    border, for every power of two that the dtype can hold; and every code under every scale byte."""
    gen = torch.Generator().manual_seed(5)
    middles = torch.cat(((FP4_VALUES[1:] + FP4_VALUES[:-1]) / 2, FP4_VALUES, torch.tensor([6.5, 6.99])))
    info = torch.finfo(dtype)
    low, high = (-150, 125) if dtype != torch.float16 else (-24, 13)
    vectors = []
    for power in range(low, high + 1):
        for top in (7.0, 7.0 * (1 + 2 * info.eps), 3.5, 3.5 * (1 + 2 * info.eps), 6.0):
            x = middles.float().to(dtype)
            near = torch.cat((x, (x.double() * (1 + info.eps)).to(dtype), (x.double() * (1 - info.eps)).to(dtype)))
            pick = near[torch.randperm(len(near), generator=gen)[:31]].double().clamp(max=top)
            signs = torch.randint(0, 2, (31,), generator=gen) * 2 - 1
            vectors.append((torch.cat((pick * signs, torch.tensor([top]))) * 2.0**power).to(dtype))
    while len(vectors) % 4:
        vectors.append(torch.zeros(32, dtype=dtype))
    k = torch.stack(vectors).reshape(-1, 1, 128).to(gpu)
    pool = filled(len(k), 1, 1, 128, gpu)
    before = bytes_of(pool)
    rows = some_rows(len(k), len(k), gpu)
    append_quantized(k, -k, rows, pool)
    check_append(k, -k, rows, pool, before)

    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1).view(256, 16, 16)  # 32 codes a scale
    scales = torch.arange(256, dtype=torch.uint8)[:, None].expand(-1, 16).contiguous()
    pool = QuantizedPool(torch.stack((codes, codes), 1).view(256, 2, 1, 1, 256).to(gpu).view(FP4),
                         torch.stack((scales, scales), 1).view(256, 2, 1, 1, 16).to(gpu).view(E8M0))
    for x in read_quantized(pool, torch.arange(256, device=gpu), dtype):
        want = widen_fp4(codes.reshape(256, 256), scales).to(dtype)
        assert torch.equal(x[:, 0].cpu().nan_to_num(-1.0), want.nan_to_num(-1.0))
        assert torch.equal(x[:, 0].cpu().isnan(), want.isnan())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_zeros_nan_infinity_and_the_smallest_and_largest_values(gpu, dtype):
    gen = torch.Generator().manual_seed(3)
    k = torch.randn(8, 2, 96, generator=gen)
    k[0] = 0
    k[0, 0, 40] = -0.0
    k[1, 0, 3] = float("nan")
    k[2, 1, 32] = float("inf")
    k[3, 0, 95] = -float("inf")
    k = k.to(dtype)
    info = torch.finfo(dtype)
    k[4], k[5] = info.max, -info.max
    k[6] = k[6] * info.smallest_normal
    k[7, 0] = 0
    k[7, 0, 1] = info.smallest_normal * info.eps
    k = k.to(gpu)
    v = k.flip(0).contiguous()
    pool = filled(1, 16, 2, 96, gpu)
    before = bytes_of(pool)
    rows = some_rows(8, 16, gpu)
    append_quantized(k, v, rows, pool)
    check_append(k, v, rows, pool, before)
    back = read_quantized(pool, rows, torch.float32)[0]
    assert back[1, 0, :32].isnan().all() and back[1, 0, 32:].isfinite().all() and back[1, 1].isfinite().all()
    assert back[2, 1, 32:64].isnan().all() and back[2, 1, :32].isfinite().all() and (back[0] == 0).all()


@pytest.mark.gpu
def test_strided_and_misaligned_inputs_and_pools(gpu):
    tokens, kv, dim = 7, 2, 64
    for offset, pad, at in ((0, 16, 0), (1, 3, 0), (8, 8, 1), (4, 4, 2), (0, 0, 4)):
        buffer = torch.randn(tokens * (3 * kv * dim + pad) + 16, device=gpu).to(torch.bfloat16)
        packed = buffer[offset : offset + tokens * (3 * kv * dim + pad)].view(tokens, -1)
        k = packed[:, : kv * dim].view(tokens, kv, dim)  # slices of a packed projection
        v = packed[:, kv * dim : 2 * kv * dim].view(tokens, kv, dim).flip(1).transpose(0, 1).contiguous().transpose(0, 1)
        codes, scales = bytes_of(filled(1, 16, kv, dim, "cpu"))
        parts = []
        for x in (codes, scales):
            room = torch.empty(x.numel() + at, dtype=torch.uint8, device=gpu)
            parts.append(room[at:].view(x.shape))
            parts[-1].copy_(x)
        pool = QuantizedPool(parts[0].view(FP4), parts[1].view(E8M0))
        rows = some_rows(tokens, 16, gpu)
        append_quantized(k, v, rows, pool)
        check_append(k, v, rows, pool, (codes, scales))
        for dtype in DTYPES:
            room = torch.full((tokens * kv * dim + 1,), 7.0, dtype=dtype, device=gpu)
            out = (room[1:].view(tokens, kv, dim), torch.empty(tokens, kv, dim, dtype=dtype, device=gpu))
            read_quantized(pool, rows, dtype, out=out)
            want = store_of(pool)
            for plane, x in enumerate(out):
                assert torch.equal(x.cpu(), want[0, plane, rows.cpu()].to(dtype))
            assert room[0] == 7


@pytest.mark.gpu
def test_no_rows_long_prompts_and_rows_past_32_bit_offsets(gpu):
    pool = filled(2, 16, 2, 64, gpu)
    before = bytes_of(pool)
    none = torch.empty(0, dtype=torch.int64, device=gpu)
    append_quantized(torch.empty(0, 2, 64, device=gpu), torch.empty(0, 2, 64, device=gpu), none, pool)
    assert all(torch.equal(x, y) for x, y in zip(bytes_of(pool), before))
    assert read_quantized(pool, none, torch.float16)[0].shape == (0, 2, 64)

    blocks, page, kv, dim = 140_000, 16, 8, 128  # 4.6e9 values
    pool = QuantizedPool.empty(blocks, page, kv, dim, FP4, gpu)
    tokens = 20_011
    rows = torch.randperm(blocks * page, device=gpu)[:tokens]
    rows[:5] = torch.tensor([blocks * page - 1, 2**31 // (kv * dim) // 2 + 3, 2**32 // (kv * dim) + 1, 0,
                             2**32 // (kv * dim) // 2 + 1], device=gpu)  # the third is past the pool
    rows[5:] = torch.where((rows[5:, None] == rows[:5]).any(1), -1, rows[5:])
    k, v = (torch.randn(tokens, kv, dim, device=gpu).to(torch.bfloat16) for _ in range(2))
    append_quantized(k, v, rows, pool)
    kept = (rows >= 0) & (rows < blocks * page)
    for plane, (x, y) in enumerate(zip((k, v), read_quantized(pool, rows, torch.float32))):
        codes, scales = quantise_fp4(x)
        want = widen_fp4(pack_fp4(codes), scales)
        assert torch.equal(y.cpu().double()[kept.cpu()], want[kept.cpu()])
    assert pool.scales.view(torch.uint8).count_nonzero().item() == int(kept.sum()) * 2 * kv * dim // 32


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [2, 20_000])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv,dim", [(28, 4, 128), (14, 2, 64), (4, 2, 32), (8, 8, 128), (20, 1, 64), (36, 1, 128),
                                          (12, 3, 96), (3, 1, 256), (5, 5, 160), (2, 2, 512), (22, 11, 64), (2, 1, 480)])
def test_attention_matches_the_formula(gpu, heads, kv, dim, dtype, wide):
    for page in (16, 3, 48):
        args = case(3, heads, kv, dim, page, [333, 1, 97], "fp4", dtype, gpu, wide=wide)
        check(attend_pages(*args), args)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 256])
def test_attention_lengths_absent_pages_and_tables_per_head(gpu, dim):
    for wide in (2, 20_000):
        for lengths in ([0], [1], [31, 32, 33], [63, 64, 65, 0, 127, 128, 129], [511, 512, 513], [4000, 3, 0]):
            args = case(len(lengths), 8, 2, dim, 16, lengths, "fp4", "bf16", gpu, wide=wide)
            check(attend_pages(*args), args)
        for page in (16, 5):
            for per_head in (False, True):
                for absent in (0.4, 1.0):
                    args = case(3, 14, 2, dim, page, [700, 33, 16], "fp4", "bf16", gpu, absent=absent,
                                per_head=per_head, wide=wide)
                    check(attend_pages(*args), args)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 256])
def test_a_nan_group_reaches_its_heads_alone(gpu, dim):
    """A scale of NaN in a key takes all of its heads' outputs, in a value the 32 of its group."""
    for plane in (0, 1):
        for group in range(dim // 32):
            query, pool, tables, lengths = case(2, 4, 2, dim, 16, [40, 40], "fp4", "bf16", gpu)
            block = tables[0, 1].item()
            pool.scales.view(torch.uint8)[block, plane, 3, 1, group] = 255  # of request 0, KV head 1
            got = attend_pages(query, pool, tables, lengths)
            bad = got[0, 2:].isnan()
            assert got[0, :2].isfinite().all() and got[1].isfinite().all()
            if plane == 0:
                assert bad.all()
            else:
                want = torch.zeros(dim, dtype=torch.bool)
                want[32 * group : 32 * group + 32] = True
                assert torch.equal(bad.cpu(), want.expand(2, -1))


@pytest.mark.gpu
def test_small_and_large_values(gpu):
    """Values of any power of two that bfloat16 outputs can hold, one key that leads by far, codes of
    the smallest scales (zeros of a fresh pool among them)."""
    for power in (-100, -20, 0, 20, 100):
        for dim in (128, 160):
            query, pool, tables, lengths = args = case(2, 8, 2, dim, 16, [300, 1], "fp4", "bf16", gpu)
            scales = pool.scales.view(torch.uint8)
            part = scales[:, 1].int()
            scales[:, 1] = torch.where(part < 255, part + power, part).to(torch.uint8)
            check(attend_pages(*args), args)
    pool = QuantizedPool.empty(20, 16, 2, 128, FP4, gpu)
    query = torch.randn(1, 4, 128, device=gpu).to(torch.float16)
    tables = torch.arange(20, dtype=torch.int32, device=gpu)[None]
    lengths = torch.tensor([300], dtype=torch.int32, device=gpu)
    assert (attend_pages(query, pool, tables, lengths) == 0).all()


@pytest.mark.gpu
def test_other_streams_and_captured_replays(gpu):
    """Rows written and attended on another stream, and in a graph replayed with other rows and lengths."""
    kv, dim, page = 2, 64, 16
    pool = QuantizedPool.empty(40, page, kv, dim, FP4, gpu)
    tables = torch.randperm(40, device=gpu).to(torch.int32)[None]
    lengths = torch.tensor([0], dtype=torch.int32, device=gpu)
    query = torch.randn(1, 14, dim, device=gpu).to(torch.bfloat16)
    k, v = (torch.randn(1, kv, dim, device=gpu).to(torch.bfloat16) for _ in range(2))

    def step():
        at = lengths.long()
        append_quantized(k, v, tables[0].long()[at // page] * page + at % page, pool)
        lengths.add_(1)
        return attend_pages(query, pool, tables, lengths)

    side = torch.cuda.Stream(torch.device(gpu))
    side.wait_stream(torch.cuda.current_stream(torch.device(gpu)))
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream(torch.device(gpu)).wait_stream(side)
    check(got, (query, pool, tables, lengths))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(20):
        k.normal_()
        v.normal_()
        graph.replay()
        assert torch.equal(out, attend_pages(query, pool, tables, lengths))
        check(out, (query, pool, tables, lengths))
    assert lengths.item() == 21


def test_refusals_without_a_gpu():
    codes = torch.zeros(2, 2, 4, 3, 32, dtype=torch.uint8)
    scales = torch.zeros(2, 2, 4, 3, 2, dtype=torch.uint8)
    pool = QuantizedPool(codes.view(FP4), scales.view(E8M0))
    assert (pool.page_size, pool.kv_heads, pool.head_dim, pool.rows, pool.row_bytes) == (4, 3, 64, 8, 2 * 3 * 34)
    assert QuantizedPool.empty(1, 2, 3, 96, FP4, "cpu").head_dim == 96
    for bad in ((codes, scales.view(E8M0)), (codes.view(FP4), scales), (codes.view(FP4), scales.view(E8M0)[..., :1]),
                (codes.view(FP4), torch.zeros(2, 2, 4, 3)), (codes.view(FP4)[..., :8], scales.view(E8M0)[..., :1]),
                (codes.view(FP4), scales.view(E8M0)[:1]), (codes[:0].view(FP4), scales[:0].view(E8M0)),
                (codes.transpose(2, 3).view(FP4), scales.view(E8M0))):
        with pytest.raises(ValueError):
            QuantizedPool(*bad)
    with pytest.raises(ValueError, match="multiple of 32"):
        QuantizedPool.empty(1, 2, 3, 80, FP4, "cpu")
    k, rows = torch.zeros(5, 3, 64), torch.arange(5)
    with pytest.raises(ValueError, match="K and V"):
        append_quantized(k[..., :32], k[..., :32], rows, pool)
    with pytest.raises(ValueError, match="ROCm"):
        append_quantized(k, k, rows, pool)
    with pytest.raises(ValueError, match="out"):
        read_quantized(pool, rows, torch.float32, out=(k, k[:4]))
    with pytest.raises(ValueError, match="ROCm"):
        read_quantized(pool, rows)
    with pytest.raises(ValueError, match="head_dim"):
        attend_pages(torch.zeros(1, 6, 32), pool, torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


def test_entry_point_refusals_without_a_gpu():
    lib = _lib.load()
    buffer = ctypes.create_string_buffer(256)
    at = ctypes.addressof(buffer)
    at += -at % 16
    for dim in (8, 48, 544):
        assert lib.hs_append_quantized(at, dim, dim, at, dim, dim, 0, at, 1, at, at, 6, 4, 4, 1, dim, None) == -1
        assert lib.hs_read_quantized(at, at, 6, 4, 4, 1, dim, at, 1, at, at, 0, None) == -1
    for pool_rows, page in ((4, 8), (7, 4), (0, 1)):
        assert lib.hs_append_quantized(at, 32, 32, at, 32, 32, 0, at, 1, at, at, 6, pool_rows, page, 1, 32, None) == -1
    assert lib.hs_append_quantized(at, 32, 32, at, 32, 32, 0, at, 1, at, None, 6, 4, 4, 1, 32, None) == -1
    assert lib.hs_append_quantized(None, 32, 32, None, 32, 32, 0, None, 0, at, at, 6, 4, 4, 1, 32, None) == 0
