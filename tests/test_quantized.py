"""8-bit K/V rows (append_quantized / read_quantized) against their definition in 64 bits,
bit for bit, and the calls they refuse."""

import ctypes

import pytest
import torch

from mini_hisparse_amd import _lib
from mini_hisparse_amd.quantized import QuantizedPool, append_quantized, read_quantized

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
CODES = [torch.int8, torch.float8_e4m3fn]


def grid(code):
    """The code's magnitudes, ascending; the parity of an index is that of its code."""
    if code == torch.int8:
        return torch.arange(128, dtype=torch.float64)
    return torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()


def quantise(x, code):
    """Code values and scales [.., D], [..] in 64 bits: the nearest of the grid, ties to even."""
    x = x.detach().cpu().double()
    magnitudes = grid(code)
    top = float(magnitudes[-1])
    largest = x.abs().amax(-1)
    scales = torch.where(largest.isfinite(), (largest / top).float().double(), float("nan"))
    usable = (scales > 0)[..., None]
    ratio = torch.where(usable, x.abs() / scales[..., None], 0.0).clamp(max=top)
    low = (torch.searchsorted(magnitudes, ratio.contiguous(), right=True) - 1).clamp(0, len(magnitudes) - 2)
    middle = (magnitudes[low] + magnitudes[low + 1]) / 2
    up = (ratio > middle) | ((ratio == middle) & (low % 2 == 1))
    values = torch.where(up, magnitudes[low + 1], magnitudes[low]) * x.sign()
    return torch.where(usable, values, 0.0), scales


def code_values(pool):
    return pool.codes.cpu().float().double()


def filled(blocks, page, kv, dim, code, device, seed=0):
    """A pool whose every byte is set (codes any, scales any): what must stay is seen to stay."""
    gen = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 127, (blocks, 2, page, kv, dim), generator=gen, dtype=torch.uint8)
    return QuantizedPool(codes.view(code).to(device), torch.rand(blocks, 2, page, kv, generator=gen).to(device))


def some_rows(tokens, total, device, seed=0, skipped=0):
    gen = torch.Generator().manual_seed(seed)
    rows = torch.randperm(total, generator=gen)[:tokens]
    if skipped:
        bad = torch.randperm(tokens, generator=gen)[:skipped]
        rows[bad] = torch.tensor([-1, total, total + 5, -(2**40), 2**40])[torch.arange(skipped) % 5]
    return rows.to(device)


def check_append(k, v, rows, pool, before):
    blocks, _, page, kv, dim = pool.codes.shape
    want_codes, want_scales = before.codes.cpu().float().double(), before.scales.cpu().double()
    for plane, x in enumerate((k, v)):
        values, scales = quantise(x, pool.codes.dtype)
        for i, r in enumerate(rows.tolist()):
            if 0 <= r < blocks * page:
                want_codes[r // page, plane, r % page] = values[i]
                want_scales[r // page, plane, r % page] = scales[i]
    assert torch.equal(code_values(pool), want_codes)
    assert torch.equal(pool.scales.cpu().double().nan_to_num(-1), want_scales.nan_to_num(-1))


def copy_of(pool):
    return QuantizedPool(pool.codes.clone(), pool.scales.clone())


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv,dim,page", [(4, 128, 16), (2, 64, 16), (1, 32, 1), (3, 96, 12), (5, 80, 8), (1, 256, 64),
                                         (2, 20, 16), (1, 1, 3), (2, 512, 16), (1, 515 - 4, 2)])
def test_append_and_read_are_the_definition(gpu, code, dtype, kv, dim, page):
    gen = torch.Generator().manual_seed(dim)
    tokens, blocks = 37, -(-50 // page) + 1
    k, v = ((torch.randn(tokens, kv, dim, generator=gen) * torch.rand(tokens, kv, 1, generator=gen) * 9).to(dtype)
            .to(gpu) for _ in range(2))
    pool = filled(blocks, page, kv, dim, code, gpu)
    before = copy_of(pool)
    rows = some_rows(tokens, blocks * page, gpu, skipped=5)
    append_quantized(k, v, rows, pool)
    check_append(k, v, rows, pool, before)
    for out in DTYPES:
        got = read_quantized(pool, rows, out)
        for plane, x in enumerate(got):
            assert x.shape == (tokens, kv, dim) and x.dtype == out
            for i, r in enumerate(rows.tolist()):
                if not 0 <= r < blocks * page:
                    assert (x[i] == 0).all()
                    continue
                want = (pool.codes[r // page, plane, r % page].cpu().float().double()
                        * pool.scales[r // page, plane, r % page].cpu().double()[:, None])
                error = (x[i].cpu().double() - want).abs()
                # the product's rounding to fp32, then to the dtype (float16: half a subnormal step)
                tol = want.abs() * (2.0**-24 + (torch.finfo(out).eps / 2 if out != torch.float32 else 0))
                assert (error <= tol + (2.0**-25 if out == torch.float16 else 0)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_on_and_next_to_the_borders(gpu, code, dtype):
    """Head vectors whose elements are the borders between two codes, and their neighbours in
    the dtype, for many scales: each code is the exact quotient's."""
    magnitudes = grid(code)
    gen = torch.Generator().manual_seed(5)
    middles = (magnitudes[1:] + magnitudes[:-1]) / 2
    tops = torch.cat((torch.tensor([1.0, 2.0, 7.0, 448.0, 127.0, 0.4375]), torch.rand(58, generator=gen) * 20 + 0.01))
    vectors = []
    for top in tops.to(dtype).double():
        scale = (top / magnitudes[-1]).float().double()
        x = (middles * scale).to(dtype)
        near = torch.cat((x, torch.nextafter(x.float(), torch.tensor(9e9)).to(dtype),
                          torch.nextafter(x.float(), torch.tensor(-9e9)).to(dtype)))
        pick = torch.randperm(len(near), generator=gen)[:127]
        signs = torch.randint(0, 2, (127,), generator=gen) * 2 - 1
        vectors.append(torch.cat((near[pick].clamp(max=float(top)) * signs, top.to(dtype)[None])))
    k = torch.stack(vectors).reshape(16, 4, 128).to(gpu)
    pool = filled(2, 16, 4, 128, code, gpu)
    before = copy_of(pool)
    rows = some_rows(16, 32, gpu)
    append_quantized(k, -k, rows, pool)
    check_append(k, -k, rows, pool, before)


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 50])
def test_zeros_nan_infinity_and_the_smallest_and_largest_values(gpu, code, dtype, dim):
    gen = torch.Generator().manual_seed(3)
    k = torch.randn(10, 2, dim, generator=gen)
    k[0] = 0
    k[1, 0, 3] = float("nan")
    k[2, 1, 0] = float("inf")
    k[3, 0, dim - 1] = -float("inf")
    k = k.to(dtype)
    info = torch.finfo(dtype)
    k[4] = info.max
    k[5] = -info.max
    k[6] = k[6] * info.smallest_normal  # subnormal and smallest normal values
    k[7, 0] = 0
    k[7, 0, 1] = info.smallest_normal
    if dtype != torch.float16:  # scales that are subnormal in float32, or round to nothing
        ulps = torch.arange(2 * dim).reshape(2, dim) % 200
        k[8] = (ulps.double() * 2.0 ** (-149 if dtype == torch.float32 else -133)).to(dtype)
        k[9] = (torch.full((2, dim), 1.0).double() * 2.0 ** (-149 if dtype == torch.float32 else -133)).to(dtype)
    k = k.to(gpu)
    v = k.flip(0).contiguous()
    pool = filled(1, 16, 2, dim, code, gpu)
    before = copy_of(pool)
    rows = some_rows(10, 16, gpu)
    append_quantized(k, v, rows, pool)
    check_append(k, v, rows, pool, before)
    back = read_quantized(pool, rows, torch.float32)[0]
    assert back[1, 0].isnan().all() and back[1, 1].isfinite().all() and (back[0] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
def test_strided_and_misaligned_inputs(gpu, code):
    tokens, kv, dim = 7, 2, 64
    for offset, pad in ((0, 16), (1, 3), (8, 8), (4, 4)):
        buffer = torch.randn(tokens * (3 * kv * dim + pad) + 16, device=gpu).to(torch.bfloat16)
        packed = buffer[offset : offset + tokens * (3 * kv * dim + pad)].view(tokens, -1)
        k = packed[:, : kv * dim].view(tokens, kv, dim)  # slices of a packed projection
        v = packed[:, kv * dim : 2 * kv * dim].view(tokens, kv, dim).flip(1).transpose(0, 1).contiguous().transpose(0, 1)
        pool = filled(1, 16, kv, dim, code, gpu)
        before = copy_of(pool)
        rows = some_rows(tokens, 16, gpu)
        append_quantized(k, v, rows, pool)
        check_append(k, v, rows, pool, before)


@pytest.mark.gpu
def test_no_rows_and_given_outputs(gpu):
    pool = filled(2, 16, 2, 64, torch.int8, gpu)
    before = copy_of(pool)
    none = torch.empty(0, dtype=torch.int64, device=gpu)
    append_quantized(torch.empty(0, 2, 64, device=gpu), torch.empty(0, 2, 64, device=gpu), none, pool)
    assert torch.equal(pool.codes, before.codes) and torch.equal(pool.scales, before.scales)
    k, v = read_quantized(pool, none, torch.float16)
    assert k.shape == v.shape == (0, 2, 64)
    rows = torch.arange(32, device=gpu)
    guarded = torch.full((34, 2, 64), 7.0, dtype=torch.bfloat16, device=gpu)
    out = (guarded[1:33], torch.empty(32, 2, 64, dtype=torch.bfloat16, device=gpu))
    got = read_quantized(pool, rows, torch.bfloat16, out=out)
    assert got[0].data_ptr() == out[0].data_ptr() and (guarded[0] == 7).all() and (guarded[33] == 7).all()
    assert torch.equal(got[0], read_quantized(pool, rows, torch.bfloat16)[0])


@pytest.mark.gpu
def test_long_prompt(gpu):
    """More head vectors than one round of workgroups; compared on the GPU in 64 bits."""
    tokens, kv, dim, page = 20_011, 4, 128, 16
    blocks = -(-tokens // page) + 1
    k, v = (torch.randn(tokens, kv, dim, device=gpu).to(torch.bfloat16) for _ in range(2))
    for code, top in ((torch.int8, 127.0), (torch.float8_e4m3fn, 448.0)):
        pool = QuantizedPool.empty(blocks, page, kv, dim, code, gpu)
        rows = torch.randperm(blocks * page, device=gpu)[:tokens]
        append_quantized(k, v, rows, pool)
        got = read_quantized(pool, rows, torch.float32)
        for x, y in zip((k, v), got):
            scale = (x.double().abs().amax(-1, keepdim=True) / top).float().double()
            q = x.double() / scale
            if code == torch.int8:
                want = q.round() * scale
            else:
                step = torch.exp2((torch.frexp(q)[1] - 4).clamp(min=-9).double())
                want = (q / step).round() * step * scale
            # the read's one product
            assert ((y.double() - want).abs() <= 2.0**-24 * want.abs()).all()
        assert pool.scales.view(-1).count_nonzero().item() == tokens * 2 * kv  # every other row as it was


@pytest.mark.gpu
def test_rows_past_32_bit_offsets(gpu):
    blocks, page, kv, dim = 140_000, 16, 8, 128  # 4.6e9 codes
    pool = QuantizedPool.empty(blocks, page, kv, dim, torch.int8, gpu)
    rows = torch.tensor([blocks * page - 1, 2**31 // (kv * dim) // 2 + 3, 2**32 // (2 * kv * dim) + 1, 0], device=gpu)
    k, v = (torch.randn(4, kv, dim, device=gpu).to(torch.bfloat16) for _ in range(2))
    append_quantized(k, v, rows, pool)
    for plane, (x, y) in enumerate(zip((k, v), read_quantized(pool, rows, torch.float32))):
        values, scales = quantise(x, torch.int8)
        want = values * scales[..., None]
        assert ((y.cpu().double() - want).abs() <= 2.0**-24 * want.abs()).all()
        for i, r in enumerate(rows.tolist()):
            assert torch.equal(pool.codes[r // page, plane, r % page].cpu().double(), values[i])
    assert pool.scales.view(-1).count_nonzero().item() == 4 * 2 * kv


@pytest.mark.gpu
def test_other_stream_and_captured_replays(gpu):
    kv, dim = 2, 64
    pool = QuantizedPool.empty(2, 16, kv, dim, torch.int8, gpu)
    rows = torch.tensor([3, 17], device=gpu)
    k, v = (torch.randn(2, kv, dim, device=gpu) for _ in range(2))
    side = torch.cuda.Stream(torch.device(gpu))
    side.wait_stream(torch.cuda.current_stream(torch.device(gpu)))
    with torch.cuda.stream(side):
        append_quantized(k, v, rows, pool)
        got = read_quantized(pool, rows, torch.float32)
    torch.cuda.current_stream(torch.device(gpu)).wait_stream(side)
    values, scales = quantise(k, torch.int8)
    assert torch.equal(code_values(pool)[[0, 1], 0, [3, 1]], values)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        append_quantized(k, v, rows, pool)
        got = read_quantized(pool, rows, torch.float32)
    for step in range(3):
        rows += 1
        k.normal_()
        graph.replay()
        eager = read_quantized(pool, rows, torch.float32)
        values, scales = quantise(k, torch.int8)
        want = values * scales[..., None]
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])
        assert ((got[0].cpu().double() - want).abs() <= 2.0**-24 * want.abs()).all()


def test_pool_and_call_refusals_without_a_gpu():
    codes, scales = torch.zeros(2, 2, 4, 3, 8, dtype=torch.int8), torch.zeros(2, 2, 4, 3)
    pool = QuantizedPool(codes, scales)
    assert (pool.page_size, pool.kv_heads, pool.head_dim, pool.rows, pool.row_bytes) == (4, 3, 8, 8, 72)
    assert QuantizedPool.empty(1, 2, 3, 4, torch.float8_e4m3fn, "cpu").codes.float().abs().sum() == 0
    for bad in ((codes.float(), scales), (codes.to(torch.uint8), scales), (codes[0], scales), (codes, scales.double()),
                (codes, scales[..., :2]), (codes[:, :1], scales[:, :1]), (codes[..., ::2], scales),
                (codes[:0], scales[:0]), (codes.transpose(2, 3), scales.transpose(2, 3))):
        with pytest.raises(ValueError):
            QuantizedPool(*bad)
    k, rows = torch.zeros(5, 3, 8), torch.arange(5)
    with pytest.raises(ValueError, match="K and V"):
        append_quantized(k[:4], k, rows, pool)
    with pytest.raises(ValueError, match="K and V"):
        append_quantized(k, k.half(), rows, pool)
    with pytest.raises(ValueError, match="K and V"):
        append_quantized(k.transpose(1, 2).contiguous().transpose(1, 2), k, rows, pool)
    with pytest.raises(ValueError, match="dtype"):
        append_quantized(k.double(), k.double(), rows, pool)
    with pytest.raises(ValueError, match="rows"):
        append_quantized(k, k, rows.int(), pool)
    with pytest.raises(ValueError, match="rows"):
        append_quantized(k, k, rows.repeat(2)[::2], pool)
    with pytest.raises(ValueError, match="K and V"):
        append_quantized(k, k, torch.tensor(3), pool)
    with pytest.raises(ValueError, match="ROCm"):
        append_quantized(k, k, rows, pool)
    with pytest.raises(ValueError, match="dtype"):
        read_quantized(pool, rows, torch.float64)
    with pytest.raises(ValueError, match="rows"):
        read_quantized(pool, rows[None])
    with pytest.raises(ValueError, match="out"):
        read_quantized(pool, rows, torch.float32, out=(k, k[:4]))
    with pytest.raises(ValueError, match="ROCm"):
        read_quantized(pool, rows)
    wide = QuantizedPool(torch.zeros(1, 2, 1, 1, 513, dtype=torch.int8), torch.zeros(1, 2, 1, 1))
    with pytest.raises(ValueError, match="512"):
        read_quantized(wide, rows)


def test_entry_point_refusals_without_a_gpu():
    lib = _lib.load()
    buffer = ctypes.create_string_buffer(256)
    at = ctypes.addressof(buffer)
    at += -at % 16

    def append(k=at, rows=at, tokens=1, codes=at, scales=at, code=3, pool_rows=4, page=4, kv=1, dim=8, dtype=0,
               stride=8):
        return lib.hs_append_quantized(k, stride, stride, at, stride, stride, dtype, rows, tokens, codes, scales, code,
                                       pool_rows, page, kv, dim, None)

    def read(k=at, rows=at, n=1, codes=at, scales=at, code=3, pool_rows=4, page=4, kv=1, dim=8, dtype=0):
        return lib.hs_read_quantized(codes, scales, code, pool_rows, page, kv, dim, rows, n, k, at, dtype, None)

    shared = (dict(codes=None), dict(scales=None), dict(code=2), dict(code=5), dict(pool_rows=0), dict(page=0),
              dict(kv=0), dict(dim=0), dict(dim=513), dict(dtype=3), dict(k=None), dict(rows=None), dict(scales=at + 2))
    for bad in (*shared, dict(tokens=-1), dict(tokens=2**40), dict(stride=-8)):
        assert append(**bad) == -1, bad
    for bad in (*shared, dict(n=-1), dict(n=2**40)):
        assert read(**bad) == -1, bad
    assert append(tokens=0, k=None, rows=None) == 0 and read(n=0, k=None, rows=None) == 0  # nothing to do


def test_pools_that_are_no_whole_pages_are_refused_without_a_gpu():
    """A page longer than the pool (2^32 rows would be 0 in 32 bits) and a last page that the pool ends in."""
    lib = _lib.load()
    buffer = ctypes.create_string_buffer(256)
    at = ctypes.addressof(buffer)
    at += -at % 16
    for pool_rows, page in ((4, 8), (4, 2**32), (2**31, 2**32), (4, 2**62), (7, 4), (2**33 + 1, 2**32)):
        assert lib.hs_append_quantized(at, 8, 8, at, 8, 8, 0, at, 1, at, at, 3, pool_rows, page, 1, 8, None) == -1
        assert b"whole pages" in lib.hs_last_error()
        assert lib.hs_read_quantized(at, at, 3, pool_rows, page, 1, 8, at, 1, at, at, 0, None) == -1
        assert b"whole pages" in lib.hs_last_error()
