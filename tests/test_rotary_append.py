"""Normed rotary embedding with K and V written to a pool on the way (norm_rotary_append): q and K
against the formula in 64 bits, V and unturned K bit for bit, and the calls it refuses."""

import ctypes

import pytest
import torch

from mini_hisparse_amd import _lib
from mini_hisparse_amd.dense import norm_rotary_append, prepare_norm_rotary_append
from mini_hisparse_amd.quantized import QuantizedPool

from page_cases import FP4, FP4_VALUES, pack_fp4, quantise_fp4, widen_fp4
from test_norm_rotary import check, formula, inputs
from test_quantized import grid, quantise

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
CODES = [None, torch.int8, torch.float8_e4m3fn, FP4]  # None: a plain pool of the projection's dtype
SHAPES = [(28, 4, 128), (14, 2, 64), (4, 2, 32), (3, 1, 256), (12, 3, 96), (5, 5, 80), (2, 1, 6), (1, 1, 2), (2, 2, 512),
          (3, 1, 100), (2, 2, 160), (1, 3, 480)]


def filled(blocks, page, kv, dim, code, dtype, device):
    """A pool whose every byte is set."""
    gen = torch.Generator().manual_seed(dim)
    if code is None:
        return torch.randn(blocks, 2, page, kv, dim, generator=gen).to(dtype).to(device)
    if code == FP4:
        codes = torch.randint(0, 256, (blocks, 2, page, kv, dim // 2), generator=gen, dtype=torch.uint8)
        scales = torch.randint(0, 255, (blocks, 2, page, kv, dim // 32), generator=gen, dtype=torch.uint8)
        return QuantizedPool(codes.to(device).view(FP4), scales.to(device).view(torch.float8_e8m0fnu))
    codes = torch.randint(0, 127, (blocks, 2, page, kv, dim), generator=gen, dtype=torch.uint8)
    return QuantizedPool(codes.view(code).to(device), torch.rand(blocks, 2, page, kv, generator=gen).to(device))


def planes(pool):
    """(codes as bytes or plain values, scales) [2, rows, Hkv, ..] on the CPU."""
    flat = lambda x: x.cpu().movedim(1, 0).flatten(1, 2).clone()  # noqa: E731
    if not isinstance(pool, QuantizedPool):
        return flat(pool), None
    scales = pool.scales.view(torch.uint8) if pool.codes.dtype == FP4 else pool.scales
    return flat(pool.codes.view(torch.uint8)), flat(scales)


def some_rows(tokens, total, device, skipped=0):
    gen = torch.Generator().manual_seed(tokens)
    rows = torch.randperm(total, generator=gen)[:tokens]
    if skipped:
        bad = torch.randperm(tokens, generator=gen)[:skipped]
        rows[bad] = torch.tensor([-1, total, total + 5, -(2**40), 2**40])[torch.arange(skipped) % 5]
    return rows.to(device)


def stored_exactly(x, code, dtype):
    """What a pool holds for head vectors that reach it exactly: (bytes or values, scales)."""
    if code is None:
        return x.to(dtype), None
    if code == FP4:
        codes, scales = quantise_fp4(x)
        return pack_fp4(codes), scales
    values, scales = quantise(x, code)
    return values.float().to(code).view(torch.uint8), scales.float()


def alike(code, got, want):
    """The same codes: of two zeros either sign."""
    if code == torch.float8_e4m3fn:
        return torch.equal(got.view(code).float(), want.view(code).float())
    return torch.equal(got, want)


def nearest(ratio, magnitudes):
    """The nearest of the grid, ties to the even code."""
    size = ratio.abs().clamp(max=float(magnitudes[-1]))
    low = (torch.searchsorted(magnitudes, size.contiguous(), right=True) - 1).clamp(0, len(magnitudes) - 2)
    middle = (magnitudes[low] + magnitudes[low + 1]) / 2
    up = (size > middle) | ((size == middle) & (low % 2 == 1))
    return torch.where(up, magnitudes[low + 1], magnitudes[low]) * ratio.sign()


def check_keys(got, scales, want, size, code, dtype):
    """Keys as stored, of fp32 values within 64 half steps of 2^-24 of the two terms (d) of the
    formula's: plain ones as q is checked; a scale is that of a largest magnitude within d; a
    code lies between those of the values d below and above, rounding being monotone."""
    if code is None:
        return check(got, want, size, dtype)
    d = 64 * 2.0**-24 * size
    if code == FP4:
        top, slack = (x.unflatten(-1, (-1, 32)).amax(-1) for x in (want.abs(), d))
        power = scales.double() - 127
        assert (7 * torch.exp2(power) >= top - slack).all()
        assert ((7 * torch.exp2(power - 1) < top + slack) | (power == -126)).all()
        values, scale = widen_fp4(got, torch.full_like(scales, 127)), torch.exp2(power).repeat_interleave(32, -1)
        magnitudes = FP4_VALUES
    else:
        magnitudes = grid(code)
        top, slack = want.abs().amax(-1), d.amax(-1)
        limit = float(magnitudes[-1])
        assert ((scales.double() - top / limit).abs() <= (slack + 2.0**-23 * top) / limit).all()
        values, scale = got.view(code).float().double(), scales.double()[..., None].expand(want.shape)
    low, high = nearest((want - d) / scale, magnitudes), nearest((want + d) / scale, magnitudes)
    assert ((low <= values) & (values <= high)).all()


def run_and_check(rows, heads, kv, dim, code, dtype, device, page=16, norm=True, skipped=0, qkv=None, theta=1e6,
                  positions=None):
    base, wq, wk, at = inputs(rows, heads, kv, dim, dtype, device)
    qkv = base if qkv is None else qkv
    positions = at if positions is None else positions
    wq, wk = (wq, wk) if norm else (None, None)
    blocks = -(-rows // page) + 2
    pool = filled(blocks, page, kv, dim, code, dtype, device)
    stored, scales = planes(pool)
    to = some_rows(rows, blocks * page, device, skipped)
    q = norm_rotary_append(qkv, wq, wk, 1e-6, positions, to, pool, heads, theta)
    ones = torch.ones(dim)
    if norm:
        (want_q, want_k), (size_q, size_k), want_v = formula(qkv, wq, wk, 1e-6, positions, heads, kv, dim, theta)
    else:
        (want_q, want_k), (size_q, size_k), want_v = plain_formula(qkv, positions, heads, kv, dim, theta)
    check(q, want_q, size_q, dtype)
    got, got_scales = planes(pool)
    kept = ((to >= 0) & (to < blocks * page)).cpu()
    there = to.cpu()[kept]
    check_keys(got[0, there], None if scales is None else got_scales[0, there], want_k[kept], size_k[kept], code, dtype)
    values, value_scales = stored_exactly(want_v, code, dtype)
    stored[1, there], stored[0, there] = values[kept], got[0, there]
    assert alike(code, got, stored)  # V bit for bit, and every other row as it was
    if scales is not None:
        scales[1, there], scales[0, there] = value_scales[kept], got_scales[0, there]
        assert torch.equal(got_scales, scales)
    return q, pool


def plain_formula(qkv, positions, heads, kv, dim, theta):
    x = qkv.double().cpu().reshape(len(qkv), heads + 2 * kv, dim)
    half = dim // 2
    angle = positions.double().cpu()[:, None] * theta ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x[:, : heads + kv, :half], x[:, : heads + kv, half:]
    out = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    size = torch.cat((a.abs() + b.abs(),) * 2, -1)
    return (out[:, :heads], out[:, heads:]), (size[:, :heads], size[:, heads:]), x[:, heads + kv :]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,dim,code", [(*shape, code) for shape in SHAPES for code in CODES
                                               if code != FP4 or shape[2] % 32 == 0])
def test_matches_the_formula(gpu, dtype, heads, kv, dim, code):
    for rows, page, norm in ((1, 16, True), (70, 12, True), (9, 1, False)):
        run_and_check(rows, heads, kv, dim, code, dtype, gpu, page, norm, skipped=min(3, rows - 1))


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("rows", [511, 513, 2049, 5000])
def test_prompts_of_many_rows(gpu, rows, code):
    """The sizes on both sides of the workgroup rules (one row or several to a workgroup)."""
    run_and_check(rows, 6, 2, 128, code, torch.bfloat16, gpu, skipped=7)
    run_and_check(rows, 4, 2, 32, code, torch.float16, gpu, page=64, norm=False)


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_and_misaligned_rows_and_pools(gpu, dtype, code):
    heads, kv, rows = 4, 2, 9
    for dim in (64, 96):
        width = (heads + 2 * kv) * dim
        for offset, stride in ((0, width + 8), (1, width + 3), (4, width + 4)):
            buffer = torch.randn(rows * stride + 8, device=gpu).to(dtype)
            run_and_check(rows, heads, kv, dim, code, dtype, gpu,
                          qkv=buffer[offset : offset + rows * stride].view(rows, stride)[:, :width])
        args = inputs(rows, heads, kv, dim, dtype, gpu)
        want_q, want = run_and_check(rows, heads, kv, dim, code, dtype, gpu)
        for off in (1, 2, 4):  # a pool that starts at an odd element
            fresh = filled(-(-rows // 16) + 2, 16, kv, dim, code, dtype, gpu)
            to = some_rows(rows, 16 * len(fresh if code is None else fresh.codes), gpu)
            store = fresh if code is None else fresh.codes.view(torch.uint8)
            room = torch.empty(store.numel() + off, dtype=store.dtype, device=gpu)
            moved = room[off:].view(store.shape)
            moved.copy_(store)
            pool = moved if code is None else QuantizedPool(moved.view(code), fresh.scales)
            q = norm_rotary_append(args[0], *args[1:3], 1e-6, args[3], to, pool, heads, 1e6)
            (want_q, want_k), (size_q, size_k), want_v = formula(*args[:3], 1e-6, args[3], heads, kv, dim, 1e6)
            check(q, want_q, size_q, dtype)
            got, scales = planes(pool)
            there = to.cpu()
            check_keys(got[0, there], None if scales is None else scales[0, there], want_k, size_k, code, dtype)
            assert alike(code, got[1, there], stored_exactly(want_v, code, dtype)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 224, 256, 512])
def test_unturned_keys_bit_for_bit(gpu, dtype, code, dim):
    """At position 0 without a norm a key reaches the pool exactly: its codes are the definition's,
    values at borders, zeros and groups with a NaN among them."""
    rows, heads, kv = 40, 2, 3
    gen = torch.Generator().manual_seed(dim)
    qkv = torch.randn(rows, heads + 2 * kv, dim, generator=gen) * torch.rand(rows, 1, 1, generator=gen) * 9
    borders = (torch.cat(((FP4_VALUES[1:] + FP4_VALUES[:-1]) / 2, FP4_VALUES)) * 2.0).float()
    qkv[5:15] = borders[torch.randint(0, len(borders), (10, heads + 2 * kv, dim), generator=gen)]
    qkv[3] = 0
    qkv[4, heads, dim // 2 - 1] = float("nan")
    qkv[4, heads + kv + 1, dim // 2] = float("nan")
    qkv = qkv.to(dtype)
    pool = filled(4, 16, kv, dim, code, dtype, gpu)
    to = some_rows(rows, 64, gpu)
    q = norm_rotary_append(qkv.reshape(rows, -1).to(gpu), None, None, 1e-6, torch.zeros(rows, dtype=torch.int64, device=gpu),
                           to, pool, heads, 1e4)
    assert torch.equal(q.cpu(), qkv[:, :heads])
    got, scales = planes(pool)
    x = qkv.clone()
    x[4, heads, -1] = float("nan")  # the pair of a NaN: 0 NaN is NaN
    for plane, part in enumerate((x[:, heads : heads + kv], x[:, heads + kv :])):
        want, want_scales = stored_exactly(part, code, dtype)
        if code is None:
            assert torch.equal(got[plane, to.cpu()].nan_to_num(-99.0), want.nan_to_num(-99.0))
        elif code == FP4:
            ones = torch.full_like(want_scales, 127)  # (a zero's sign may turn)
            assert torch.equal(widen_fp4(got[plane, to.cpu()], ones), widen_fp4(want, ones))
            assert torch.equal(scales[plane, to.cpu()], want_scales)
        else:
            assert alike(code, got[plane, to.cpu()], want)
            assert torch.equal(scales[plane, to.cpu()].nan_to_num(-1), want_scales.nan_to_num(-1))


@pytest.mark.gpu
def test_no_rows_given_outputs_streams_and_replays(gpu):
    heads, kv, dim, rows = 6, 2, 128, 4
    for code in CODES:
        qkv, wq, wk, positions = inputs(rows, heads, kv, dim, torch.bfloat16, gpu)
        pool = filled(3, 16, kv, dim, code, torch.bfloat16, gpu)
        before = planes(pool)
        none = norm_rotary_append(qkv[:0], wq, wk, 1e-6, positions[:0], positions[:0], pool, heads, 1e6)
        assert none.shape == (0, heads, dim) and torch.equal(planes(pool)[0], before[0])
        to = some_rows(rows, 20, gpu)
        guarded = torch.full((rows + 2, heads, dim), 7.0, dtype=torch.bfloat16, device=gpu)
        got = norm_rotary_append(qkv, wq, wk, 1e-6, positions, to, pool, heads, 1e6, out=guarded[1:-1])
        assert got.data_ptr() == guarded[1].data_ptr() and (guarded[0] == 7).all() and (guarded[-1] == 7).all()
        after = planes(pool)
        out = torch.empty_like(got)
        pool = filled(3, 16, kv, dim, code, torch.bfloat16, gpu)
        launch = prepare_norm_rotary_append(qkv, wq, wk, 1e-6, positions, to, pool, heads, 1e6, out)
        side = torch.cuda.Stream(gpu)
        side.wait_stream(torch.cuda.current_stream(torch.device(gpu)))
        with torch.cuda.stream(side):
            launch(side.cuda_stream)
        torch.cuda.current_stream(torch.device(gpu)).wait_stream(side)
        assert torch.equal(out, got) and torch.equal(planes(pool)[0], after[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = norm_rotary_append(qkv, wq, wk, 1e-6, positions, to, pool, heads, 1e6)
        for _ in range(3):  # the positions and rows of the moment are read
            positions += 17
            to += 5
            eager_pool = filled(3, 16, kv, dim, code, torch.bfloat16, gpu)
            store = pool if code is None else pool.codes.view(torch.uint8)
            store.copy_(eager_pool if code is None else eager_pool.codes.view(torch.uint8))
            graph.replay()
            want = norm_rotary_append(qkv, wq, wk, 1e-6, positions, to, eager_pool, heads, 1e6)
            assert torch.equal(captured, want) and torch.equal(planes(pool)[0], planes(eager_pool)[0])


@pytest.mark.gpu
def test_rows_past_32_bit_offsets(gpu):
    blocks, page, kv, dim = 140_000, 16, 8, 128
    qkv, wq, wk, positions = inputs(3, 8, kv, dim, torch.bfloat16, gpu)
    to = torch.tensor([blocks * page - 1, 2**32 // (2 * kv * dim) + 1, 5], device=gpu)
    for code in (FP4, torch.int8):
        pool = QuantizedPool.empty(blocks, page, kv, dim, code, gpu)
        small = QuantizedPool.empty(1, 16, kv, dim, code, gpu)
        norm_rotary_append(qkv, wq, wk, 1e-6, positions, to, pool, 8, 1e6)
        norm_rotary_append(qkv, wq, wk, 1e-6, positions, torch.arange(3, device=gpu), small, 8, 1e6)
        for name in ("codes", "scales"):
            big, want = (getattr(x, name).view(torch.uint8) for x in (pool, small))
            assert torch.equal(big[to // page, :, to % page], want[0].movedim(1, 0)[:3])
            assert int(big.count_nonzero()) == int(want.count_nonzero())


def test_refusals_without_a_gpu():
    qkv, wq, wk, positions = inputs(2, 2, 1, 32, torch.bfloat16, "cpu")
    rows = torch.arange(2)
    plain = torch.zeros(2, 2, 4, 1, 32, dtype=torch.bfloat16)
    four = QuantizedPool.empty(2, 4, 1, 32, FP4, "cpu")
    good = (qkv, wq, wk, 1e-6, positions, rows, plain, 2, 1e4)

    def but(**changes):
        names = ("qkv", "wq", "wk", "eps", "positions", "rows", "pool", "heads", "theta")
        return tuple(changes.get(n, g) for n, g in zip(names, good))

    for match, args in (
        ("qkv", but(qkv=qkv[:, :-1])), ("qkv", but(qkv=qkv[:1].expand(2, -1))), ("qkv", but(heads=3)),
        ("dtype", but(qkv=qkv.double())), ("dtype", but(pool=plain.half())), ("contiguous", but(pool=plain.transpose(0, 2))),
        ("plain pool", but(pool=plain[:, :1])), ("plain pool", but(pool=plain[0])), ("query heads", but(heads=0)),
        ("q_weight", but(wq=wq[:-1])), ("k_weight", but(wk=wk.float())), ("both", but(wk=None)), ("both", but(wq=None)),
        ("positions", but(positions=positions.int())), ("rows", but(rows=rows.int())), ("rows", but(rows=rows[:1])),
        ("rows", but(rows=rows.repeat(2)[::2])), ("qkv", but(pool=QuantizedPool.empty(2, 4, 2, 32, FP4, "cpu"))),
        ("ROCm", good), ("ROCm", but(pool=four)), ("ROCm", but(wq=None, wk=None)),
    ):
        with pytest.raises(ValueError, match=match):
            norm_rotary_append(*args)
    with pytest.raises(ValueError, match="norm_rotary_append"):
        norm_rotary_append(*good, out=torch.zeros(2, 2, 16))


def test_entry_point_refusals_without_a_gpu():
    lib = _lib.load()
    buffer = ctypes.create_string_buffer(256)
    at = ctypes.addressof(buffer)
    at += -at % 16

    def call(rows=1, heads=1, kv=1, dim=32, stride=96, theta=1e4, eps=1e-6, dtype=2, qkv=at, pool=at, scales=at, code=6,
             pool_rows=4, page=4, to=at, wq=at, wk=at, q=at):
        return lib.hs_norm_rotary_append(qkv, stride, wq, wk, eps, q, at, to, rows, heads, theta, dtype, pool, scales,
                                         code, pool_rows, page, kv, dim, None)

    for bad in (dict(rows=-1), dict(heads=0), dict(kv=0), dict(dim=33), dict(dim=16, stride=48), dict(dim=544, stride=4000),
                dict(stride=95), dict(theta=0.0), dict(theta=float("nan")), dict(eps=-1.0), dict(eps=float("nan")),
                dict(dtype=3), dict(qkv=None), dict(pool=None), dict(scales=None), dict(code=5), dict(code=2),
                dict(code=2, scales=None, dtype=1), dict(pool_rows=0), dict(pool_rows=7), dict(page=0), dict(page=8),
                dict(to=None), dict(wq=None), dict(wk=None), dict(q=None), dict(code=3, scales=at + 2),
                dict(rows=2**31), dict(rows=2**24, dim=512, stride=1536), dict(pool_rows=4, page=2**32)):
        assert call(**bad) == -1, bad
        assert lib.hs_last_error()
    assert call(rows=0, qkv=None, to=None, q=None) == 0
