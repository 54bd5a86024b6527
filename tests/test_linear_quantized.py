"""Projections with 4-bit weights (linear_quantized) against the product in 64 bits, the quantiser
against its definition, and the calls they refuse."""

import ctypes

import pytest
import torch

from mini_hisparse_amd import _lib
from mini_hisparse_amd.dense import QuantizedWeight, linear_quantized, prepare_linear_quantized, quantize_weight

from page_cases import FP4, FP4_VALUES, pack_fp4, quantise_fp4, widen_fp4

DTYPES = [torch.bfloat16, torch.float16]


def unpack(weight):
    """Row-major codes [n, k / 2] and scale bytes [n, k / 32] of a laid-out weight, by the layout's words."""
    tiles, scales, n, k = weight.tiles.cpu(), weight.scales.cpu(), weight.n, weight.k
    codes, bytes_ = torch.zeros(n, k // 2, dtype=torch.uint8), torch.zeros(n, k // 32, dtype=torch.uint8)
    for row in range(n):
        for run in range(k // 32):
            at = 16 * (run % 4) + row % 16
            codes[row, 16 * run : 16 * run + 16] = tiles[row // 16, run // 4, at]
            bytes_[row, run] = scales[row // 16, run // 16, at, run // 4 % 4]
    return codes, bytes_


def random_weight(n, k, device, seed=0, low=115, high=128):
    gen = torch.Generator().manual_seed(seed + n + k)
    codes = torch.randint(0, 256, (n, k // 2), generator=gen, dtype=torch.uint8)
    scales = torch.randint(low, high, (n, k // 32), generator=gen, dtype=torch.uint8)
    return codes, scales, QuantizedWeight.pack(codes.to(device), scales.to(device))


def check(got, x, codes, scales, bias):
    """Half a step of the dtype, and before it the fp32 sums: weights and x are held exactly (float16
    x as two parts, the smaller at most 2^-8 of it) and their products too (at most 8 + 2 bits), so
    the additions, one for each part of K elements, in any order and each off by at most a step,
    2^-23, are off by that many steps of the sum of magnitudes, and the bias by one more of all."""
    w = widen_fp4(codes, scales)
    x = x.double().cpu()
    want, size = x @ w.T, x.abs() @ w.abs().T
    if bias is not None:
        want, size = want + bias.double().cpu(), size + bias.double().cpu().abs()
    parts = 2 if got.dtype == torch.float16 else 1
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() + (parts * x.shape[1] + 2) * 2.0**-23 * size * (1 + 2.0**-8)
    if got.dtype == torch.float16:
        tol = tol + 2.0**-25  # half a subnormal step
    error = (got.double().cpu() - want).abs()
    over = ~(error <= tol)
    assert not over.any(), (error[over].max().item(), tol[over].max().item())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k", [(1, 32), (16, 128), (17, 96), (1152, 896), (896, 896), (100, 4864), (33, 160), (5, 2080),
                                 (640, 512), (24_000, 512), (40_000, 256), (33_000, 160), (16_400, 672), (16, 27_648),
                                 (5000, 640), (9000, 288), (16_500, 1568), (16_401, 4096), (17_000, 3616),
                                 (16_385, 4128)])
def test_matches_the_product(gpu, dtype, n, k):
    codes, scales, weight = random_weight(n, k, gpu)
    gen = torch.Generator().manual_seed(1)
    for rows in (1, 5, 16):
        x = torch.randn(rows, k, generator=gen).to(dtype).to(gpu)
        bias = torch.randn(n, generator=gen).to(dtype).to(gpu) if rows != 5 else None
        check(linear_quantized(x, weight, bias), x, codes, scales, bias)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_number_of_rows_alike(gpu, dtype):
    """A row's bits do not depend on the rows beside it."""
    for n, k in ((1152, 896), (5000, 640), (17_000, 288), (16_400, 2080)):
        codes, scales, weight = random_weight(n, k, gpu)
        x = torch.randn(16, k, device=gpu).to(dtype)
        full = linear_quantized(x, weight)
        check(full, x, codes, scales, None)
        for rows in range(1, 16):
            assert torch.equal(linear_quantized(x[:rows], weight), full[:rows])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_scales_of_every_size(gpu, dtype):
    """Weights from 2^-60 to 2^60, far outside float16's range, with x of either sign of it."""
    for low, high, size in ((67, 70, 2.0**10), (185, 188, 2.0**-14), (67, 187, 1.0)):
        codes, scales, weight = random_weight(64, 640, gpu, low=low, high=high)
        x = (torch.randn(3, 640) * size).to(dtype).to(gpu)
        got = linear_quantized(x, weight)
        if dtype == torch.bfloat16:
            check(got, x, codes, scales, None)
        else:  # an output past float16's range is infinite, below it zero
            want = (x.double().cpu() @ widen_fp4(codes, scales).T)
            assert torch.equal(got.isinf().cpu(), want.abs() >= 65520)
            if high == 70:
                assert (got == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_and_infinity_reach_their_rows_alone(gpu, dtype):
    for n, k in ((40, 160), (16_400, 1568)):
        codes, scales, _ = random_weight(n, k, "cpu")
        scales[7, 3] = 255
        weight = QuantizedWeight.pack(codes.to(gpu), scales.to(gpu))
        x = torch.randn(4, k).to(dtype)
        x[2, k - 1] = float("nan")
        x[3, 0] = float("inf")
        y = linear_quantized(x.to(gpu), weight).cpu()
        assert y[:, 7].isnan().all() and y[2].isnan().all()
        good = torch.arange(n) != 7
        assert y[:2][:, good].isfinite().all()
        # an infinity times its weight: NaN for a weight of 0, as in the plain product
        first = widen_fp4(codes, scales)[:, 0]
        want = torch.where(first == 0, float("nan"), first.sign() * float("inf"))[good]
        assert torch.equal(y[3, good].isnan(), want.isnan())
        assert torch.equal(y[3, good].nan_to_num(0.0, 1.0, -1.0).double(), want.nan_to_num(0.0, 1.0, -1.0))


@pytest.mark.gpu
def test_strided_rows_outputs_streams_and_replays(gpu):
    n, k, rows = 200, 224, 5
    codes, scales, weight = random_weight(n, k, gpu)
    wide = torch.full((rows, k + 40), float("nan"), dtype=torch.bfloat16, device=gpu)
    wide[:, 8 : 8 + k] = torch.randn(rows, k, device=gpu)
    x = wide[:, 8 : 8 + k]
    bias = torch.randn(n, device=gpu).to(torch.bfloat16)
    want = linear_quantized(x.contiguous(), weight, bias)
    check(want, x, codes, scales, bias)
    guarded = torch.full((rows + 2, n + 3), 7.0, dtype=torch.bfloat16, device=gpu)
    out = guarded[1:-1, 1 : n + 1]
    got = linear_quantized(x, weight, bias, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, want)
    out.fill_(7.0)
    assert (guarded == 7).all()
    launch = prepare_linear_quantized(x, weight, bias, out)
    side = torch.cuda.Stream(torch.device(gpu))
    side.wait_stream(torch.cuda.current_stream(torch.device(gpu)))
    with torch.cuda.stream(side):
        launch(side.cuda_stream)
    torch.cuda.current_stream(torch.device(gpu)).wait_stream(side)
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = linear_quantized(x, weight, bias)
    for _ in range(3):
        wide[:, 8 : 8 + k].normal_()
        graph.replay()
        assert torch.equal(captured, linear_quantized(x, weight, bias))
        check(captured, x, codes, scales, bias)


def quantised_exactly(weight, w):
    codes, scales = quantise_fp4(w)
    got_codes, got_scales = unpack(weight)
    assert torch.equal(got_scales, scales)
    assert torch.equal(got_codes, pack_fp4(codes))


@pytest.mark.parametrize("n,k", [(1, 32), (18, 160), (40, 640), (3, 2080)])
@pytest.mark.parametrize("dtype", [torch.float32, *DTYPES])
def test_quantised_weights_are_the_definition(dtype, n, k):
    gen = torch.Generator().manual_seed(n)
    w = torch.randn(n, k, generator=gen) * torch.rand(n, 1, generator=gen) * 0.05
    borders = (torch.cat(((FP4_VALUES[1:] + FP4_VALUES[:-1]) / 2, FP4_VALUES, torch.tensor([7.0]))) * 2.0**-5).float()
    w[0] = borders[torch.randint(0, len(borders), (k,), generator=gen)]
    w[-1, :32] = 0
    if n > 1:
        w[1, 3], w[1, 31] = float("nan"), float("inf")
    if dtype != torch.float16:
        w[-1, -32:] = 2.0**-130
    w = w.to(dtype)
    quantised_exactly(quantize_weight(w), w)


@pytest.mark.gpu
def test_quantised_on_the_gpu(gpu):
    w = (torch.randn(300, 640, device=gpu) * 0.02).to(torch.bfloat16)
    weight = quantize_weight(w)
    quantised_exactly(weight, w)
    x = torch.randn(4, 640, device=gpu).to(torch.bfloat16)
    check(linear_quantized(x, weight), x, *unpack(weight), None)


def test_layouts_and_refusals_without_a_gpu():
    codes, scales, weight = random_weight(19, 672, "cpu")
    assert all(torch.equal(a, b) for a, b in zip(unpack(weight), (codes, scales)))
    same = QuantizedWeight.pack(codes.view(FP4), scales.view(torch.float8_e8m0fnu))
    assert torch.equal(same.tiles, weight.tiles) and torch.equal(same.scales, weight.scales)
    turned = QuantizedWeight.pack(codes.T.contiguous().T, scales)
    assert torch.equal(turned.tiles, weight.tiles)
    for bad in ((codes.int(), scales), (codes[:, :-1], scales), (codes, scales[:, :-1]), (codes, scales.float()),
                (codes[0], scales[0]), (codes[:0], scales[:0])):
        with pytest.raises(ValueError):
            QuantizedWeight.pack(*bad)
    for bad in ((weight.tiles, weight.scales, 40, 672), (weight.tiles, weight.scales, 19, 670),
                (weight.tiles[:1], weight.scales, 19, 672), (weight.tiles.int(), weight.scales, 19, 672),
                (weight.tiles.transpose(0, 1), weight.scales, 19, 672), (weight.tiles, weight.scales, 0, 672)):
        with pytest.raises(ValueError):
            QuantizedWeight(*bad)
    for bad in (torch.zeros(3, 48), torch.zeros(32), torch.zeros(0, 32), torch.zeros(2, 32).double()):
        with pytest.raises(ValueError):
            quantize_weight(bad)
    x = torch.zeros(4, 672, dtype=torch.bfloat16)
    for match, args in (
        ("1-16 rows", (torch.zeros(17, 672, dtype=torch.bfloat16), weight)), ("1-16 rows", (x[:0], weight)),
        ("1-16 rows", (x.float(), weight)), ("1-16 rows", (x[:, :640], weight)), ("1-16 rows", (x[0], weight)),
        ("1-16 rows", (torch.zeros(4, 676, dtype=torch.bfloat16)[:, :672], weight)),
        ("1-16 rows", (torch.zeros(4, 680, dtype=torch.bfloat16)[:, 4:676], weight)),
        ("1-16 rows", (x[:1].expand(4, -1), weight)),
        ("bias", (x, weight, torch.zeros(19))), ("bias", (x, weight, torch.zeros(18, dtype=torch.bfloat16))),
        ("ROCm", (x, weight)), ("ROCm", (x, weight, torch.zeros(19, dtype=torch.bfloat16))),
    ):
        with pytest.raises(ValueError, match=match):
            linear_quantized(*args)
    with pytest.raises(ValueError, match="out"):
        linear_quantized(x, weight, out=torch.zeros(4, 18, dtype=torch.bfloat16))


def test_entry_point_refusals_without_a_gpu():
    lib = _lib.load()
    buffer = ctypes.create_string_buffer(256)
    at = ctypes.addressof(buffer)
    at += -at % 16

    def call(x=at, stride=64, tiles=at, scales=at, n=16, k=64, out=at, out_stride=16, rows=2, dtype=2):
        return lib.hs_skinny_gemm_fp4(x, stride, tiles, scales, n, k, None, out, out_stride, rows, dtype, None)

    for bad in (dict(x=None), dict(tiles=None), dict(scales=None), dict(out=None), dict(stride=60), dict(stride=56),
                dict(n=0), dict(n=2**28 + 1, out_stride=2**29), dict(k=0), dict(k=48), dict(k=2**30, stride=2**30), dict(out_stride=15),
                dict(rows=0), dict(rows=17), dict(dtype=0), dict(dtype=3), dict(x=at + 2), dict(tiles=at + 8),
                dict(scales=at + 2)):
        assert call(**bad) == -1, bad
        assert lib.hs_last_error()
