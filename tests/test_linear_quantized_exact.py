"""Projections with 4-bit weights (linear_quantized) where every sum is exact: bit for bit, at long K above
all, where a tolerance for any order of the sums says little."""

import pytest
import torch

from mini_hisparse_amd.dense import QuantizedWeight, linear_quantized

from page_cases import widen_fp4

DTYPES = [torch.bfloat16, torch.float16]
# one, two and four row tiles a workgroup and the walk; K of several rounds a wave, ending with a round, a
# block and inside one
SHAPES = [(16, 27_648), (33, 18_944), (20, 27_680), (5000, 18_976), (9000, 9024), (16_400, 4256), (16_400, 3616), (24_000, 1056)]


def weight_of(n, k, low, high):
    gen = torch.Generator().manual_seed(n + k)
    codes = torch.randint(0, 256, (n, k // 2), generator=gen, dtype=torch.uint8)
    scales = torch.randint(low, high, (n, k // 32), generator=gen, dtype=torch.uint8)
    return codes, scales, gen


@pytest.mark.gpu
@pytest.mark.parametrize("n,k", SHAPES)
def test_whole_numbers(gpu, n, k):
    """Weights are multiples of 2^-7 (scale bytes 121 and 122, halves) of at most 24 of them, x whole numbers:
    0 or +-1 but for 128 of a row with the type's 8 or 11 significant bits.  The sums of magnitudes are
    at most 24 (k + 128 * 2049) < 2^24 of the unit, float16's second part counted, so fp32 sums are exact in any order
    and an output is the exact product's rounding.  Rows of few tokens are the same as of many."""
    assert 24 * (k + 128 * 2049) < 2**24
    codes, scales, gen = weight_of(n, k, 121, 123)
    w = widen_fp4(codes, scales)
    assert w.abs().max() <= 24 * 2.0**-7 and torch.equal(w * 2**7, (w * 2**7).round())
    weight = QuantizedWeight.pack(codes.to(gpu), scales.to(gpu))
    for dtype, bits in zip(DTYPES, (8, 11)):
        x = torch.randint(-1, 2, (16, k), generator=gen).double()
        for row in x:
            at = torch.randperm(k, generator=gen)[:128]
            row[at] = torch.randint(2 ** (bits - 1), 2**bits, (128,), generator=gen).double() * torch.sign(torch.randn(128, generator=gen))
        x = x.to(dtype)
        bias = torch.randint(-64, 65, (n,), generator=gen).to(dtype)
        product = x.double() @ w.T
        for rows in (16, 1, 7):
            got = linear_quantized(x[:rows].to(gpu), weight).cpu()
            assert torch.equal(got, product[:rows].float().to(dtype))
        got = linear_quantized(x.to(gpu), weight, bias.to(gpu)).cpu()
        assert torch.equal(got, (product + bias.double()).float().to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("n,k", SHAPES)
def test_one_element_at_a_time(gpu, n, k):
    """An x of one element gives that column of the weight times it, rounded: every block, group and
    element is read once, with its own scale, and x in full (255 has bfloat16's 8 bits, 2047
    float16's 11: without its second part it is 2048)."""
    codes, scales, gen = weight_of(n, k, 118, 130)
    w = widen_fp4(codes, scales).float().to(gpu)
    weight = QuantizedWeight.pack(codes.to(gpu), scales.to(gpu))
    step = 1 if n < 64 else 37  # of wide weights some elements of every group of 32 in three
    columns = torch.cat((torch.arange(0, k, step), torch.tensor([k - 1])))
    for dtype, value in zip(DTYPES, (255.0, 2047.0)):
        wrong = torch.zeros((), dtype=torch.int64, device=gpu)
        for at in columns.split(16):
            x = torch.zeros(len(at), k, dtype=dtype, device=gpu)
            x[torch.arange(len(at)), at.to(gpu)] = value
            want = (w[:, at.to(gpu)].T * value).to(dtype)
            wrong += (linear_quantized(x, weight) != want).sum()
        assert int(wrong) == 0
