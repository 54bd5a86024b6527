"""Per-head norms of q and k with the rotary embedding (norm_rotary_split) against the
formula in 64 bits, and the calls it refuses."""

import ctypes

import pytest
import torch

from mini_hisparse_amd import _lib
from mini_hisparse_amd.dense import norm_rotary_split, prepare_norm_rotary_split, rotary_split

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def inputs(rows, heads, kv, dim, dtype, device, seed=0):
    gen = torch.Generator().manual_seed(seed + rows + dim)
    qkv = (torch.randn(rows, (heads + 2 * kv) * dim, generator=gen) * 2).to(dtype)
    wq, wk = ((torch.rand(dim, generator=gen) * 2 - 0.5).to(dtype) for _ in range(2))
    positions = torch.randint(0, 200_000, (rows,), generator=gen)
    positions[0] = 0
    return tuple(t.to(device) for t in (qkv, wq, wk, positions))


def formula(qkv, wq, wk, eps, positions, heads, kv, dim, theta):
    """(q, k, v) in 64 bits and, for q and k, the sum of magnitudes of each output's two terms."""
    x = qkv.double().cpu().reshape(len(qkv), heads + 2 * kv, dim)
    half = dim // 2
    inverse = theta ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    angle = positions.double().cpu()[:, None] * inverse
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    out, terms = [], []
    for part, w in ((x[:, :heads], wq), (x[:, heads : heads + kv], wk)):
        n = part * torch.rsqrt(part.square().mean(-1, keepdim=True) + eps) * w.double().cpu()
        a, b = n[..., :half], n[..., half:]
        out.append(torch.cat((a * cos - b * sin, b * cos + a * sin), -1))
        size = a.abs() + b.abs()
        terms.append(torch.cat((size, size), -1))
    return out, terms, x[:, heads + kv :]


def check(got, want, terms, dtype):
    """One rounding to the dtype, and in fp32 before it: the mean of squares (at most D/16 + 8
    steps a lane and its butterfly, halved by the root), the root, two products, cos and sin
    and the rotation: under 64 half steps of 2^-24 of the two terms for D <= 512."""
    error = (got.double().cpu() - want).abs()
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 64 * 2.0**-24 * terms
    if dtype == torch.float16:
        tol = tol + 2.0**-25  # half a subnormal step
    assert (error <= tol).all(), (error - tol).max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,dim", [(28, 4, 128), (14, 2, 64), (4, 2, 32), (3, 1, 256), (12, 3, 96), (5, 5, 80),
                                          (2, 1, 6), (1, 1, 2), (2, 2, 512), (3, 1, 100)])
@pytest.mark.parametrize("rows", [1, 3, 70])
def test_matches_the_formula(gpu, dtype, heads, kv, dim, rows):
    args = inputs(rows, heads, kv, dim, dtype, gpu)
    qkv, wq, wk, positions = args
    q, k, v = norm_rotary_split(qkv, wq, wk, 1e-6, positions, heads, kv, dim, 1e6)
    (want_q, want_k), (size_q, size_k), want_v = formula(qkv, wq, wk, 1e-6, positions, heads, kv, dim, 1e6)
    check(q, want_q, size_q, dtype)
    check(k, want_k, size_k, dtype)
    assert torch.equal(v.double().cpu(), want_v)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [511, 513, 2049, 5000])
def test_prompts_of_many_rows(gpu, rows):
    """The sizes on both sides of the workgroup rules (one row or several to a workgroup)."""
    heads, kv, dim = 6, 2, 128
    qkv, wq, wk, _ = inputs(rows, heads, kv, dim, torch.bfloat16, gpu)
    positions = torch.arange(100_000, 100_000 + rows, device=gpu)
    q, k, v = norm_rotary_split(qkv, wq, wk, 1e-6, positions, heads, kv, dim, 1e4)
    (want_q, want_k), (size_q, size_k), want_v = formula(qkv, wq, wk, 1e-6, positions, heads, kv, dim, 1e4)
    check(q, want_q, size_q, torch.bfloat16)
    check(k, want_k, size_k, torch.bfloat16)
    assert torch.equal(v.double().cpu(), want_v)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_and_misaligned_rows(gpu, dtype):
    heads, kv, dim, rows = 4, 2, 64, 9
    width = (heads + 2 * kv) * dim
    for offset, stride in ((0, width + 8), (1, width + 3), (4, width + 4)):
        buffer = torch.randn(rows * stride + 8, device=gpu).to(dtype)
        qkv = buffer[offset : offset + rows * stride].view(rows, stride)[:, :width]
        _, wq, wk, positions = inputs(rows, heads, kv, dim, dtype, gpu)
        got = norm_rotary_split(qkv, wq, wk, 1e-5, positions, heads, kv, dim, 1e4)
        (want_q, want_k), (size_q, size_k), want_v = formula(qkv, wq, wk, 1e-5, positions, heads, kv, dim, 1e4)
        check(got[0], want_q, size_q, dtype)
        check(got[1], want_k, size_k, dtype)
        assert torch.equal(got[2].double().cpu(), want_v)


@pytest.mark.gpu
def test_zero_rows_nan_rows_and_large_values(gpu):
    heads, kv, dim = 2, 1, 128
    qkv, wq, wk, positions = inputs(4, heads, kv, dim, torch.float32, gpu)
    qkv[0] = 0
    qkv[1, 5] = float("nan")  # head 0 of row 1
    qkv[2] *= 1e15
    q, k, v = norm_rotary_split(qkv, wq, wk, 1e-6, positions, heads, kv, dim, 1e6)
    assert (q[0] == 0).all() and (k[0] == 0).all()
    assert q[1, 0].isnan().all() and q[1, 1].isfinite().all() and k[1].isfinite().all()
    (want_q, want_k), (size_q, size_k), _ = formula(qkv, wq, wk, 1e-6, positions, heads, kv, dim, 1e6)
    check(q[2:], want_q[2:], size_q[2:], torch.float32)
    check(k[2:], want_k[2:], size_k[2:], torch.float32)


@pytest.mark.gpu
def test_unit_weights_at_unit_rows_agree_with_rotary_split(gpu):
    """Heads of unit mean square and unit weights: the norm leaves them, so the rotation is
    rotary_split's up to its own roundings (cos, sin, products and sum in bfloat16)."""
    heads, kv, dim, rows = 4, 2, 64, 5
    gen = torch.Generator().manual_seed(1)
    signs = (torch.randint(0, 2, (rows, (heads + 2 * kv) * dim), generator=gen) * 2 - 1).to(torch.bfloat16).to(gpu)
    ones = torch.ones(dim, dtype=torch.bfloat16, device=gpu)
    positions = torch.arange(rows, device=gpu)
    got = norm_rotary_split(signs, ones, ones, 0.0, positions, heads, kv, dim, 1e4)
    ref = rotary_split(signs, positions, heads, kv, dim, 1e4)
    for a, b in zip(got, ref):
        assert (a.float() - b.float()).abs().max().item() <= 5 * 2.0**-8 * 2


@pytest.mark.gpu
def test_prepared_call_stream_and_graph(gpu):
    heads, kv, dim, rows = 6, 2, 128, 4
    qkv, wq, wk, positions = inputs(rows, heads, kv, dim, torch.bfloat16, gpu)
    out = (torch.empty(rows, heads, dim, dtype=torch.bfloat16, device=gpu),
           *(torch.empty(rows, kv, dim, dtype=torch.bfloat16, device=gpu) for _ in range(2)))
    launch = prepare_norm_rotary_split(qkv, wq, wk, 1e-6, positions, heads, kv, dim, 1e6, out)
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(torch.device(gpu)))
    with torch.cuda.stream(side):
        launch(side.cuda_stream)
    torch.cuda.current_stream(torch.device(gpu)).wait_stream(side)
    for a, b in zip(out, norm_rotary_split(qkv, wq, wk, 1e-6, positions, heads, kv, dim, 1e6)):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = norm_rotary_split(qkv, wq, wk, 1e-6, positions, heads, kv, dim, 1e6)
    for step in range(3):  # the positions of the moment are read
        positions += 17
        graph.replay()
        for a, b in zip(captured, norm_rotary_split(qkv, wq, wk, 1e-6, positions, heads, kv, dim, 1e6)):
            assert torch.equal(a, b)


def test_refusals_without_a_gpu():
    qkv, wq, wk, positions = inputs(2, 2, 1, 8, torch.bfloat16, "cpu")
    call = lambda *a, **kw: norm_rotary_split(*a, **kw)  # noqa: E731
    with pytest.raises(ValueError, match="qkv"):
        call(qkv[:, :-1], wq, wk, 1e-6, positions, 2, 1, 8, 1e4)
    with pytest.raises(ValueError, match="even head_dim"):
        call(qkv, wq, wk, 1e-6, positions, 2, 1, 7, 1e4)
    with pytest.raises(ValueError, match="even head_dim"):
        call(qkv, wq, wk, 1e-6, positions, 0, 1, 8, 1e4)
    with pytest.raises(ValueError, match="q_weight"):
        call(qkv, wq[:-1], wk, 1e-6, positions, 2, 1, 8, 1e4)
    with pytest.raises(ValueError, match="k_weight"):
        call(qkv, wq, wk.float(), 1e-6, positions, 2, 1, 8, 1e4)
    with pytest.raises(ValueError, match="positions"):
        call(qkv, wq, wk, 1e-6, positions.int(), 2, 1, 8, 1e4)
    with pytest.raises(ValueError, match="positions"):
        call(qkv, wq, wk, 1e-6, positions.repeat(2)[::2], 2, 1, 8, 1e4)
    with pytest.raises(ValueError, match="at least one row"):
        call(qkv[:0], wq, wk, 1e-6, positions[:0], 2, 1, 8, 1e4)
    with pytest.raises(ValueError, match="overlap"):
        call(qkv[:1].expand(2, -1), wq, wk, 1e-6, positions, 2, 1, 8, 1e4)
    with pytest.raises(ValueError, match="out"):
        call(qkv, wq, wk, 1e-6, positions, 2, 1, 8, 1e4, out=(qkv, qkv, qkv))
    with pytest.raises(ValueError, match="ROCm"):
        call(qkv, wq, wk, 1e-6, positions, 2, 1, 8, 1e4)


def test_entry_point_refusals_without_a_gpu():
    lib = _lib.load()
    buffer = ctypes.create_string_buffer(256)
    at = ctypes.addressof(buffer)

    def call(rows=1, heads=1, kv=1, dim=8, stride=24, theta=1e4, eps=1e-6, dtype=2, qkv=at):
        return lib.hs_norm_rotary_split(qkv, stride, at, at, eps, at, at, at, at, rows, heads, kv, dim, theta, dtype,
                                        None)

    for bad in (dict(rows=0), dict(heads=0), dict(dim=7), dict(dim=514, stride=4000), dict(stride=23), dict(theta=0.0),
                dict(theta=float("inf")), dict(theta=float("nan")), dict(eps=-1.0), dict(eps=float("nan")),
                dict(dtype=3), dict(qkv=None)):
        assert call(**bad) == -1, bad
        assert lib.hs_last_error()


def test_more_rows_than_a_grid_holds_are_refused_without_a_gpu():
    lib = _lib.load()
    buffer = ctypes.create_string_buffer(256)
    at = ctypes.addressof(buffer)
    for rows in (2**24, 2**31 - 1, 2**31):
        assert lib.hs_norm_rotary_split(at, 1536, at, at, 1e-6, at, at, at, at, rows, 1, 1, 512, 1e4, 2, None) == -1
        assert b"too many rows" in lib.hs_last_error()
