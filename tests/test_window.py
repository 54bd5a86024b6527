"""Attention over page tables through a sliding window with first tokens that stay, against softmax
attention in 64 bits; every row outside the window holds NaN or its page is gone."""

import ctypes
import shutil
import subprocess

import pytest
import torch

from mini_hisparse_amd import _lib, build
from mini_hisparse_amd.quantized import QuantizedPool
from mini_hisparse_amd.row_kernels import attend_pages

from page_cases import case, check

POOLS = [("fp4", "bf16"), ("fp4", "f16"), ("fp4", "f32"), ("int8", "bf16"), ("e4m3", "f32"), ("bf16", "bf16"),
         ("f16", "f16"), ("f32", "f32")]
WIDE = 20_000  # columns more of a table: the launch for long histories, where the window is long too
WINDOWS = [(1, 0), (1, 1), (31, 4), (32, 4), (33, 0), (64, 33), (100, 16), (100, 70), (500, 1), (4000, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("code,dtype", POOLS)
def test_windows_of_every_pool(gpu, code, dtype, window, sinks):
    for page in (16, 5):
        lengths = [333, 0, window, window + sinks, window + sinks + 1, 97, 1]
        args = case(7, 14, 2, 64, page, lengths, code, dtype, gpu, window=window, sinks=sinks, wide=page * 7)
        check(attend_pages(*args, window=window, sinks=sinks), args, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,dim", [(28, 4, 128), (4, 2, 32), (6, 3, 96), (3, 1, 256), (5, 5, 160), (20, 1, 64),
                                          (2, 2, 512)])
@pytest.mark.parametrize("code,dtype", [("fp4", "bf16"), ("int8", "bf16"), ("f32", "f32")])
def test_head_layouts(gpu, heads, kv, dim, code, dtype):
    for window, sinks in ((48, 4), (777, 40)):
        args = case(2, heads, kv, dim, 16, [1500, 700], code, dtype, gpu, window=window, sinks=sinks)
        check(attend_pages(*args, window=window, sinks=sinks), args, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("code,dtype", [("fp4", "bf16"), ("e4m3", "bf16"), ("bf16", "bf16")])
@pytest.mark.parametrize("page", [1, 12, 16, 48, 64])
def test_lengths_around_the_window_and_pages(gpu, page, code, dtype):
    for window, sinks in ((64, 32), (65, 31), (90, 7)):
        lengths = [window + sinks + n for n in (-2, -1, 0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 160)]
        args = case(len(lengths), 8, 4, 128, page, lengths, code, dtype, gpu, window=window, sinks=sinks)
        check(attend_pages(*args, window=window, sinks=sinks), args, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("code,dtype", [("fp4", "bf16"), ("int8", "f16"), ("f16", "f16"), ("f32", "f32")])
def test_long_windows_absent_pages_and_tables_per_head(gpu, code, dtype):
    """Windows over the launch for long histories, and over several parts of a short one."""
    for page in (16, 12):
        for window, sinks in ((9000, 100), (1500, 0)):
            for per_head in (False, True):
                args = case(2, 14, 2, 64, page, [12_000, 1600], code, dtype, gpu, window=window, sinks=sinks, absent=0.3,
                            per_head=per_head, wide=WIDE)
                check(attend_pages(*args, window=window, sinks=sinks), args, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [64, 65, 200, 1100])
def test_many_requests(gpu, batch):
    """The schedule of a wave's lanes and the one written out, with windows shorter than some requests."""
    gen = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, 400, (batch,), generator=gen)
    lengths[::9] = 0
    lengths[batch // 2], lengths[-1] = 9000, 5000
    for window, sinks in ((100, 4), (4500, 40)):
        args = case(batch, 4, 2, 32, 16, lengths.tolist(), "int8", "bf16", gpu, window=window, sinks=sinks, wide=200)
        check(attend_pages(*args, window=window, sinks=sinks), args, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("code,dtype", [("fp4", "bf16"), ("int8", "bf16"), ("f32", "f32")])
def test_a_window_of_everything_is_no_window(gpu, code, dtype):
    """The same launch gives the same bits with and without a window that every token is in; a window
    of any size is accepted."""
    for dim, wide in ((64, 2), (64, WIDE), (160, 2)):
        args = case(3, 14, 2, dim, 16, [500, 33, 0], code, dtype, gpu, wide=wide)
        want = attend_pages(*args)
        everything = args[2].shape[1] * 16
        for window, sinks in ((everything, 0), (2**31 - 1, 2**31 - 1), (2**31, 7), (2**62, 2**62)):
            assert torch.equal(attend_pages(*args, window=window, sinks=sinks), want)
        check(attend_pages(*args, window=1, sinks=2**40), args)  # every token is a first one


@pytest.mark.gpu
def test_replays_with_other_lengths(gpu):
    """A captured call follows the lengths and tables of the moment, with work between the replays."""
    window, sinks = 300, 20
    for code, dtype, dim in (("fp4", "bf16", 128), ("bf16", "bf16", 64), ("int8", "bf16", 80)):
        query, pool, tables, lengths = case(3, 8, 2, dim, 16, [2000, 900, 321], code, dtype, gpu)
        graph, out = torch.cuda.CUDAGraph(), torch.empty_like(query)
        attend_pages(query, pool, tables, lengths, window=window, sinks=sinks)
        with torch.cuda.graph(graph):
            attend_pages(query, pool, tables, lengths, window=window, sinks=sinks, out=out)
        for now in ([2000, 900, 310], [0, 1, 299], [300, 320, 321], [1777, 0, 33]):
            lengths.copy_(torch.tensor(now, dtype=torch.int32))
            out.fill_(7.0)
            graph.replay()
            assert torch.equal(out, attend_pages(query, pool, tables, lengths, window=window, sinks=sinks))
            check(out, (query, pool, tables, lengths), window, sinks)


@pytest.mark.gpu
def test_offsets_past_32_bits_and_misaligned_pools(gpu):
    """A window at the far end of a pool of more than 2^32 elements, and pools that start at odd bytes."""
    blocks, page, kv, dim = 140_000, 16, 8, 128
    pool = QuantizedPool.empty(blocks, page, kv, dim, torch.float4_e2m1fn_x2, gpu)
    lengths = torch.tensor([100_000], dtype=torch.int32, device=gpu)
    tables = torch.arange(blocks - 6250, blocks, dtype=torch.int32, device=gpu)[None]
    codes, scales = pool.codes.view(torch.uint8), pool.scales.view(torch.uint8)
    gen = torch.Generator(device=gpu).manual_seed(0)
    codes[-700:] = torch.randint(0, 256, codes[-700:].shape, dtype=torch.uint8, device=gpu, generator=gen)
    codes[blocks - 6250] = torch.randint(0, 256, codes[0].shape, dtype=torch.uint8, device=gpu, generator=gen)
    scales[-6250:] = torch.randint(125, 129, scales[-6250:].shape, dtype=torch.uint8, device=gpu, generator=gen)
    query = torch.randn(1, 16, dim, device=gpu, generator=gen).to(torch.bfloat16)
    got = attend_pages(query, pool, tables, lengths, window=10_000, sinks=16)
    small = QuantizedPool(codes[-6250:].clone().view(torch.float4_e2m1fn_x2),
                          scales[-6250:].clone().view(torch.float8_e8m0fnu))
    args = (query, small, tables - (blocks - 6250), lengths)
    assert torch.equal(got, attend_pages(*args, window=10_000, sinks=16))
    check(got, args, 10_000, 16)
    for dim in (64, 128, 160, 256):
        args = query, pool, tables, lengths = case(2, 4, 2, dim, 16, [900, 40], "fp4", "bf16", gpu, window=100, sinks=5)
        for codes_off, scales_off in ((1, 0), (0, 1), (2, 3), (16, 8), (8, 8)):
            parts = []
            for x, off in ((pool.codes.view(torch.uint8), codes_off), (pool.scales.view(torch.uint8), scales_off)):
                room = torch.empty(x.numel() + off, dtype=torch.uint8, device=gpu)
                parts.append(room[off:].view(x.shape))
                parts[-1].copy_(x)
            moved = QuantizedPool(parts[0].view(torch.float4_e2m1fn_x2), parts[1].view(torch.float8_e8m0fnu))
            check(attend_pages(query, moved, tables, lengths, window=100, sinks=5), args, 100, 5)


def test_refusals_without_a_gpu():
    pool = torch.zeros(4, 2, 16, 2, 8)
    query, lengths = torch.zeros(3, 4, 8), torch.zeros(3, dtype=torch.int32)
    tables = torch.zeros(3, 2, dtype=torch.int32)
    for match, options in (("sinks", dict(sinks=4)), ("at least one", dict(window=0)), ("at least one", dict(window=-5)),
                           ("not negative", dict(window=5, sinks=-1)), ("2\\^63", dict(window=2**63)),
                           ("2\\^63", dict(window=5, sinks=2**63)), ("ROCm", dict(window=5, sinks=2))):
        with pytest.raises(ValueError, match=match):
            attend_pages(query, pool, tables, lengths, **options)


def test_entry_point_refusals_without_a_gpu():
    lib = _lib.load()
    buffer = ctypes.create_string_buffer(256)
    at = ctypes.addressof(buffer)
    at += -at % 16

    def call(code=6, dim=64, window=0, sinks=0, pages=1000, scales=at, nbytes=1 << 40):
        return lib.hs_attend_pages_window(at, 2 * dim, dim, 2, at, scales, code, 4, 16, 1, dim, at, pages, 0, pages, at,
                                          1, 2, window, sinks, at, 2 * dim, dim, at, nbytes, None)

    for bad in (dict(window=-1), dict(sinks=-1), dict(sinks=3), dict(window=5, sinks=-2), dict(dim=80), dict(dim=544),
                dict(scales=None), dict(code=5), dict(code=7), dict(nbytes=16)):
        assert call(**bad) == -1, bad
        assert lib.hs_last_error()
    size = lib.hs_attend_pages_window_workspace_bytes
    assert size(2, 6, 4, 14, 2, 64, 16, 1000, 0, 0) == lib.hs_attend_pages_workspace_bytes(2, 6, 4, 14, 2, 64, 16, 1000)
    assert size(2, 6, 4, 14, 2, 64, 16, 1000, 0, 0) > 0 and size(2, 6, 4, 14, 2, 64, 16, 1000, 100, 4) == 0
    assert size(2, 6, 4, 14, 2, 64, 16, 1000, -1, 4) == 256


SEEN = r"""
#include "page_parts.h"
using namespace hs;
// Whether the tiles that a window of a request of n tokens walks show exactly its tokens, each once.
extern "C" int64_t shown(int32_t n, int32_t window, int32_t sinks, int32_t* first, int32_t* last) {
  const Seen v = seen_of(n, window, sinks);
  const int32_t tiles = seen_tiles(n, window, sinks);
  int64_t count = 0;
  *first = -1;
  *last = -1;
  for (int32_t t = 0; t < tiles; ++t) {
    const int32_t base = PM_TILE * (t + (t >= v.front ? v.gap : 0));
    const int32_t left = n - base;
    uint32_t mask = left >= PM_TILE ? 0xffffffffu : (1u << left) - 1u;
    if (base < v.lo) mask &= seen_mask(base, v.lo, sinks);
    for (int i = 0; i < PM_TILE; ++i)
      if (mask >> i & 1) {
        const int32_t token = base + i;
        if (token <= *last || token >= n || (token < n - static_cast<int64_t>(window) && token >= sinks)) return -1;
        if (*first < 0) *first = token;
        *last = token;
        ++count;
      }
  }
  if (tiles > most_seen_tiles(n, window, sinks)) return -2;
  return count;
}
extern "C" int64_t most(int64_t tokens, int32_t window, int32_t sinks) { return most_seen_tiles(tokens, window, sinks); }
extern "C" int64_t walked(int32_t n, int32_t window, int32_t sinks) { return seen_tiles(n, window, sinks); }
"""


@pytest.fixture(scope="module")
def seen(tmp_path_factory):
    if shutil.which(build.HIPCC) is None:
        pytest.skip("hipcc is not installed")
    folder = tmp_path_factory.mktemp("seen")
    (folder / "seen.hip").write_text(SEEN)
    command = [build.HIPCC, "--offload-arch=gfx950", "-O2", "-std=c++17", "-fPIC", "-shared", f"-I{build.CSRC}",
               str(folder / "seen.hip"), "-o", str(folder / "seen.so")]
    subprocess.run(command, check=True, capture_output=True)
    lib = ctypes.CDLL(str(folder / "seen.so"))
    lib.shown.restype = lib.most.restype = lib.walked.restype = ctypes.c_int64
    lib.most.argtypes = [ctypes.c_int64, ctypes.c_int32, ctypes.c_int32]
    return lib


def test_the_tiles_walked_show_exactly_the_window(seen):
    first, last = ctypes.c_int32(), ctypes.c_int32()
    for n in [*range(0, 140), 200, 321, 1000]:
        for window in (1, 2, 31, 32, 33, 63, 64, 65, 100, 2**31 - 1):
            for sinks in (0, 1, 4, 31, 32, 33, 64, 90, 2**31 - 1):
                count = seen.shown(n, window, sinks, ctypes.byref(first), ctypes.byref(last))
                assert count == min(n, window + sinks), (n, window, sinks, count)
                assert count == 0 or (last.value == n - 1 and first.value == (0 if sinks else max(0, n - window)))


def test_long_windows_keep_to_32_bits(seen):
    longest = 2**31 - 1
    for n in (longest, longest - 1, 2**30):
        for window in (1, 4096, 2**30, longest):
            for sinks in (0, 50, 2**30, longest):
                walked = seen.walked(n, window, sinks)
                assert -(-min(n, window + sinks) // 32) <= walked <= seen.most(n, window, sinks) <= -(-n // 32)
