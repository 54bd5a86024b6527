"""Batches over page tables with pools of every kind, a window, and attention over them in 64 bits."""

import torch

from mini_hisparse_amd.quantized import QuantizedPool

PLAIN = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EIGHT = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
FP4 = torch.float4_e2m1fn_x2
FP4_VALUES = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def quantise_fp4(x):
    """Codes (0 .. 15) [.., D] and scale bytes [.., D / 32] by the definition, in 64 bits on the CPU."""
    x = x.detach().cpu().double().unflatten(-1, (-1, 32))
    largest = x.abs().amax(-1)
    finite = largest.isfinite()
    powers = torch.full_like(largest, -126.0)
    for k in range(-126, 127):  # the smallest power of two that is at least a seventh of the largest
        powers = torch.where(largest > 7 * 2.0**k, float(k + 1), powers)
    ratio = torch.where(finite[..., None], x, 0.0) / torch.exp2(powers)[..., None]
    size = ratio.abs().clamp(max=6.0)
    low = (torch.searchsorted(FP4_VALUES, size, right=True) - 1).clamp(0, 6)
    middle = (FP4_VALUES[low] + FP4_VALUES[low + 1]) / 2
    up = (size > middle) | ((size == middle) & (low % 2 == 1))
    codes = low + up.long() + 8 * ratio.signbit().long()
    return codes.flatten(-2).to(torch.uint8), torch.where(finite, powers + 127, 255.0).to(torch.uint8)


def pack_fp4(codes):
    return (codes[..., 0::2] | codes[..., 1::2] << 4).contiguous()


def widen_fp4(codes, scales):
    """Values in 64 bits of packed codes and scale bytes."""
    codes, scales = codes.cpu().view(torch.uint8), scales.cpu().view(torch.uint8)
    codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    values = FP4_VALUES[codes & 7] * torch.where(codes > 7, -1.0, 1.0)
    powers = torch.where(scales == 255, float("nan"), torch.exp2(scales.double() - 127))
    return values * powers.repeat_interleave(32, -1)


def store_of(pool):
    """A pool's values in 64 bits."""
    if not isinstance(pool, QuantizedPool):
        return pool.cpu().double()
    if pool.codes.dtype == FP4:
        return widen_fp4(pool.codes, pool.scales)
    return pool.codes.cpu().float().double() * pool.scales.cpu().double()[..., None]


def pool_of(values, code, junk, device):
    """A pool of values [blocks, 2, P, Hkv, D] whose rows `junk` [blocks, P, Hkv] hold NaN."""
    junk = junk[:, None].expand(-1, 2, -1, -1)
    if code in PLAIN:
        stored = values.to(PLAIN[code])
        stored[junk] = float("nan")
        return stored.to(device)
    if code == "fp4":
        codes, scales = quantise_fp4(values)
        codes[junk], scales[junk] = 0xB, 255
        return QuantizedPool(pack_fp4(codes).to(device).view(FP4), scales.to(device).view(torch.float8_e8m0fnu))
    top = 127.0 if code == "int8" else 448.0
    scales = values.abs().amax(-1) / top
    stored = values / scales[..., None]
    stored = (stored.round() if code == "int8" else stored).clamp(-top, top).to(EIGHT[code])
    scales[junk] = float("nan")
    stored.view(torch.int8)[junk] = 0x7F
    return QuantizedPool(stored.to(device), scales.to(device))


def seen_tokens(n, window, sinks):
    token = torch.arange(n)
    return token if window is None else token[(token >= n - window) | (token < sinks)]


def case(batch, heads, kv, dim, page, lengths, code, dtype, device, window=None, sinks=0, seed=0, absent=0.0,
         per_head=False, spare=3, wide=2):
    """A batch whose tables are scattered over the pool.  Rows that no request sees (past a
    length, outside its window, of blocks in no table) hold NaN, pages of which none is seen
    are gone from the tables every other time, and of the others `absent` are too."""
    gen = torch.Generator().manual_seed(seed + dim + page + sum(lengths))
    lists = kv if per_head else 1
    pages = [-(-n // page) for n in lengths]
    width = max(1, max(pages)) + wide
    blocks = lists * sum(pages) + spare
    order = torch.randperm(blocks, generator=gen)
    tables = torch.randint(-3, blocks + 3, (batch, lists, width), generator=gen)  # past the pages: anything
    values = torch.randn(blocks, 2, page, kv, dim, generator=gen)
    values[..., : max(1, dim // 50)] *= 8
    used = torch.zeros(blocks, page, kv, dtype=torch.bool)
    taken = 0
    for b, n in enumerate(lengths):
        token = seen_tokens(n, window, sinks)
        some = torch.zeros(pages[b], dtype=torch.bool)
        some[token // page] = True
        for h in range(lists):
            mine = order[taken : taken + pages[b]]
            taken += pages[b]
            tables[b, h, : pages[b]] = mine
            gone = torch.where(some, torch.rand(pages[b], generator=gen) < absent, torch.rand(pages[b], generator=gen) < 0.5)
            where = gone.nonzero()[:, 0]
            tables[b, h, where] = torch.tensor([-1, blocks, -(2**31), 2**31 - 1])[where % 4]
            here = token[~gone[token // page]]
            if per_head:
                used[mine[here // page], here % page, h] = True
            else:
                used[mine[here // page], here % page] = True
    pool = pool_of(values, code, ~used, device)
    query = torch.randn(batch, heads, dim, generator=gen).to(PLAIN[dtype])
    tables = (tables if per_head else tables[:, 0]).to(torch.int32)
    return query.to(device), pool, tables.to(device), torch.tensor(lengths, dtype=torch.int32, device=device)


def formula(query, pool, tables, lengths, window=None, sinks=0):
    """(out, weighted sum of |V|, largest sum of |q K| D^-1/2, largest |score|, tokens) in 64 bits."""
    store = store_of(pool)
    query, tables, lengths = query.cpu().double(), tables.cpu().long(), lengths.cpu().tolist()
    blocks, _, page, kv, dim = store.shape
    batch, heads, _ = query.shape
    group = heads // kv
    out, weight, size, top, count = (torch.zeros(batch, heads, n, dtype=torch.float64) for n in (dim, dim, 1, 1, 1))
    for b, n in enumerate(lengths):
        token = seen_tokens(max(0, min(n, tables.shape[-1] * page)), window, sinks)
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


def check(got, args, window=None, sinks=0):
    """|error| <= half a step of the dtype, and before that rounding the weights' error times the
    weighted |V| twice (numerator and sum): with u = 2^-24, a score is off by at most D u of
    its sum of magnitudes, three roundings of the score and 4 u of its size again in the
    exponential's argument; the exponential by 4 u; the sums of n tokens and their rescalings by
    (n + 16) u; a weight held as the sum of two bfloat16 parts by 2^-16, of two float16 parts
    (float16 pools) by 2^-22 and 2^-25 of the largest, of three bfloat16 parts (float32
    queries) by 2^-24.  4-bit values and their products with the powers of two are exact.  A
    weight below 2^-126 of the largest may be held as 0."""
    query, pool = args[0], args[1]
    want, weight, size, top, count = formula(*args, window, sinks)
    u, dim = 2.0**-24, query.shape[-1]
    f16 = not isinstance(pool, QuantizedPool) and query.dtype == torch.float16
    held = 2.0**-24 if query.dtype == torch.float32 else 2.0**-22 if f16 else 2.0**-16
    weights = (dim + 4) * u * size + 8 * u * top + 4 * u + (count + 16) * u + held
    largest = store_of(pool).nan_to_num(0.0).abs().amax().item()
    tol = torch.finfo(query.dtype).eps / 2 * want.abs() + 2 * weights * weight
    tol = tol + count * 2.0**-126 * largest + (count * 2.0**-25 * largest if f16 else 0)
    if query.dtype == torch.float16:
        tol = tol + 2.0**-25  # half a subnormal step
    error = (got.double().cpu() - want).abs()
    over = ~(error <= tol)
    assert not over.any(), (error[over].max().item(), tol[over].max().item())
