"""The 4-bit decode operators' measured cases: each operator in plain torch and as a user calls it.

A case is a plain dict with a ``kind`` (which operator) and its sizes:

  store    K/V rows written in 4 bits into a paged pool and a history read back from it:
           ``append_quantized`` then ``read_quantized``
  rotary   a packed q|k|v projection, q and k normed per head (or not) and rotated, K and V
           written to a paged pool on the way: ``norm_rotary_append``
  attend   one new token's attention over page tables, the cache held in 4 bits, or seen
           through a sliding window with a few first tokens, or both: ``attend_pages``
  linear   a decode projection with 4-bit weights and group scales: ``linear_quantized``

4-bit values are e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), two to a byte (the even
index in the low half), with one power of two for every 32 neighbours, held as a byte: e
stands for 2^(e - 127), 255 for NaN.

``own`` chooses between the plain forms and the package's kernels.  ``run`` is one pass of
a case's operator; ``exact`` is the same result from the definition in 64 bits.
"""

from __future__ import annotations

from math import ceil

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127, "e4m3": 448}
BYTES = {"bf16": 2, "f16": 2, "f32": 4, "int8": 1, "e4m3": 1, "fp4": 0.5}
GROUP = 32  # neighbours that share a scale of 4-bit values
EPS = 1e-6


def listed():
    return [
        # one new token's K/V at the 0.5B shape, read back alone: latency only
        dict(name="store-one", kind="store", tokens=1, history=0, kv=2, dim=64, page=16, dtype="bf16"),
        # a 16k-token prompt written in one call at the 7B shape and read back for its prefill
        dict(name="store-prompt", kind="store", tokens=16384, history=0, kv=4, dim=128, page=16, dtype="bf16"),
        # a decode batch at the 7B shape, positions spread up to 128k, into a plain pool
        dict(name="rotary-decode", kind="rotary", rows=16, heads=28, kv=4, dim=128, first=-1, theta=1e6, norm=False,
             page=16, code="bf16", dtype="bf16"),
        # a 16k-token prompt of normed heads at the 7B shape, one token short of a power of two, into 8 bits
        dict(name="rotary-prompt", kind="rotary", rows=16383, heads=28, kv=4, dim=128, first=0, theta=1e6, norm=True,
             page=16, code="int8", dtype="bf16"),
        # one short conversation at the 0.5B shape, the cache in 4 bits
        dict(name="attend-one", kind="attend", batch=1, heads=14, kv=2, dim=64, tokens=1999, ragged=0, page=16,
             code="fp4", dtype="bf16", window=0, sinks=0, idle=False),
        # the 7B shape's whole histories of 128k tokens in 4 bits
        dict(name="attend-7b", kind="attend", batch=8, heads=28, kv=4, dim=128, tokens=131072, ragged=1021, page=16,
             code="fp4", dtype="bf16", window=0, sinks=0, idle=False),
        # the 32B shape: many histories of uneven lengths in 4 bits, one slot idle
        dict(name="attend-32b", kind="attend", batch=16, heads=40, kv=8, dim=128, tokens=65536, ragged=3001, page=16,
             code="fp4", dtype="f16", window=0, sinks=0, idle=True),
        # one long conversation at the 0.5B shape, its newest 1024 tokens and the first four, unquantised
        dict(name="window-one", kind="attend", batch=1, heads=14, kv=2, dim=64, tokens=32749, ragged=0, page=16,
             code="bf16", dtype="bf16", window=1024, sinks=4, idle=False),
        # a batch of the 7B shape's 64k-token histories through a window of 4096 tokens, in 8 bits
        dict(name="window-7b", kind="attend", batch=16, heads=28, kv=4, dim=128, tokens=65536, ragged=1021, page=16,
             code="int8", dtype="bf16", window=4096, sinks=16, idle=False),
        # the 0.5B shape's packed q|k|v projection of one token
        dict(name="linear-one", kind="linear", rows=1, n=1152, k=896, bias=True, dtype="bf16"),
        # the 7B shape's packed gate|up projection of a full decode batch
        dict(name="linear-batch", kind="linear", rows=16, n=37888, k=3584, bias=False, dtype="bf16"),
        # the 7B shape's LM head for four requests
        dict(name="linear-head", kind="linear", rows=4, n=152064, k=3584, bias=False, dtype="f16"),
    ]


def _log(rng, low, high):
    """A whole number from low to high, spread over its logarithm."""
    return min(high, max(low, round(low * (high / low) ** rng.random())))


# (query heads, KV heads, head dim): the framework's configurations, then other groupings
_HEADS = ((14, 2, 64), (28, 4, 128), (40, 8, 128), (64, 8, 128), (4, 2, 32), (8, 8, 64), (16, 1, 128), (12, 3, 96))


def draw(rng):
    kind = rng.choice(("store", "rotary", "rotary", "attend", "attend", "attend", "linear", "linear"))
    heads, kv, dim = rng.choice(_HEADS)
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    page = rng.choice((16, 16, 16, 32, 64, 8, 1, 12))
    if kind == "store":
        tokens = _log(rng, 1, 12000 if kv * dim <= 512 else 6000)
        return dict(kind=kind, tokens=tokens, history=rng.choice((0, 0, _log(rng, 16, 12000))), kv=kv, dim=dim,
                    page=page, dtype=dtype)
    if kind == "rotary":
        far = rng.random() < 0.4
        rows = _log(rng, 1, 200) if far else _log(rng, 1, min(12000, 16383 * 4608 * 2 // ((heads + 2 * kv) * dim * 4)))
        code = rng.choice((dtype, "int8", "e4m3")) if dtype != "f32" else dtype
        return dict(kind=kind, rows=rows, heads=heads, kv=kv, dim=dim, first=-1 if far else rng.randint(0, 100000),
                    theta=rng.choice((1e4, 1e6)), norm=rng.random() < 0.5, page=page, code=code, dtype=dtype)
    if kind == "linear":
        rows, k = rng.randint(1, 16), 32 * _log(rng, 2, 256)
        return dict(kind=kind, rows=rows, n=_log(rng, 1, min(40000, 37888 * 3584 // k)), k=k,
                    bias=rng.random() < 0.5, dtype=rng.choice(("bf16", "f16")))
    code = rng.choice(("fp4", "fp4", "int8", "e4m3", dtype))
    batch = _log(rng, 1, 32)
    tokens = _log(rng, 1, {"f32": 100000, "f16": 300000, "bf16": 300000}.get(code, 600000) // batch)
    window = _log(rng, 1, tokens) if code != "fp4" or rng.random() < 0.4 else 0
    return dict(kind=kind, batch=batch, heads=heads, kv=kv, dim=dim, tokens=tokens,
                ragged=rng.randint(0, max(0, tokens // (2 * batch))), page=page, code=code, dtype=dtype,
                window=window, sinks=rng.choice((0, 1, 4, 16, 50)) if window else 0,
                idle=batch > 1 and rng.random() < 0.3)


# ------------------------------------------------------------------------------- inputs


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _kv_values(shape, gen, dtype):
    """K/V ~ N(0, 1) with 2% of the channels (at least one) eight times as large."""
    x = torch.randn(shape, generator=gen, device=DEVICE)
    channels = torch.randperm(shape[-1], generator=gen, device=DEVICE)[: max(1, round(0.02 * shape[-1]))]
    x[..., channels] *= 8
    return x.to(dtype)


def _filled_pool(blocks, case, gen):
    """A paged pool [blocks, 2, P, Hkv, D] of random rows (4-bit ones [.., D / 2] bytes) and,
    where it is quantised, its scales."""
    shape, code = (blocks, 2, case["page"], case["kv"], case["dim"]), case["code"]
    if code in DTYPES:
        return _kv_values(shape, gen, DTYPES[code]), None
    if code == "fp4":
        codes = torch.empty((*shape[:-1], shape[-1] // 2), dtype=torch.uint8, device=DEVICE)
        scales = torch.empty((*shape[:-1], shape[-1] // GROUP), dtype=torch.uint8, device=DEVICE)
    else:
        codes = torch.empty(shape, dtype=torch.uint8, device=DEVICE)
        scales = torch.empty(shape[:-1], device=DEVICE)
    step = max(1, (1 << 26) // (2 * shape[2] * shape[3] * shape[4]))
    for i in range(0, blocks, step):
        part = _kv_values((min(step, blocks - i), *shape[1:]), gen, torch.bfloat16)
        codes[i : i + step], scales[i : i + step] = _plain_fp4(part) if code == "fp4" else _plain_8bit(part, code)
    return codes, scales


def _lengths(case):
    lengths = [max(1, case["tokens"] - i * case["ragged"]) for i in range(case["batch"])]
    if case["idle"]:
        lengths[case["batch"] // 2] = 0
    return lengths


def _tables(case, gen):
    """Page tables of a batch of whole histories, their blocks in any order."""
    pages = [ceil(n / case["page"]) for n in _lengths(case)]
    blocks = max(1, sum(pages))
    order = torch.randperm(blocks, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.full((case["batch"], max(1, max(pages))), -1, dtype=torch.int32, device=DEVICE)
    first = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[first : first + n]
        first += n
    return table, blocks


def prepare(case, seed):
    gen = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    heads, kv, dim = case.get("heads"), case.get("kv"), case.get("dim")
    state = dict(case=case)
    if case["kind"] == "linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        state["x"] = torch.randn(rows, k, generator=gen, device=DEVICE).to(dtype)
        state["bias"] = torch.randn(n, generator=gen, device=DEVICE).to(dtype) if case["bias"] else None
        state["codes"] = torch.empty(n, k // 2, dtype=torch.uint8, device=DEVICE)
        state["scales"] = torch.empty(n, k // GROUP, dtype=torch.uint8, device=DEVICE)
        step = max(1, (1 << 26) // k)
        for i in range(0, n, step):
            part = torch.randn(min(step, n - i), k, generator=gen, device=DEVICE) * k**-0.5
            state["codes"][i : i + step], state["scales"][i : i + step] = _plain_fp4(part)
        if own:  # laid out once, as a program keeps its weights
            from mini_hisparse_amd.dense import QuantizedWeight

            state["weight"] = QuantizedWeight.pack(state["codes"], state["scales"])
        return state
    if case["kind"] == "attend":
        state["host_lengths"] = _lengths(case)
        state["tables"], blocks = _tables(case, gen)
        state["lengths"] = torch.tensor(state["host_lengths"], dtype=torch.int32, device=DEVICE)
        state["query"] = torch.randn(case["batch"], heads, dim, generator=gen, device=DEVICE).to(dtype)
    else:
        written = case["rows"] if case["kind"] == "rotary" else case["tokens"]
        total = written + case.get("history", 0)
        pages = ceil(total / case["page"])
        blocks = pages + 3  # blocks of other requests, left as they are
        table = torch.randperm(blocks, generator=gen, device=DEVICE)[:pages]
        token = torch.arange(total, device=DEVICE)
        state["read"] = table[token // case["page"]] * case["page"] + token % case["page"]
        state["rows"] = state["read"][total - written :].contiguous()
    state["codes"], state["scales"] = _filled_pool(blocks, {"code": "fp4", **case}, gen)
    if case["kind"] == "store":
        state["k"] = _kv_values((case["tokens"], kv, dim), gen, dtype)
        state["v"] = _kv_values((case["tokens"], kv, dim), gen, dtype)
    if case["kind"] == "rotary":
        rows = case["rows"]
        state["qkv"] = (torch.randn(rows, (heads + 2 * kv) * dim, generator=gen, device=DEVICE) * 2).to(dtype)
        state["wq"] = (torch.rand(dim, generator=gen, device=DEVICE) + 0.5).to(dtype) if case["norm"] else None
        state["wk"] = (torch.rand(dim, generator=gen, device=DEVICE) + 0.5).to(dtype) if case["norm"] else None
        if case["first"] < 0:  # a decode batch: every request at a position of its own
            state["positions"] = torch.randint(0, 131072, (rows,), generator=gen, device=DEVICE)
        else:
            state["positions"] = torch.arange(case["first"], case["first"] + rows, device=DEVICE)
    if own:
        from mini_hisparse_amd.quantized import QuantizedPool

        if case.get("code", "fp4") == "fp4":
            state["pool"] = QuantizedPool(state["codes"].view(torch.float4_e2m1fn_x2),
                                          state["scales"].view(torch.float8_e8m0fnu))
        elif case["code"] in CODES:
            state["pool"] = QuantizedPool(state["codes"].view(CODES[case["code"]]), state["scales"])
        else:
            state["pool"] = state["codes"]
    return state


# --------------------------------------------------------------------------- plain forms


def _plain_fp4(x):
    """4-bit codes and scale bytes of groups of 32: the scale is the smallest power of two, from
    2^-126 on, that takes the largest magnitude to at most 7; a code is the nearest of the
    quotient, ties to the even one, no larger than 6."""
    wide = x.float().unflatten(-1, (-1, GROUP))
    largest = wide.abs().amax(-1)
    finite = largest.isfinite()
    part, power = torch.frexp(torch.where(finite, largest, 0.0))
    power = torch.where(largest > 0, torch.where(part <= 0.875, power - 3, power - 2), -126).clamp(min=-126)
    quotient = torch.where(finite[..., None], wide, 0.0).double() * torch.exp2(-power.double())[..., None]
    size = quotient.abs()
    code = ((size > 0.25).byte() + (size >= 0.75).byte() + (size > 1.25).byte() + (size >= 1.75).byte()
            + (size > 2.5).byte() + (size >= 3.5).byte() + (size > 5).byte())
    code = (code | (quotient.signbit().byte() << 3)).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.where(finite, power + 127, 255).to(torch.uint8)


def _plain_widen_fp4(codes, scales):
    """The values of 4-bit codes [.., D / 2] with scale bytes [.., D / 32], in 32 bits."""
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    size = (code & 7).float()
    value = torch.where(size < 2, size * 0.5, (1 + 0.5 * (size % 2)) * torch.exp2(torch.floor(size / 2) - 1))
    value = torch.where(code > 7, -value, value).unflatten(-1, (-1, GROUP))
    scale = torch.where(scales < 255, torch.exp2(scales.float() - 127), float("nan"))
    return (value * scale[..., None]).flatten(-2)


def _plain_8bit(x, code):
    """8-bit codes (as bytes) and scales of head vectors: the scale is the largest magnitude over
    the code's largest, a code the nearest of the quotient (taken in 64 bits: values next to a
    border)."""
    wide = x.float()
    largest = wide.abs().amax(-1)
    scales = torch.where(largest.isfinite(), (largest.double() / TOP[code]).float(), float("nan"))
    quotient = wide.double() / scales.double()[..., None]
    quotient = torch.where((scales > 0)[..., None], quotient, 0.0).clamp(-TOP[code], TOP[code])
    if code == "int8":
        return quotient.round().to(torch.int8).view(torch.uint8), scales
    step = torch.exp2((torch.frexp(quotient)[1] - 4).clamp(min=-9).double())  # spacing of the grid there
    return ((quotient / step).round() * step).float().to(torch.float8_e4m3fn).view(torch.uint8), scales


def _plain_widen(codes, scales, code):
    """Rows of a pool in 32 bits."""
    if code == "fp4":
        return _plain_widen_fp4(codes, scales)
    if code in CODES:
        return codes.view(CODES[code]).float() * scales[..., None]
    return codes.float()


def _plain_write(state, k, v, code):
    """K and V rows [n, Hkv, D] of 32 bits into the pool, and the whole history back in the dtype."""
    case, codes, scales = state["case"], state["codes"], state["scales"]
    block, within = state["rows"] // case["page"], state["rows"] % case["page"]
    for plane, x in enumerate((k, v)):
        if code in DTYPES:
            codes[block, plane, within] = x.to(codes.dtype)
        else:
            codes[block, plane, within], scales[block, plane, within] = (_plain_fp4(x) if code == "fp4"
                                                                         else _plain_8bit(x, code))
    if code in DTYPES:
        return codes
    block, within = state["read"] // case["page"], state["read"] % case["page"]
    k, v = (_plain_widen(codes[block, p, within], scales[block, p, within], code).to(DTYPES[case["dtype"]])
            for p in (0, 1))
    return k, v, scales


def _plain_rotary(state):
    case, qkv = state["case"], state["qkv"]
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    parts = qkv.view(len(qkv), heads + 2 * kv, dim).float()
    # angles of far positions need 64 bits: one part in 2^24 of 10^5 radians is a hundredth
    inverse = case["theta"] ** (-torch.arange(0, dim, 2, device=qkv.device).double() / dim)
    angle = state["positions"].double()[:, None] * inverse
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x, weight):
        if weight is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
        a, b = x[..., : dim // 2], x[..., dim // 2 :]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    q = turned(parts[:, :heads], state["wq"]).to(qkv.dtype)
    k = turned(parts[:, heads : heads + kv], state["wk"])
    return q, _plain_write(state, k, parts[:, heads + kv :], case["code"])


def _plain_attend(state):
    case, codes, scales = state["case"], state["codes"], state["scales"]
    page, kv, dim = case["page"], case["kv"], case["dim"]
    out = torch.zeros_like(state["query"])
    for b, n in enumerate(state["host_lengths"]):
        if n == 0:
            continue
        token = torch.arange(n, device=codes.device)
        if case["window"] and case["window"] + case["sinks"] < n:  # the first tokens and the newest ones
            token = torch.cat((token[: case["sinks"]], token[n - case["window"] :]))
        block, within = state["tables"][b][token // page].long(), token % page
        k, v = (_plain_widen(codes[block, p, within], None if scales is None else scales[block, p, within],
                             case["code"]).transpose(0, 1) for p in (0, 1))
        q = state["query"][b].float().view(kv, -1, dim)
        scores = torch.matmul(q, k.transpose(1, 2)) * dim**-0.5
        weights = (scores - scores.amax(-1, keepdim=True)).exp()
        out[b] = (torch.matmul(weights, v) / weights.sum(-1, keepdim=True)).view(-1, dim).to(out.dtype)
    return out


def _plain_linear(state):
    y = state["x"].float() @ _plain_widen_fp4(state["codes"], state["scales"]).T
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(state["x"].dtype)


# --------------------------------------------------------------------------------- passes


def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        if kind == "store":
            return _plain_write(state, state["k"], state["v"], "fp4")
        return {"rotary": _plain_rotary, "attend": _plain_attend, "linear": _plain_linear}[kind](state)
    if kind == "linear":
        from mini_hisparse_amd.dense import linear_quantized

        return linear_quantized(state["x"], state["weight"], state["bias"])
    if kind == "attend":
        from mini_hisparse_amd.row_kernels import attend_pages

        return attend_pages(state["query"], state["pool"], state["tables"], state["lengths"],
                            window=case["window"] or None, sinks=case["sinks"])
    from mini_hisparse_amd.quantized import append_quantized, read_quantized

    if kind == "store":
        append_quantized(state["k"], state["v"], state["rows"], state["pool"])
        return (*read_quantized(state["pool"], state["read"], DTYPES[case["dtype"]]), state["scales"])
    from mini_hisparse_amd.dense import norm_rotary_append

    q = norm_rotary_append(state["qkv"], state["wq"], state["wk"], EPS, state["positions"], state["rows"],
                           state["pool"], case["heads"], case["theta"])
    if case["code"] in DTYPES:
        return q, state["codes"]
    return q, (*read_quantized(state["pool"], state["read"], DTYPES[case["dtype"]]), state["scales"])


def _row_bytes(kv, dim, code):
    scales = dim / GROUP if code == "fp4" else 4 if code in CODES else 0
    return 2 * kv * (dim * BYTES[code] + scales)


def work(case):
    size = BYTES[case["dtype"]]
    if case["kind"] == "linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": n * (k // 2 + k // GROUP) + rows * (n + k) * size + (n * size if case["bias"] else 0),
                "flops": 2 * rows * n * k}
    kv, dim = case["kv"], case["dim"]
    if case["kind"] == "attend":
        tokens = entries = 0
        for n in _lengths(case):
            seen = min(n, case["window"] + case["sinks"]) if case["window"] else n
            tokens += seen
            entries += ceil(seen / case["page"])
        return {"bytes": tokens * _row_bytes(kv, dim, case["code"]) + 4 * entries
                + 2 * case["batch"] * case["heads"] * dim * size,
                "flops": 4 * tokens * case["heads"] * dim}
    if case["kind"] == "store":
        written, read, code, moved = case["tokens"], case["tokens"] + case["history"], "fp4", 0
        row = 2 * kv * dim * size
        flops = (4 * written + read) * 2 * kv * dim
    else:
        written, code = case["rows"], case["code"]
        read = 0 if code in DTYPES else written
        row = 2 * kv * dim * size
        moved = written * (2 * case["heads"] * dim * size + 8)  # q in and out, the positions
        flops = 10 * written * (case["heads"] + 2 * kv) * dim
    stored = _row_bytes(kv, dim, code)
    return {"bytes": moved + written * (row + 8 + stored) + read * (8 + stored + row), "flops": flops}


# ------------------------------------------------------------------- the definition, 64 bits


def _exact_grid(code):
    """The magnitudes a code can stand for, ascending."""
    if code == "int8":
        values = list(range(128))
    elif code == "fp4":
        values = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    else:  # e4m3: eight steps an octave from 2^-6 up to 448, and multiples of 2^-9 below
        values = [m * 2.0**-9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127]
    return torch.tensor(values, dtype=torch.float64, device=DEVICE)


def _exact_rounded(x, scale, code):
    """x as the nearest multiple of scale that the code can stand for, ties to the even code."""
    grid = _exact_grid(code)
    ratio = (x.abs() / scale.clamp(min=1e-300)).clamp(max=float(grid[-1]))
    low = (torch.searchsorted(grid, ratio, right=True) - 1).clamp(0, len(grid) - 2)
    middle = (grid[low] + grid[low + 1]) / 2
    up = (ratio > middle) | ((ratio == middle) & (low % 2 == 1))
    return torch.where(up, grid[low + 1], grid[low]) * x.sign() * scale


def _exact_stored(x, code):
    """Head vectors as a quantised pool holds them, and its scales (4-bit ones as bytes)."""
    if code != "fp4":
        scale = (x.abs().amax(-1) / TOP[code]).float().double()  # held in float32
        return _exact_rounded(x, scale[..., None], code), scale
    groups = x.unflatten(-1, (-1, GROUP))
    power = torch.ceil(torch.log2(groups.abs().amax(-1).clamp(min=1e-300) / 7)).clamp(min=-126)
    # the logarithm next to a whole number, settled
    power = torch.where(groups.abs().amax(-1) <= 7 * torch.exp2(power - 1), power - 1, power)
    power = torch.where(groups.abs().amax(-1) > 7 * torch.exp2(power), power + 1, power).clamp(min=-126)
    return _exact_rounded(groups, torch.exp2(power)[..., None], code).flatten(-2), power + 127


def _exact_values(codes, scales, code):
    """Any rows of a pool in 64 bits."""
    if code == "fp4":
        grid = _exact_grid("fp4")
        table = torch.cat((grid, -grid))
        pairs = torch.stack((table[(codes % 16).long()], table[(codes // 16).long()]), -1).flatten(-2)
        powers = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=codes.device), scales.double() - 127)
        return pairs * powers.repeat_interleave(GROUP, -1)
    if code in CODES:
        return codes.view(CODES[code]).float().double() * scales.double()[..., None]
    return codes.double()


def _exact_pool(case, state, k, v):
    """What a pool and its reader give after K and V (64 bits) have been written."""
    code, page = case.get("code", "fp4"), case["page"]
    if code in DTYPES:
        planes = state["codes"].double().movedim(1, 0).flatten(1, 2).contiguous()  # [2, rows, Hkv, D]
        planes[:, state["rows"]] = torch.stack((k, v))
        return planes.unflatten(1, (-1, page)).movedim(0, 1)
    planes = _exact_values(state["codes"], state["scales"], code).movedim(1, 0).flatten(1, 2).contiguous()
    scales = state["scales"].double().movedim(1, 0).flatten(1, 2).contiguous()
    for plane, x in enumerate((k, v)):
        planes[plane, state["rows"]], scales[plane, state["rows"]] = _exact_stored(x, code)
    scales = scales.unflatten(1, (-1, page)).movedim(0, 1)
    return planes[0, state["read"]], planes[1, state["read"]], scales.to(torch.uint8) if code == "fp4" else scales


def _exact_rotary(case, state):
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    x = state["qkv"].to(torch.float64).reshape(-1, heads + 2 * kv, dim)
    exponent = torch.arange(dim // 2, dtype=torch.float64, device=x.device) * (-2.0 / dim)
    turn = torch.outer(state["positions"].to(torch.float64), torch.pow(case["theta"], exponent))
    unit = torch.polar(torch.ones_like(turn), turn)[:, None, :]
    result = []
    for part, weight in ((x[:, :heads], state["wq"]), (x[:, heads : heads + kv], state["wk"])):
        if weight is not None:
            part = part / ((part * part).sum(-1, keepdim=True) / dim + EPS).sqrt() * weight.to(torch.float64)
        turned = torch.complex(part[..., : dim // 2], part[..., dim // 2 :]) * unit
        result.append(torch.cat((turned.real, turned.imag), -1))
    return result[0], _exact_pool(case, state, result[1], x[:, heads + kv :])


def _exact_attend(case, state):
    page, kv, heads, dim = case["page"], case["kv"], case["heads"], case["dim"]
    group, scales = heads // kv, state["scales"]
    result = torch.zeros(case["batch"], heads, dim, dtype=torch.float64, device=DEVICE)
    for b, n in enumerate(state["host_lengths"]):
        token = torch.arange(n, device=DEVICE)
        if case["window"]:
            token = token[(token >= n - case["window"]) | (token < case["sinks"])]
        if len(token) == 0:
            continue
        block, within = state["tables"][b][token // page].long(), token % page
        for h in range(kv):
            k, v = (_exact_values(state["codes"][block, p, within, h],
                                  None if scales is None else scales[block, p, within, h], case["code"])
                    for p in (0, 1))
            q = state["query"][b, h * group : (h + 1) * group].double()
            result[b, h * group : (h + 1) * group] = torch.softmax((q @ k.T) / dim**0.5, -1) @ v
    return result


def _exact_linear(case, state):
    result = torch.empty(case["rows"], case["n"], dtype=torch.float64, device=DEVICE)
    for i in range(0, case["n"], 16384):
        weight = _exact_values(state["codes"][i : i + 16384], state["scales"][i : i + 16384], "fp4")
        result[:, i : i + 16384] = state["x"].double() @ weight.T
    return result if state["bias"] is None else result + state["bias"].double()


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = kept
    if case["kind"] == "store":
        return _exact_pool(case, state, state["k"].double(), state["v"].double())
    return {"rotary": _exact_rotary, "attend": _exact_attend, "linear": _exact_linear}[case["kind"]](case, state)
