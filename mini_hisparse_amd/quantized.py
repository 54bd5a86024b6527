"""8- and 4-bit K/V rows: a quantised paged pool, written and read by the gfx950 kernels.

A :class:`QuantizedPool` has the layout of a plain pool, ``codes`` [blocks, 2, P, Hkv, D]
(int8 or float8_e4m3fn) beside ``scales`` [blocks, 2, P, Hkv] float32, one scale per head
vector; a row takes ``2 Hkv (D + 4)`` bytes.  In 4 bits, ``codes`` [blocks, 2, P, Hkv, D / 2]
(float4_e2m1fn_x2: two values a byte, the even one in the low half) stand beside ``scales``
[blocks, 2, P, Hkv, D / 32] (float8_e8m0fnu), a power of two for every 32 neighbours; a row
takes ``2 Hkv (D / 2 + D / 32)`` bytes.  :func:`append_quantized` quantises rows as
they are written (a prompt's or one token of each request), :func:`read_quantized` widens
rows again, and ``row_kernels.attend_pages`` attends over the codes themselves.  Rows are
named by physical row (block * P + offset), as everywhere in this package; a call takes up
to 2^25 head vectors of K (rows times KV heads).  No counterpart in the reference, whose
cache holds the model dtype.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib

FP4_GROUP = 32  # neighbours that share a scale of 4-bit codes
# the dtypes of 4-bit codes and their scales; None in builds of torch that lack them
FP4_CODES = getattr(torch, "float4_e2m1fn_x2", None)
FP4_SCALES = getattr(torch, "float8_e8m0fnu", None)


@dataclass(frozen=True, eq=False)
class QuantizedPool:
    """Codes and scales of one pool; ``blocks``, ``page_size``, ``kv_heads``, ``head_dim`` and
    ``rows`` (blocks * page_size) are read off them."""

    codes: torch.Tensor  # [blocks, 2, P, Hkv, D] int8 or float8_e4m3fn, or [.., D / 2] float4_e2m1fn_x2
    scales: torch.Tensor  # [blocks, 2, P, Hkv] float32, or for 4-bit codes [.., D / 32] float8_e8m0fnu

    def __post_init__(self):
        codes, scales = self.codes, self.scales
        code = _lib.cache_code(codes.dtype)
        if codes.dim() != 5 or codes.shape[1] != 2 or 0 in codes.shape or not codes.is_contiguous():
            raise ValueError("codes must be contiguous [blocks, 2, page_size, kv_heads, head_dim]")
        four = code == _lib.HS_DTYPE_E2M1
        if four:
            if codes.shape[4] % (FP4_GROUP // 2):
                raise ValueError("4-bit pools need a head_dim of a multiple of 32")
            if scales.shape != (*codes.shape[:-1], codes.shape[4] * 2 // FP4_GROUP) \
                    or scales.dtype != FP4_SCALES or not scales.is_contiguous():
                raise ValueError("scales must be contiguous float8_e8m0fnu [blocks, 2, page_size, kv_heads, head_dim / 32]")
        elif scales.shape != codes.shape[:-1] or scales.dtype != torch.float32 or not scales.is_contiguous():
            raise ValueError("scales must be contiguous float32 [blocks, 2, page_size, kv_heads]")
        if scales.device != codes.device:
            raise ValueError("codes and scales must be on one device")
        blocks, _, page_size, kv_heads, head_dim = codes.shape
        head_dim = 2 * head_dim if four else head_dim
        for name, value in (("blocks", blocks), ("page_size", page_size), ("kv_heads", kv_heads),
                            ("head_dim", head_dim), ("rows", blocks * page_size), ("code", code),
                            ("device", codes.device), ("vector", (kv_heads, head_dim))):
            object.__setattr__(self, name, value)  # plain attributes: every call reads them

    @classmethod
    def empty(cls, blocks, page_size, kv_heads, head_dim, dtype=torch.int8, device="cuda"):
        """A pool of zeros: every row reads back as zero until it is written."""
        shape = (blocks, 2, page_size, kv_heads, head_dim)
        if dtype is not None and dtype == FP4_CODES:
            if head_dim % FP4_GROUP:
                raise ValueError("4-bit pools need a head_dim of a multiple of 32")
            codes, scales = (torch.zeros((*shape[:-1], n), dtype=torch.uint8, device=device)
                             for n in (head_dim // 2, head_dim // FP4_GROUP))
            return cls(codes.view(dtype), scales.view(FP4_SCALES))
        codes = torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype)
        return cls(codes, torch.zeros(shape[:-1], device=device))

    @property
    def row_bytes(self):
        """Bytes of one token row: codes and scales of K and V of every KV head."""
        if self.code == _lib.HS_DTYPE_E2M1:
            return 2 * self.kv_heads * (self.head_dim // 2 + self.head_dim // FP4_GROUP)
        return 2 * self.kv_heads * (self.head_dim + 4)


def _check_rows(rows, pool, what):
    if rows.dtype != torch.int64 or rows.dim() != 1 or not rows.is_contiguous() or rows.device != pool.device:
        raise ValueError(f"{what}: rows must be contiguous int64 [n] on the pool's device")
    if pool.head_dim > 512:
        raise ValueError(f"{what}: head_dim above 512 is not supported")


def append_quantized(k, v, rows, pool):
    """Quantise K and V rows into ``pool``: token i of ``k`` / ``v`` [tokens, Hkv, D]
    (float32, float16 or bfloat16; any token and head strides) to physical row ``rows[i]``
    (int64, device).  Rows outside the pool (-1) are skipped; the rows of a call must
    differ.  Other rows keep their bits."""
    shape = (*rows.shape[:1], *pool.vector)
    k_stride, v_stride, device, dtype = k.stride(), v.stride(), pool.device, k.dtype
    if (k.shape != shape or v.shape != shape or v.dtype != dtype or k.device != device or v.device != device
            or len(shape) != 3 or (k_stride[2] != 1 or v_stride[2] != 1) and shape[2] > 1):
        raise ValueError("append_quantized: K and V must be [tokens, kv_heads, head_dim] of one dtype on the pool's "
                         "device, head_dim of unit stride")
    code = _lib.dtype_code(dtype)
    _check_rows(rows, pool, "append_quantized")
    if device.type != "cuda":
        raise ValueError("append_quantized needs ROCm device tensors (HIP kernels only)")
    with _lib.on_device(device):
        status = _lib.load().hs_append_quantized(
            k.data_ptr(), k_stride[0], k_stride[1], v.data_ptr(), v_stride[0], v_stride[1], code, rows.data_ptr(),
            shape[0], pool.codes.data_ptr(), pool.scales.data_ptr(), pool.code, pool.rows, pool.page_size,
            pool.kv_heads, pool.head_dim, _lib.stream_handle(device),
        )
    if status:
        _lib.check(status, "hs_append_quantized")


def read_quantized(pool, rows, dtype=torch.bfloat16, out=None):
    """K and V [n, Hkv, D] in ``dtype`` of the physical rows ``rows`` (int64 [n], device):
    code * scale, rounded once (exact from 4 bits, but where the dtype cannot hold it).  A row outside the pool (-1) gives zeros.  ``out``: a (k, v)
    pair to write instead."""
    code = _lib.dtype_code(dtype)
    _check_rows(rows, pool, "read_quantized")
    shape, device = (rows.shape[0], *pool.vector), pool.device
    if out is not None:
        for x in out:
            if x.shape != shape or x.dtype != dtype or x.device != device or not x.is_contiguous():
                raise ValueError("read_quantized: out must be two contiguous [n, kv_heads, head_dim] tensors of "
                                 "dtype on the pool's device")
    if device.type != "cuda":
        raise ValueError("read_quantized needs ROCm device tensors (HIP kernels only)")
    if out is None:
        k = torch.empty(shape, dtype=dtype, device=device)
        v = torch.empty_like(k)
    else:
        k, v = out
    with _lib.on_device(device):
        status = _lib.load().hs_read_quantized(
            pool.codes.data_ptr(), pool.scales.data_ptr(), pool.code, pool.rows, pool.page_size, pool.kv_heads,
            pool.head_dim, rows.data_ptr(), shape[0], k.data_ptr(), v.data_ptr(), code, _lib.stream_handle(device),
        )
    if status:
        _lib.check(status, "hs_read_quantized")
    return k, v
