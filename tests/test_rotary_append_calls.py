"""Calls of norm_rotary_append at the edges of what it documents."""

import ctypes

import pytest
import torch

from mini_hisparse_amd import _lib
from mini_hisparse_amd.dense import norm_rotary_append
from mini_hisparse_amd.quantized import QuantizedPool

from test_norm_rotary import check, formula, inputs
from test_rotary_append import (CODES, DTYPES, alike, check_keys, filled, plain_formula, planes, some_rows,
                                stored_exactly)


def test_eps_without_a_norm_is_not_looked_at_by_the_entry_point():
    lib = _lib.load()
    buffer = ctypes.create_string_buffer(256)
    at = ctypes.addressof(buffer)
    at += -at % 16

    def call(weight, eps):  # no rows: nothing is launched
        return lib.hs_norm_rotary_append(None, 96, weight, weight, eps, None, None, None, 0, 1, 1e4, 2, at, at, 6, 4, 4, 1,
                                         32, None)

    for eps in (-1.0, float("nan"), float("inf")):
        assert call(None, eps) == 0
    assert call(at, -1.0) == -1 and call(at, float("nan")) == -1 and call(at, 0.0) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
def test_eps_without_a_norm_may_be_anything(gpu, code):
    heads, kv, dim, rows = 4, 2, 64, 3
    qkv, _, _, positions = inputs(rows, heads, kv, dim, torch.bfloat16, gpu)
    results = []
    for eps in (1e-6, None, -1.0):
        pool = filled(2, 16, kv, dim, code, torch.bfloat16, gpu)
        q = norm_rotary_append(qkv, None, None, eps, positions, torch.arange(rows, device=gpu), pool, heads, 1e6)
        results.append((q, planes(pool)[0]))
    assert all(torch.equal(a, b) for other in results[1:] for a, b in zip(other, results[0]))


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm", [True, False])
def test_pools_at_odd_elements_in_full(gpu, norm, dtype, code):
    """Pools that start at an odd element, whose stores are narrow or single bytes: keys as the formula
    has them, values and their scales bit for bit, and every other row, scale and byte as it was."""
    heads, kv, rows, blocks, page = 4, 2, 9, 3, 16
    for dim in (32, 64, 96, 128):
        qkv, wq, wk, positions = inputs(rows, heads, kv, dim, dtype, gpu)
        if norm:
            (want_q, want_k), (size_q, size_k), want_v = formula(qkv, wq, wk, 1e-6, positions, heads, kv, dim, 1e6)
        else:
            wq = wk = None
            (want_q, want_k), (size_q, size_k), want_v = plain_formula(qkv, positions, heads, kv, dim, 1e6)
        values, value_scales = stored_exactly(want_v, code, dtype)
        to = some_rows(rows, blocks * page, gpu, skipped=2)
        written = ((to >= 0) & (to < blocks * page)).cpu()
        there = to.cpu()[written]
        for off in (1, 2, 3, 4, 8):
            fresh = filled(blocks, page, kv, dim, code, dtype, gpu)
            store = fresh if code is None else fresh.codes.view(torch.uint8)
            room = torch.full((off + store.numel() + 64,), 77, dtype=store.dtype, device=gpu)
            moved = room[off : off + store.numel()].view(store.shape)
            moved.copy_(store)
            pool = moved if code is None else QuantizedPool(moved.view(code), fresh.scales)
            stored, scales = planes(pool)
            q = norm_rotary_append(qkv, wq, wk, 1e-6, positions, to, pool, heads, 1e6)
            assert (room[:off] == 77).all() and (room[off + store.numel() :] == 77).all()
            check(q, want_q, size_q, dtype)
            got, got_scales = planes(pool)
            check_keys(got[0, there], None if scales is None else got_scales[0, there], want_k[written],
                       size_k[written], code, dtype)
            stored[1, there], stored[0, there] = values[written], got[0, there]
            assert alike(code, got, stored)
            if scales is not None:
                scales[1, there], scales[0, there] = value_scales[written], got_scales[0, there]
                assert torch.equal(got_scales, scales)
