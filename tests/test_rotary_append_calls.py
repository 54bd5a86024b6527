"""Calls of norm_rotary_append at the edges of what it documents."""

import ctypes

import pytest
import torch

from mini_hisparse_amd import _lib
from mini_hisparse_amd.dense import norm_rotary_append

from test_norm_rotary import inputs
from test_rotary_append import CODES, filled, planes


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
