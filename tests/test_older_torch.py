"""A torch without the 4-bit dtypes: everything else works, and 4-bit pools are refused."""

import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent

PROGRAM = """
import torch

del torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
from mini_hisparse_amd import _lib
from mini_hisparse_amd.dense import quantize_weight, QuantizedWeight
from mini_hisparse_amd.quantized import QuantizedPool

codes = [_lib.dtype_code(t) for t in (torch.float32, torch.float16, torch.bfloat16)]
assert codes == [_lib.HS_DTYPE_F32, _lib.HS_DTYPE_F16, _lib.HS_DTYPE_BF16]
for dtype, code in ((torch.int8, _lib.HS_DTYPE_I8), (torch.float8_e4m3fn, _lib.HS_DTYPE_E4M3)):
    pool = QuantizedPool.empty(2, 16, 2, 64, dtype, device="cpu")
    assert pool.code == code and pool.row_bytes == 2 * 2 * 68
weight = quantize_weight(torch.eye(32))  # codes and scales are bytes: no 4-bit dtype is needed
assert (weight.n, weight.k) == (32, 32)
for refused in (lambda: QuantizedPool(torch.zeros(2, 2, 16, 2, 32, dtype=torch.uint8), torch.zeros(2, 2, 16, 2, 2)),
                lambda: _lib.cache_code(torch.uint8), lambda: _lib.dtype_code(torch.int8)):
    try:
        refused()
    except ValueError:
        continue
    raise SystemExit("not refused")
print("done")
"""


def test_other_dtypes_do_not_need_the_4_bit_ones():
    ran = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert ran.returncode == 0 and ran.stdout.strip() == "done", ran.stderr
