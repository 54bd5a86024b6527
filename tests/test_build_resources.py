"""Registers of kernels whose launches are planned for two workgroups a CU, as the build wrote them down."""

import re
from pathlib import Path

import pytest

USAGE = Path(__file__).resolve().parent.parent / "_build" / "resource_usage.txt"
# hs::pages_mfma_kernel<pool, query, 64 of the head dim, pages of 16 rows, launch, no window ..>
KERNEL = re.compile(r"pages_mfma_kernelILi([1-4])ELi([0-2])ELi64ELb1ELb([01])ELb0E")


@pytest.mark.skipif(not USAGE.exists(), reason="the library was not built in this tree")
def test_page_attention_keeps_two_workgroups_a_cu():
    """A workgroup of eight waves has two on a SIMD, which holds 512 registers a lane: at most 128 each
    leave room for a second workgroup.  16- and 8-bit pools of 64 of the head dim stand just below."""
    kernels = {}
    for line in USAGE.read_text().splitlines()[1:]:
        name, vgprs, agprs = line.split()[1:4]
        found = KERNEL.search(name)
        if found:
            kernels[found.groups()] = int(vgprs) + int(agprs)
    # plain pools with a query of their own, 8-bit ones with any; the long launch and the short one
    assert len(kernels) == 2 * (2 + 2 * 3), sorted(kernels)
    over = {key: registers for key, registers in kernels.items() if registers > 128}
    assert not over, over
