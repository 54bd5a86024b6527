"""What the build wrote down of its kernels: registers where a launch is planned for two workgroups a CU,
and forms that no call reaches."""

import re
from pathlib import Path

import pytest

USAGE = Path(__file__).resolve().parent.parent / "_build" / "resource_usage.txt"
# hs::pages_mfma_kernel<pool, query, 64 of the head dim, pages of 16 rows, launch, no window ..>
KERNEL = re.compile(r"pages_mfma_kernelILi([1-4])ELi([0-2])ELi64ELb1ELb([01])ELb0E")


built = pytest.mark.skipif(not USAGE.exists(), reason="the library was not built in this tree")


def rows():
    return [line.split() for line in USAGE.read_text().splitlines()[1:]]


@built
def test_page_attention_keeps_two_workgroups_a_cu():
    """A workgroup of eight waves has two on a SIMD, which holds 512 registers a lane: at most 128 each
    leave room for a second workgroup.  16- and 8-bit pools of 64 of the head dim stand just below."""
    kernels = {}
    for _, name, vgprs, agprs, *_ in rows():
        found = KERNEL.search(name)
        if found:
            kernels[found.groups()] = int(vgprs) + int(agprs)
    # plain pools with a query of their own, 8-bit ones with any; the long launch and the short one
    assert len(kernels) == 2 * (2 + 2 * 3), sorted(kernels)
    over = {key: registers for key, registers in kernels.items() if registers > 128}
    assert not over, over


@built
def test_projections_in_4_bits_have_the_forms_that_calls_reach():
    """A form for each of two types: one, two and four tiles in eight waves, with and without streaming
    loads, and for more than 1024 row tiles, above 4 MB at any K, four tiles in four waves and the
    walk with streaming ones."""
    names = sorted(name for _, name, *_ in rows() if "fp4_gemm" in name)
    assert len(names) == len(set(names)) == 2 * (3 * 2 + 2), names
    for name in names:
        if "walk" in name or "ELi4ELi4E" in name:
            assert "Lb0E" not in name, name
