"""Checks on the generated gfx950 code of the paged kernels (host-side compile, no GPU needed).

They write M0 inside their direct-to-LDS inline assembly, so nothing else may
use it; and only the wide tiles' second pass over values that are not finite,
which no ordinary call takes, may keep registers in scratch.
"""

from __future__ import annotations

import re

import pytest

from test_build_isa import _asm


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    path = tmp_path_factory.mktemp("isa")
    return {src: _asm(src, path).splitlines() for src in ("paged_attn.hip", "paged_tables.hip")}


def test_m0_only_inside_inline_asm(asm):
    inside = False
    for line in asm["paged_attn.hip"]:
        s = line.strip()
        if s.startswith(";;#ASMSTART"):
            inside = True
        elif s.startswith(";;#ASMEND"):
            inside = False
        elif not inside and not s.startswith(";") and re.search(r"\bm0\b", s):
            pytest.fail(f"compiler-generated M0 use outside the DMA asm: {s}")


@pytest.mark.parametrize("src", ["paged_attn.hip", "paged_tables.hip"])
def test_no_scratch_in_the_loops(src, asm):
    """No spills but in wide tiles of 128 dimensions, and there none in a block with the tile step's 32 MFMAs."""
    kernel, block, mfmas, scratch = "", "", 0, 0
    for line in asm[src] + [".LBB_end:"]:
        head = re.match(r"(_ZN\S+|\.LBB\S+):", line)
        if head:
            if scratch:
                assert re.search(r"paged_wide_kernelILi\dELi128|paged_prefix_kernelILi\dELi128ELb1", kernel), kernel
                assert mfmas != 32, f"{kernel} {block}: {scratch} scratch accesses in the tile step"
            if head.group(1).startswith("_ZN"):
                kernel = head.group(1)
            block, mfmas, scratch = head.group(1), 0, 0
        mfmas += "v_mfma" in line
        scratch += "scratch_store" in line or "scratch_load" in line
