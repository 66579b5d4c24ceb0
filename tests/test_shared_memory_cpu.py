"""Dynamic shared memory says the alignment that its readers rely on: the sort reads its ids 16 bytes at a time."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "cute-moe-train_b200" / "csrc"


@pytest.mark.parametrize("name", ["moe_permute.cu", "fp8_block_gemm.cu", "moe_gemm_sm100.cu"])
def test_dynamic_shared_memory_read_in_wide_words_is_aligned_for_them(name):
    lines = re.findall(r"extern __shared__[^;]*;", (CSRC / name).read_text())
    assert lines
    for line in lines:
        m = re.search(r"__align__\((\d+)\)", line)
        assert m and int(m.group(1)) >= 16, line
