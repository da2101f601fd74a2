"""The order of the kernels' launches, as far as it shows in the sources: no GPU is needed."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "kv_skill_v2_b200" / "csrc"


def kernels(path):
    """The text of every kernel of a file that waits for the launch before it."""
    for text in re.split(r"(?=__global__)", path.read_text())[1:]:
        if "pdl_wait()" in text:
            yield re.search(r"\b\w+_kernel\b", text).group(), text


@pytest.mark.parametrize("name", ["gemm_f8.cuh", "gemm_f16x3.cuh", "mass.cuh", "read_shared.cuh"])
def test_operands_are_loaded_behind_the_wait(name):
    """A launch may begin while the one before it runs; what that one wrote is there behind the wait only."""
    seen = 0
    for kernel, text in kernels(CSRC / name):
        loads = text.find("tma_load")
        assert loads < 0 or loads > text.rfind("pdl_wait()"), kernel
        seen += loads >= 0
    assert seen
