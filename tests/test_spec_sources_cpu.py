"""A rule of the attention kernels over drafted trees and 8-bit caches that no result
shows: they start while the kernel ahead still writes (its rows, scales and queries), so
nothing is read through the read-only data path."""

from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "litevllm_b200" / "csrc"


@pytest.mark.parametrize("name", ["paged_tree.cuh", "paged_tree_tc.cuh"])
def test_no_read_only_loads_beside_the_kernel_ahead(name):
    text = (CSRC / name).read_text()
    assert text.count("pdl_wait();") == 1
    for form in ("__ldg(", "ld.global.nc", "__ldcg(", "__restrict__"):
        assert form not in text, f"{name}: {form}"
