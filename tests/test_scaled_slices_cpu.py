"""CPU test: the K slices of the 8-bit products' clusters cover the K blocks once."""
import os

from tests.test_block_scale_cpp_cpu import ROOT, build_and_run


def test_slices_cover_the_k_blocks_once():
    out = build_and_run("scaled_slices_test", "-I", os.path.join(ROOT, "composable_kernel_b200", "csrc"))
    assert "scaled slice checks passed" in out
