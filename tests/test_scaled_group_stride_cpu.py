"""CPU test: matrices of E that overlap are refused also where their size passes 64 bits."""
import pytest

import composable_kernel_b200 as ck
from composable_kernel_b200 import capi


def supported(M, N, lde, groups, stride):
    op = ck.DeviceGroupedGemmABScale(ck.CKB_GROUP_K_BLOCKS)
    arg = op.MakeArgument(0x1000, 0x2000, 0x3000, 0x4000, 0x5000, 0x6000, groups, M, N, 256, 256, 256, lde, (2, 1), (2, 1), 0, 0, stride)
    ok = op.IsSupportedArgument(arg)
    assert ok or "smaller than a matrix" in capi.last_error()
    return ok


@pytest.mark.parametrize("M,N,lde", [(5, 64, 1 << 62), (3, 64, 1 << 62), (3, 64, (1 << 62) + 1), (9, 8, 1 << 61)])
def test_sizes_beyond_64_bits(M, N, lde):
    for stride in (0, N, N + 1, (1 << 63) - 1):
        assert not supported(M, N, lde, 2, stride)
        assert supported(M, N, lde, 1, stride)  # a single group's stride is never used


def test_ordinary_sizes():
    for M, N, lde in ((1, 1, 1), (1, 64, 100), (64, 64, 64), (7, 60, 100)):
        need = (M - 1) * lde + N
        for stride in range(max(0, need - lde - 2), need + lde + 2):
            assert supported(M, N, lde, 3, stride) == (stride >= need), (M, N, lde, stride)
