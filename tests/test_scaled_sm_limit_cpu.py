"""CPU test: pinned K splits of the 8-bit products are supported only where their cluster fits the part of the GPU that
CKB_SM_LIMIT leaves (what the run refuses on such a part)."""
import pytest

import composable_kernel_b200 as ck
from composable_kernel_b200 import capi


@pytest.mark.parametrize("limit", [None, 2, 4, 6, 8, 20])
def test_clusters_that_fit(monkeypatch, limit):
    if limit is None:
        monkeypatch.delenv("CKB_SM_LIMIT", raising=False)
    else:
        monkeypatch.setenv("CKB_SM_LIMIT", str(limit))
    for ksplit in (0, 1, 2, 4, 8):
        op = ck.DeviceGemmABScale(tile_config=capi.scaled_tile(16, 1, ksplit) if ksplit else 0)
        arg = op.MakeArgument(0x1000, 0x2000, 0x3000, 0x4000, 0x5000, 5, 256, 4096, 4096, 4096, 256, (32, 1), (32, 1))
        assert op.IsSupportedArgument(arg) == (limit is None or ksplit <= limit), (ksplit, capi.last_error())
