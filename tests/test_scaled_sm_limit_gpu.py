"""GPU test of pinned K splits of the 8-bit products in a process that may use only part of the GPU (CKB_SM_LIMIT): what is
reported as supported runs, what is not is refused by the run too, and results do not change.  The limit is read once per
process, so the cases run in a child process."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = r'''
import os, sys
import torch
sys.path.insert(0, os.environ["CKB_REPO_ROOT"])
import composable_kernel_b200 as ck
from composable_kernel_b200 import capi

torch.cuda.set_device(0)
limit = int(os.environ["CKB_SM_LIMIT"])
M, N, K = 5, 256, 4096
g = torch.Generator(device="cuda").manual_seed(limit)
a = torch.randint(-3, 4, (M, K), generator=g, device="cuda").float()
b = torch.randint(-3, 4, (N, K), generator=g, device="cuda").float()
a8, b8 = a.to(torch.float8_e4m3fn), b.to(torch.float8_e4m3fn)
sa, sb = torch.ones((M, K // 128), device="cuda"), torch.ones((N // 128, K // 128), device="cuda")
want = (a.double() @ b.double().t()).float()
ran = []
for ks in (0, 1, 2, 4, 8):                     # 0: the library's own choice
    e = torch.full((M, N), -1.0, device="cuda")
    op = ck.DeviceGemmABScale(e_dtype=ck.CKB_F32, tile_config=capi.scaled_tile(16, 1, ks) if ks else 0)
    arg = op.MakeArgument(a8.data_ptr(), b8.data_ptr(), sa.data_ptr(), sb.data_ptr(), e.data_ptr(), M, N, K, K, K, N,
                          sa.stride(), sb.stride())
    supported = op.IsSupportedArgument(arg)
    try:
        op.MakeInvoker().Run(arg)
        assert supported, f"ksplit {ks} ran although it is not supported"
        torch.cuda.synchronize()
        assert ck.device_status() == 0
        assert torch.equal(e, want), (ks, capi.last_plan())   # whole numbers below 2^24: exact
        ran.append(ks)
    except capi.CkbError as err:
        assert not supported, f"ksplit {ks} is supported, but: {err}"
        assert "no tile fits" in str(err), err
# a cluster has to fit the part of the GPU that may be used
assert ran == [k for k in (0, 1, 2, 4, 8) if k <= limit], ran
print("scaled sm-limit case passed")
'''


@pytest.mark.parametrize("limit", [2, 4, 6, 8, 20])
def test_supported_and_run_agree(cuda_device, limit):
    env = dict(os.environ, CKB_SM_LIMIT=str(limit), CKB_REPO_ROOT=ROOT)
    res = subprocess.run([sys.executable, "-c", CHILD], env=env, capture_output=True, text=True, timeout=600, cwd=ROOT)
    assert res.returncode == 0, res.stdout[-2000:] + res.stderr[-3000:]
    assert "scaled sm-limit case passed" in res.stdout
