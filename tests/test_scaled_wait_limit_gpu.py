"""GPU test of the give-up path of the 8-bit products: bounded waits that run out while copies and MMAs are on their way.

A test hook (CKB_TEST_SCALED_WAIT_EXTRA) makes barriers of the kernel wait for one arrival more than will ever come, under a
limit of a few milliseconds (CKB_WAIT_LIMIT_MS): those of the scales, or those that say that a K block was multiplied; in all
CTAs, or only in the first or second one of a pair, so that the two producers stop at different stages.  Every copy and MMA
that was issued completes normally.  The kernel has to return with a status, without waiting for arrivals that nobody
will send (the limit of its exit path is two seconds), and the next launch has to be right.  Nothing faults, traps or spins
without a limit.  The cases run in a child process because the limit is read once per process."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = r'''
import ctypes, os, sys, time
import torch
sys.path.insert(0, os.environ["CKB_REPO_ROOT"])
import composable_kernel_b200 as ck
from composable_kernel_b200 import capi

torch.cuda.set_device(0)
WAIT_EMPTY_FULL = (1, 2, 3, 4)                 # the codes of the K loop's waits; 5 is the exit path's
ROW, COL = capi.CKB_ROW_MAJOR, capi.CKB_COL_MAJOR

def status():
    w = ctypes.c_uint32(0)
    rc = capi.lib().ckb_device_status(ctypes.byref(w))
    return rc, w.value

def whole(g, *shape):                          # whole numbers: sums are exact
    return torch.randint(-3, 4, shape, generator=g, device="cuda").float()

def case(kind, cols, cg, ks, M, N, K):
    g = torch.Generator(device="cuda").manual_seed(cols + cg)
    a, b = whole(g, M, K), whole(g, N, K)
    wg = kind in ("wgrad", "k_groups")
    a8 = (a.t() if wg else a).contiguous().to(torch.float8_e4m3fn)
    b8 = (b.t() if wg else b).contiguous().to(torch.float8_e4m3fn)
    kb = -(-K // 128)
    sa, sb = torch.ones((M, kb), device="cuda"), torch.ones((N if wg else -(-N // 128), kb), device="cuda")
    tile = capi.scaled_tile(cols, cg, ks)
    args = (ck.CKB_F8_E4M3, ck.CKB_F8_E4M3, ck.CKB_F32, COL if wg else ROW, ROW if wg else COL, 1, 1 if wg else 128, tile)
    lda, ldb = a8.stride(0), b8.stride(0)
    want = a.double() @ b.double().t()
    ptr = (a8.data_ptr(), b8.data_ptr(), sa.data_ptr(), sb.data_ptr())
    keep = [a8, b8, sa, sb]
    if kind == "rows":
        off = torch.tensor([0, M // 3, M // 3, M], dtype=torch.int32, device="cuda")
        e = torch.zeros((M, N), device="cuda")
        op = ck.DeviceGroupedGemmABScale(ck.CKB_GROUP_ROWS, *args)
        arg = op.MakeArgument(*ptr, e.data_ptr(), off.data_ptr(), 3, M, N, K, lda, ldb, N, sa.stride(), sb.stride())
        keep.append(off)
    elif kind == "k_groups":
        off = torch.tensor([0, kb // 2, kb], dtype=torch.int32, device="cuda")
        e = torch.zeros((2, M, N), device="cuda")
        op = ck.DeviceGroupedGemmABScale(ck.CKB_GROUP_K_BLOCKS, *args)
        arg = op.MakeArgument(*ptr, e.data_ptr(), off.data_ptr(), 2, M, N, K, lda, ldb, N, sa.stride(), sb.stride(), GroupStrideE=M * N)
        cut = kb // 2 * 128
        want = torch.stack([a[:, :cut].double() @ b[:, :cut].double().t(), a[:, cut:].double() @ b[:, cut:].double().t()])
        keep.append(off)
    else:
        e = torch.zeros((M, N), device="cuda")
        op = ck.DeviceGemmABScale(*args)
        arg = op.MakeArgument(*ptr, e.data_ptr(), M, N, K, lda, ldb, N, sa.stride(), sb.stride())
    assert op.IsSupportedArgument(arg), capi.last_error()
    def right():
        e.zero_()
        op.MakeInvoker().Run(arg)
        assert status() == (capi.CKB_OK, 0), (kind, cols, cg, ks)
        assert torch.equal(e.double(), want), (kind, cols, cg, ks, capi.last_plan())
    right()
    for hook in (1, 2, 1 | 4, 1 | 8, 2 | 4, 2 | 8):
        if hook > 3 and cg == 1 and ks == 1:
            continue                           # every CTA stands alone: nothing new
        os.environ["CKB_TEST_SCALED_WAIT_EXTRA"] = str(hook)
        t0 = time.monotonic()
        op.MakeInvoker().Run(arg)
        rc, w = status()
        took = time.monotonic() - t0
        del os.environ["CKB_TEST_SCALED_WAIT_EXTRA"]
        print(kind, cols, cg, ks, "hook", hook, "status", hex(w), f"{took * 1e3:.1f} ms", flush=True)
        assert rc == capi.CKB_ERR_DEVICE and w >> 24 in WAIT_EMPTY_FULL, (kind, cols, cg, ks, hook, rc, hex(w))
        assert took < 1.0, (kind, cols, cg, ks, hook, took)
        right()

case("forward", 16, 1, 1, 5, 256, 4096)
case("forward", 128, 1, 1, 200, 256, 4096)
case("forward", 32, 1, 2, 30, 256, 4096)
case("forward", 128, 1, 8, 100, 256, 8192)
case("forward", 256, 2, 0, 600, 700, 4096)
case("forward", 128, 2, 0, 300, 260, 4096)
case("forward", 256, 2, 0, 300, 260, 304)       # fewer K blocks than stages
case("wgrad", 192, 2, 0, 304, 400, 4000)
case("rows", 64, 1, 0, 200, 256, 4096)
case("rows", 224, 2, 0, 700, 512, 4096)
case("k_groups", 256, 2, 0, 256, 512, 5120)
print("scaled wait-limit cases passed")
'''


def test_waits_that_run_out_are_reported_and_the_context_stays_usable(cuda_device):
    env = dict(os.environ, CKB_WAIT_LIMIT_MS="5", CKB_REPO_ROOT=ROOT)
    env.pop("CKB_TEST_SCALED_WAIT_EXTRA", None)
    res = subprocess.run([sys.executable, "-c", CHILD], env=env, capture_output=True, text=True, timeout=300, cwd=ROOT)
    print(res.stdout)
    assert res.returncode == 0, res.stdout[-4000:] + res.stderr[-3000:]
    assert "scaled wait-limit cases passed" in res.stdout
