"""GPU tests: the profiler's sub-commands of the 8-bit products, the quantizer and layer norm verify every tile they time
against the CPU references (exit code 0 = within the bounds)."""
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def profiler(cuda_device):
    res = subprocess.run(["make", "-C", os.path.join(ROOT, "examples"), "bin/ck_profiler"], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-3000:]

    def run(*args):
        res = subprocess.run([os.path.join(ROOT, "examples", "bin", "ck_profiler"), *map(str, args)], capture_output=True,
                             text=True, timeout=300)
        assert res.returncode == 0, f"{args}: {res.stdout[-2000:]}{res.stderr[-2000:]}"
        return res.stdout
    return run


# type of the result, form, verify, initialisation, log, time, sizes
@pytest.mark.parametrize("args", [(2, 1, 1, 2, 0, 1, 300, 520, 700), (1, 0, 1, 1, 0, 0, 130, 300, 256), (3, 2, 1, 2, 0, 0, 300, 520, 700),
                                  (2, 1, 1, 2, 0, 0, 1, 1, 2050)])
def test_gemm_ab_scale(profiler, args):
    assert "Best Perf for gemm_ab_scale" in profiler("gemm_ab_scale", *args)


@pytest.mark.parametrize("args", [(2, 1, 1, 2, 0, 1, "100,0,37,1", 256, 300), (1, 0, 1, 2, 0, 0, "100,0,37,1", 264, 300),
                                  (3, 2, 1, 2, 0, 0, "100,0,370,1", 136, 200)])
def test_grouped_gemm_ab_scale(profiler, args):
    assert "Best Perf for grouped_gemm_ab_scale" in profiler("grouped_gemm_ab_scale", *args)


@pytest.mark.parametrize("dtype", [1, 2, 3])
def test_rows_operations(profiler, dtype):
    for block in (1, 2, 3):
        profiler("block_quantize", dtype, block, 1, 2, 0, 1, 333, 517)
    for out in (1, 2, 3):
        profiler("layernorm_fwd", dtype, out, 1, 2, 0, 1, 77, 1037)
    profiler("layernorm_bwd", dtype, 1, 2, 0, 1, 77, 1037)
