"""CPU tests of the C++ side of the 8-bit products, the block quantizer and layer norm: their class templates and CPU
references compile with g++ and answer as documented, and the products' work decomposition covers every element once."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIBDIR = os.path.join(ROOT, "composable_kernel_b200", "lib")


def build_and_run(name, *flags):
    out_dir = os.path.join(ROOT, "tests", "cpp", "bin")
    os.makedirs(out_dir, exist_ok=True)
    exe = os.path.join(out_dir, name)
    res = subprocess.run(["g++", "-std=c++17", "-O2", os.path.join(ROOT, "tests", "cpp", name + ".cpp"), "-o", exe, *flags],
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-3000:]
    run = subprocess.run([exe], capture_output=True, text=True, timeout=600)
    assert run.returncode == 0, run.stdout[-3000:]
    return run.stdout


def test_class_templates_and_references():
    from composable_kernel_b200 import capi
    capi.lib()  # the shared library must exist: the C++ layer links against it
    out = build_and_run("block_scale_api_test", "-fexcess-precision=16", "-ffp-contract=off", "-pthread", "-I",
                        os.path.join(ROOT, "include"), "-L", LIBDIR, "-lckb200", f"-Wl,-rpath,{LIBDIR}")
    assert "all block scale API checks passed" in out


def test_scaled_plan_covers_every_element_once():
    out = build_and_run("scaled_plan_test", "-I", os.path.join(ROOT, "composable_kernel_b200", "csrc"))
    assert "scaled plan checks passed" in out
