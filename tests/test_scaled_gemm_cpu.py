"""CPU tests of what the 8-bit products, the block quantizer and layer norm refuse."""
import pytest

import composable_kernel_b200 as ck
from composable_kernel_b200 import capi

ROW, COL = ck.CKB_ROW_MAJOR, ck.CKB_COL_MAJOR


def gemm(M=64, N=64, K=256, sa=None, sb=None, se=None, tile=0, p=(0x1000, 0x2000, 0x3000, 0x4000, 0x5000), strides=((2, 1), (2, 1)), **kw):
    op = ck.DeviceGemmABScale(tile_config=tile, **kw)
    arg = op.MakeArgument(*p, M, N, K, sa or K, sb or K, se or N, *strides)
    return op, arg


def refused(op, arg, text):
    assert not op.IsSupportedArgument(arg)
    assert text in capi.last_error()
    if text == "no tile fits":  # (a run asks the device first)
        return
    with pytest.raises(capi.CkbError, match="invalid setting|groups"):
        op.MakeInvoker().Run(arg)


def test_scaled_gemm_rules():
    op, arg = gemm()
    assert op.IsSupportedArgument(arg), capi.last_error()
    for kw in (dict(M=1, N=1, K=1, sa=16, sb=16), dict(M=3, N=5, K=7, sa=16, sb=32), dict(strides=((0, 0), (0, 0))),
               dict(a_layout=COL, b_layout=ROW), dict(a_dtype=ck.CKB_F8_E5M2, e_dtype=ck.CKB_F32)):
        op, arg = gemm(**kw)
        assert op.IsSupportedArgument(arg), capi.last_error()
    refused(*gemm(M=0), "positive")
    refused(*gemm(K=0, sa=16, sb=16), "positive")
    refused(*gemm(M=1 << 31), "2^31")
    refused(*gemm(K=100, sa=100, sb=112), "multiples of 16")
    refused(*gemm(sa=240), "leading dimension")
    refused(*gemm(se=63), "leading dimension")
    refused(*gemm(a_dtype=ck.CKB_BF16), "CKB_F8")
    refused(*gemm(b_dtype=ck.CKB_I8), "CKB_F8")
    refused(*gemm(e_dtype=ck.CKB_F8_E4M3), "CKB_BF16")
    refused(*gemm(scale_block_m=64), "1 or 128")
    refused(*gemm(scale_block_n=0), "1 or 128")
    refused(*gemm(a_layout=2), "layout")
    refused(*gemm(strides=((-1, 1), (1, 1))), "negative")


def test_scaled_gemm_pinned_tiles():
    for tile in (capi.scaled_tile(16, 1), capi.scaled_tile(128, 1, 1), capi.scaled_tile(128, 2), capi.scaled_tile(224, 2)):
        op, arg = gemm(tile=tile)
        assert op.IsSupportedArgument(arg), capi.last_error()
    refused(*gemm(tile=capi.scaled_tile(48, 1)), "no tile fits")
    refused(*gemm(tile=capi.scaled_tile(240, 2)), "no tile fits")
    refused(*gemm(tile=capi.scaled_tile(16, 1), a_layout=COL, sa=64), "no tile fits")     # an M-contiguous A needs 128 columns
    refused(*gemm(tile=capi.scaled_tile(16, 1, 2)), "no tile fits")                   # two K blocks per slice at least
    refused(*gemm(tile=capi.scaled_tile(256, 2) | 1 << 16), "CKB_SCALED_TILE")
    refused(*gemm(tile=capi.scaled_tile(256, 2, 2)), "no tile fits")
    refused(*gemm(tile=capi.scaled_tile(16, 3)), "CKB_SCALED_TILE")
    refused(*gemm(tile=16), "CKB_SCALED_TILE")
    refused(*gemm(tile=-1), "CKB_SCALED_TILE")
    refused(*gemm(tile=capi.scaled_tile(16, 1, 3)), "CKB_SCALED_TILE")


def test_scaled_gemm_pointers_are_checked_before_a_launch():
    for p in ((0, 0x2000, 0x3000, 0x4000, 0x5000), (0x1000, 0x2000, 0x3000, 0, 0x5000), (0x1008, 0x2000, 0x3000, 0x4000, 0x5000),
              (0x1000, 0x2000, 0x3002, 0x4000, 0x5000), (0x1000, 0x2000, 0x3000, 0x4000, 0x5001)):
        op, arg = gemm(p=p)
        with pytest.raises(capi.CkbError, match="null|16-byte|aligned"):
            op.MakeInvoker().Run(arg)


def grouped(axis, groups=4, M=64, N=64, K=256, strides=(64 * 256, 2, 64 * 64), p_offsets=0x6000, **kw):
    op = ck.DeviceGroupedGemmABScale(axis, **kw)
    arg = op.MakeArgument(0x1000, 0x2000, 0x3000, 0x4000, 0x5000, p_offsets, groups, M, N, K, K, K, N, (2, 1), (2, 1), *strides)
    return op, arg


def test_grouped_rules():
    for axis in (ck.CKB_GROUP_ROWS, ck.CKB_GROUP_K_BLOCKS):
        op, arg = grouped(axis)
        assert op.IsSupportedArgument(arg), capi.last_error()
        refused(*grouped(axis, groups=0), "groups")
        refused(*grouped(axis, groups=capi.CKB_SCALED_MAX_GROUPS + 1), "groups")
        op, arg = grouped(axis, p_offsets=0)
        with pytest.raises(capi.CkbError, match="null"):
            op.MakeInvoker().Run(arg)
    refused(*grouped(2), "axis")
    refused(*grouped(ck.CKB_GROUP_ROWS, a_layout=COL), "row-major A")
    refused(*grouped(ck.CKB_GROUP_ROWS, scale_block_m=128), "scale per row")
    refused(*grouped(ck.CKB_GROUP_ROWS, strides=(8, 2, 0)), "multiple of 16")
    refused(*grouped(ck.CKB_GROUP_K_BLOCKS, strides=(0, 0, 64 * 64 - 1)), "smaller than a matrix")


def quant(M=100, N=300, ldx=None, ldq=None, strides=(3, 1), p=(0x1000, 0x2000, 0x3000), **kw):
    op = ck.DeviceBlockQuantize(**kw)
    return op, op.MakeArgument(*p, M, N, ldx or N, ldq or N, strides)


def test_block_quantize_rules():
    for kw in (dict(), dict(block_m=128), dict(block_m=128, block_n=1, strides=(300, 1)), dict(x_dtype=ck.CKB_F32, q_dtype=ck.CKB_F8_E5M2, pow2_scale=True)):
        op, arg = quant(**kw)
        assert op.IsSupportedArgument(arg), capi.last_error()
    refused(*quant(block_m=64), "blocks are")
    refused(*quant(block_n=1), "blocks are")
    refused(*quant(x_dtype=ck.CKB_I8), "CKB_BF16")
    refused(*quant(q_dtype=ck.CKB_BF16), "CKB_F8")
    refused(*quant(M=0), "positive")
    refused(*quant(ldx=299), "pitches")
    refused(*quant(strides=(0, 1)), "scale of its own")
    refused(*quant(strides=(3, 0)), "scale of its own")
    refused(*quant(strides=(3, -1)), "negative")
    refused(*quant(pow2_scale=2), "pow2_scale")
    for p in ((0, 1, 4), (0x1000, 0, 4), (0x1001, 0x2000, 0x3000), (0x1000, 0x2000, 0x3002)):
        op, arg = quant(p=p)
        with pytest.raises(capi.CkbError, match="null|aligned"):
            op.MakeInvoker().Run(arg)


def ln(M=10, N=300, ldx=None, ldy=None, eps=1e-5, y=0x4000, q=None, scale=None, ldq=0, strides=(0, 0), x=0x1000, **kw):
    op = ck.DeviceLayernormFwd(**kw)
    return op, op.MakeArgument(x, 0x2000, 0x3000, y, 0x5000, 0x6000, M, N, ldx or N, ldy or N, eps, q, scale, ldq, strides)


def test_layernorm_forward_rules():
    for kw in (dict(), dict(y=None, q=0x7000, scale=0x8000, ldq=300, strides=(3, 1)), dict(w_dtype=ck.CKB_BF16), dict(eps=0.0)):
        op, arg = ln(**kw)
        assert op.IsSupportedArgument(arg), capi.last_error()
    refused(*ln(x_dtype=ck.CKB_F8_E4M3), "CKB_BF16")
    refused(*ln(w_dtype=ck.CKB_F16), "weights of that type")
    refused(*ln(eps=-1.0), "eps")
    refused(*ln(eps=float("nan")), "eps")
    refused(*ln(eps=float("inf")), "eps")
    refused(*ln(M=0), "positive")
    refused(*ln(ldx=299), "pitch")
    refused(*ln(ldy=299), "pitch")
    refused(*ln(q=0x7000, ldq=300), "scales")
    refused(*ln(q=0x7000, scale=0x8000, ldq=299, strides=(3, 1)), "pitch")
    refused(*ln(q=0x7000, scale=0x8000, ldq=300, strides=(0, 1)), "scale of its own")
    refused(*ln(q=0x7000, scale=0x8000, ldq=300, strides=(3, 1), q_dtype=ck.CKB_BF16), "CKB_F8")
    op, arg = ln(y=None)
    with pytest.raises(capi.CkbError, match="at least one output"):
        op.MakeInvoker().Run(arg)
    op, arg = ln(x=0x1001)
    with pytest.raises(capi.CkbError, match="aligned"):
        op.MakeInvoker().Run(arg)


def ln_bwd(M=10, N=300, ld=None, dx=0x6000, dg=0x7000, db=0x8000, **kw):
    op = ck.DeviceLayernormBwd(**kw)
    return op, op.MakeArgument(0x1000, 0x2000, 0x3000, 0x4000, 0x5000, dx, dg, db, M, N, ld or N, N, N)


def test_layernorm_backward_rules():
    op, arg = ln_bwd()
    assert op.IsSupportedArgument(arg) and op.GetWorkSpaceSize(arg) > 0
    with pytest.raises(capi.CkbError) as err:  # no workspace
        op.MakeInvoker().Run(arg)
    assert err.value.code == capi.CKB_ERR_WORKSPACE
    op.SetWorkSpacePointer(arg, 0x9000, op.GetWorkSpaceSize(arg) - 1)
    with pytest.raises(capi.CkbError) as err:
        op.MakeInvoker().Run(arg)
    assert err.value.code == capi.CKB_ERR_WORKSPACE
    op, arg = ln_bwd(dg=None, db=None)
    assert op.GetWorkSpaceSize(arg) == 0
    refused(*ln_bwd(ld=299), "pitch")
    refused(*ln_bwd(x_dtype=ck.CKB_I8), "CKB_BF16")
    op, arg = ln_bwd(dx=None, dg=None, db=None)
    with pytest.raises(capi.CkbError, match="at least one output"):
        op.MakeInvoker().Run(arg)


def test_null_descriptors_are_refused():
    for name in ("scaled_gemm", "scaled_grouped_gemm", "block_quantize", "layernorm_fwd", "layernorm_bwd"):
        assert getattr(capi.lib(), f"ckb_{name}_supported")(None) == capi.CKB_ERR_INVALID
        args = (None, None, 0, None, 0, None) if name == "layernorm_bwd" else (None, None, 0, None)
        assert getattr(capi.lib(), f"ckb_{name}_run")(*args) == capi.CKB_ERR_INVALID


def test_struct_layouts_match_the_header(tmp_path):
    import ctypes
    import os
    import subprocess
    names = {"scaled_gemm": (capi.ScaledGemmDesc, "p_a"), "scaled_grouped_gemm": (capi.ScaledGroupedGemmDesc, "e_group_stride"),
             "block_quantize": (capi.BlockQuantizeDesc, "p_scale"), "layernorm_fwd": (capi.LayernormFwdDesc, "p_rstd"),
             "layernorm_bwd": (capi.LayernormBwdDesc, "p_dbeta")}
    body = "".join(f'printf("%zu %zu\\n", sizeof(ckb_{n}_desc), offsetof(ckb_{n}_desc, {f}));' for n, (_, f) in names.items())
    src = tmp_path / "t.c"
    src.write_text('#include "ckb200.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(){' + body + "return 0;}")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "t")], check=True)
    got = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.split("\n")
    for line, (cls, field) in zip(got, names.values()):
        assert line == f"{ctypes.sizeof(cls)} {getattr(cls, field).offset}"
