"""CPU tests: strides that put the scales of two blocks in one place are refused, all others are taken."""
import itertools

import composable_kernel_b200 as ck
from composable_kernel_b200 import capi


def collide(sm, sn, m, n):
    places = [i * sm + j * sn for i in range(m) for j in range(n)]
    return len(set(places)) < len(places)


def check(op, arg, sm, sn, m, n):
    bad = collide(sm, sn, m, n)
    assert op.IsSupportedArgument(arg) != bad, (sm, sn, m, n)
    if bad:
        assert "scale of its own" in capi.last_error()


def test_quantizer():
    for block in ((1, 128), (128, 1), (128, 128)):
        op = ck.DeviceBlockQuantize(ck.CKB_BF16, ck.CKB_F8_E4M3, *block)
        for m, n, sm, sn in itertools.product(range(1, 5), range(1, 5), range(0, 7), range(0, 7)):
            M, N = (m - 1) * block[0] + 1, (n - 1) * block[1] + 1
            arg = op.MakeArgument(0x1000, 0x2000, 0x3000, M, N, N, N, (sm, sn))
            check(op, arg, sm, sn, m, n)


def test_layernorm():
    op = ck.DeviceLayernormFwd()
    for m, n, sm, sn in itertools.product(range(1, 5), range(1, 5), range(0, 7), range(0, 7)):
        N = (n - 1) * 128 + 7
        arg = op.MakeArgument(0x1000, 0x2000, 0x3000, None, None, None, m, N, N, N, 1e-5, 0x4000, 0x5000, N, (sm, sn))
        check(op, arg, sm, sn, m, n)


def test_large_strides():
    op = ck.DeviceBlockQuantize()
    for strides, ok in (((1 << 62, 1), True), ((1, 1 << 62), True), ((1 << 62, 1 << 62), False), ((3, 1), True), ((1, 1000), True),
                        ((1, 999), False), ((2, 1), False)):
        arg = op.MakeArgument(0x1000, 0x2000, 0x3000, 1000, 300, 300, 300, strides)
        assert op.IsSupportedArgument(arg) == ok, strides
