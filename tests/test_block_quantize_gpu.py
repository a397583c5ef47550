"""GPU tests of the block quantizer against its formula in 64 bits."""
import pytest
import torch

import composable_kernel_b200 as ck
from composable_kernel_b200 import capi
from tests import llm_helpers as L

pytestmark = pytest.mark.gpu

BLOCKS = [(1, 128), (128, 1), (128, 128)]
X = [ck.CKB_BF16, ck.CKB_F16, ck.CKB_F32]
Q = [ck.CKB_F8_E4M3, ck.CKB_F8_E5M2]


def quantize(x, block, qt, pow2=False, ldq=None, q_offset=0, s_pad=0, s_t=False):
    """x: [M, >= N] view of a matrix; returns (q, scale) and checks that nothing around them was written."""
    M, N = x.shape
    xt = {v: k for k, v in L.WIDE.items()}[x.dtype]
    ldq = ldq or N
    raw = torch.full((M * ldq + q_offset + 32,), 0xAA, dtype=torch.uint8, device="cuda")
    q = raw[q_offset:q_offset + M * ldq].view(M, ldq)
    bm, bn = -(-M // block[0]), -(-N // block[1])
    sc = torch.full((bn, bm + s_pad) if s_t else (bm, bn + s_pad), -1.0, device="cuda")
    view = sc.t() if s_t else sc
    op = ck.DeviceBlockQuantize(xt, qt, *block, pow2)
    arg = op.MakeArgument(x.data_ptr(), q.data_ptr(), sc.data_ptr(), M, N, x.stride(0), ldq, view.stride())
    assert op.IsSupportedArgument(arg), capi.last_error()
    L.run(op, arg)
    assert (q[:, N:] == 0xAA).all() and (raw[:q_offset] == 0xAA).all() and (raw[q_offset + M * ldq:] == 0xAA).all()
    if s_pad:
        assert (sc[:, sc.shape[1] - s_pad:] == -1.0).all()
    return q[:, :N].contiguous().view(L.F8[qt]), view[:bm, :bn]


def check(x, block, qt, pow2=False, **kw):
    q, scale = quantize(x, block, qt, pow2, **kw)
    want, want_scale = L.quantize64(x, *block, qt, pow2)
    # the scale is one correctly rounded 32-bit division: the same bits
    assert torch.equal(scale, want_scale)
    # x / scale, rounded to 32 bits and then to 8: the rounding of the 32-bit quotient.  It is within half a step of the
    # 64-bit one, and two roundings differ from one only where the quotient is within 2^-24 of a tie.
    once = (want.float().clamp(-L.QMAX[qt], L.QMAX[qt])).to(L.F8[qt])
    assert torch.equal(q.float().nan_to_num(nan=12345.0), once.float().nan_to_num(nan=12345.0))


@pytest.mark.parametrize("block", BLOCKS)
@pytest.mark.parametrize("xt", X)
@pytest.mark.parametrize("qt", Q)
@pytest.mark.parametrize("M,N", [(1, 1), (1, 128), (3, 130), (128, 128), (129, 257), (300, 1000), (1000, 24)])
def test_sizes_and_types(cuda_device, block, xt, qt, M, N):
    g = L.gen(M * 1000 + N)
    x = (torch.randn((M, N), generator=g, device="cuda") * torch.exp(2 * torch.randn((N,), generator=g, device="cuda"))).to(L.WIDE[xt])
    check(x, block, qt)


@pytest.mark.parametrize("block", BLOCKS)
@pytest.mark.parametrize("qt", Q)
def test_power_of_two_scales(cuda_device, block, qt):
    x = torch.randn((300, 400), generator=L.gen(1), device="cuda").to(torch.bfloat16)
    x[0, 0] = 448.0  # a scale that is a power of two already
    check(x, block, qt, pow2=True)
    _, scale = quantize(x, block, qt, True)
    assert torch.equal(torch.exp2(torch.round(torch.log2(scale.double()))).float(), scale)


@pytest.mark.parametrize("block", BLOCKS)
@pytest.mark.parametrize("xt", X)
def test_strides_and_alignment(cuda_device, block, xt):
    base = torch.randn((140 * 500,), generator=L.gen(2), device="cuda").to(L.WIDE[xt])
    for N, ldx, start, ldq, off in ((300, 500, 0, 304, 0), (300, 451, 0, 300, 1), (300, 456, 3, 333, 8), (256, 256, 8, 256, 4)):
        x = base[start:start + 130 * ldx].view(130, ldx)[:, :N]
        check(x, block, ck.CKB_F8_E4M3, ldq=ldq, q_offset=off, s_pad=3)
        check(x, block, ck.CKB_F8_E4M3, ldq=ldq, q_offset=off, s_pad=2, s_t=True)


@pytest.mark.parametrize("block", BLOCKS)
@pytest.mark.parametrize("qt", Q)
def test_zeros_tiny_and_huge_values(cuda_device, block, qt):
    """Blocks of zeros, of subnormal numbers, near the type's ends: scales from 2^-126 up, quotients by real division."""
    x = torch.randn((384, 640), generator=L.gen(3), device="cuda")
    x[:, :128] = 0.0
    x[:128, 128:256] *= 1e-44
    x[:, 256:384] *= 2.0 ** 100
    x[128:256, 384:512] *= 2.0 ** -85
    x[256:, 384:512] *= 1e37
    x[5, 520] = 3.4028234663852886e38
    check(x, block, qt)
    q, scale = quantize(x, block, qt)
    assert (q[:, :128].float() == 0).all() and (scale.reshape(-1)[0] == 1.0)


@pytest.mark.parametrize("block", BLOCKS)
@pytest.mark.parametrize("qt", Q)
@pytest.mark.parametrize("xt", X)
def test_infinities_and_nans_mark_their_block(cuda_device, block, qt, xt):
    x = torch.randn((256, 384), generator=L.gen(4), device="cuda").to(L.WIDE[xt])
    x[3, 5] = float("inf")
    x[130, 200] = float("nan")
    x[200, 300], x[200, 301] = float("-inf"), float("nan")
    q, scale = quantize(x, block, qt)
    back = q.double() * scale.double().repeat_interleave(block[0], 0)[:256].repeat_interleave(block[1], 1)[:, :384]
    bad = ~torch.isfinite(x)
    marked = torch.nn.functional.max_pool2d(bad.double()[None, None], block, block)[0, 0].bool()
    where = marked.repeat_interleave(block[0], 0).repeat_interleave(block[1], 1)
    assert torch.isnan(back[where]).all() and torch.isfinite(back[~where]).all()
    want, want_scale = L.quantize64(torch.where(where, torch.zeros_like(x), x), *block, qt)
    assert torch.equal(scale[~marked], want_scale[~marked])
    assert torch.isinf(scale[marked]).any() and torch.isnan(scale[marked]).any()


def test_ties_go_to_even(cuda_device):
    """With a scale of one the 8-bit neighbours of a tie are known: 17 lies between 16 and 18, 19 between 18 and 20."""
    x = torch.zeros((1, 128), device="cuda")
    x[0, :6] = torch.tensor([448.0, 17.0, 19.0, -17.0, -19.0, 2.0 ** -10])
    q, scale = quantize(x, (1, 128), ck.CKB_F8_E4M3)
    assert scale.item() == 1.0
    assert q[0, :6].float().tolist() == [448.0, 16.0, 20.0, -16.0, -20.0, 0.0]


def test_many_blocks(cuda_device):
    x = torch.randn((5000, 3000), generator=L.gen(5), device="cuda").to(torch.bfloat16)
    for block in BLOCKS:
        check(x, block, ck.CKB_F8_E4M3)


@pytest.mark.parametrize("block", BLOCKS)
@pytest.mark.parametrize("xt", X)
@pytest.mark.parametrize("N", [1, 7, 127, 128, 129, 264, 389])
def test_every_alignment_of_rows(cuda_device, block, xt, N):
    """Rows of x and q that start on every byte their elements allow, full and partial blocks, NaN between the rows."""
    g = L.gen(N)
    for pad in (0, 1, 3):
        ld = N + pad + (N + pad + 1) % 2  # odd: the rows walk through all alignments
        x = torch.full((150 * ld + 8,), float("nan"), dtype=L.WIDE[xt], device="cuda")
        for start in (0, 1, 5):
            v = x[start:start + 150 * ld].view(150, ld)[:, :N]
            v.copy_(torch.randn((150, N), generator=g, device="cuda"))
            check(v, block, ck.CKB_F8_E4M3, ldq=ld, q_offset=start)
            x.fill_(float("nan"))
