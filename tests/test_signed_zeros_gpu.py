"""GPU tests that 8-bit zeros keep their sign: the bytes of the block quantizer and of layer norm's 8-bit output, compared as
bytes (as numbers -0 equals +0)."""
import pytest
import torch

import composable_kernel_b200 as ck
from tests import llm_helpers as L
from tests.test_block_quantize_gpu import BLOCKS, Q, X, quantize
from tests.test_layernorm_gpu import forward

pytestmark = pytest.mark.gpu


def expected(x, scale, block, qt):
    """x / scale rounded to 32 bits (a 64-bit quotient of 32-bit numbers rounds to the 32-bit one) and to 8 bits."""
    s = scale.double().repeat_interleave(block[0], 0)[:x.shape[0]].repeat_interleave(block[1], 1)[:, :x.shape[1]]
    quotient = (x.double() / s).float()
    return quotient.clamp(-L.QMAX[qt], L.QMAX[qt]).to(L.F8[qt]).view(torch.uint8)


@pytest.mark.parametrize("block", BLOCKS)
@pytest.mark.parametrize("xt", X)
@pytest.mark.parametrize("qt", Q)
@pytest.mark.parametrize("N,ld", [(640, 640), (640, 653), (389, 401)])
def test_quantizer(cuda_device, block, xt, qt, N, ld):
    """Blocks with zeros of both signs among ordinary values, blocks of negative zeros alone, values that round to zero,
    and (32 bits) blocks so small or large that they are divided for real."""
    g = L.gen(N + ld)
    x = torch.full((256, ld), float("nan"), dtype=L.WIDE[xt], device="cuda")[:, :N]
    x.copy_(torch.randn((256, N), generator=g, device="cuda"))
    x[::3, ::5] = -0.0
    x[1::3, 1::5] = 0.0
    x[2::3, 2::5] *= -2.0 ** -12
    x[:128, 128:256] = -0.0
    if xt == ck.CKB_F32:
        x[128:, :128] *= 2.0 ** -100
        x[128:, 128:256] *= 2.0 ** 122
    q, scale = quantize(x, block, qt, ldq=ld)
    want = expected(x, scale, block, qt)
    assert (want == 0x80).sum() > 1000 and (want == 0).sum() > 1000
    assert torch.equal(q.view(torch.uint8), want)


@pytest.mark.parametrize("xt", X)
@pytest.mark.parametrize("N", [300, 1000, 5000, 9000, 17000])
def test_layernorm(cuda_device, xt, N):
    """Rows of zeros, gamma = -1: y = -0 + beta, so the 8-bit values are those of beta, zeros with their signs."""
    g = L.gen(N)
    x = torch.zeros((3, N), device="cuda").to(L.WIDE[xt])
    gamma = torch.full((N,), -1.0, device="cuda")
    beta = torch.randn((N,), generator=g, device="cuda")
    beta[::3] = -0.0
    beta[1::3] = 0.0
    y, q, scale, _, _ = forward(x, gamma, beta, xt, ck.CKB_F32, ck.CKB_F8_E4M3)
    assert torch.equal(torch.signbit(y), torch.signbit(beta).expand(3, N))
    want = expected(beta.expand(3, N), scale, (1, 128), ck.CKB_F8_E4M3)
    assert (want == 0x80).sum() >= N // 4
    assert torch.equal(q.view(torch.uint8), want)
