"""GPU test of power-of-two scales where the largest magnitude of a block is the largest 8-bit value times a power of two, or
one step above or below it: the scale is that power, the next one, or that power again."""
import pytest
import torch

import composable_kernel_b200 as ck
from tests import llm_helpers as L
from tests.test_block_quantize_gpu import BLOCKS, Q, quantize

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("block", BLOCKS)
@pytest.mark.parametrize("qt", Q)
def test_next_power_that_is_not_below(cuda_device, block, qt):
    power = torch.ldexp(torch.ones(120, device="cuda"), torch.arange(-20, 20, device="cuda").repeat_interleave(3))
    top = power * L.QMAX[qt]
    step = torch.tensor([0.0, 2.0 ** -8, -2.0 ** -8], device="cuda").repeat(40)  # a step of bf16 next to 1.75 * 2^n: 2^-7 of 2^n
    top = (top + step * top).to(torch.bfloat16)
    want = power * torch.tensor([1.0, 2.0, 1.0], device="cuda").repeat(40)
    assert (top[1::3].float() > top[0::3].float()).all() and (top[2::3].float() < top[0::3].float()).all()
    # one block for each of them, the value somewhere inside, smaller ones around
    rows, cols = block
    x = torch.zeros((120 * rows, cols), dtype=torch.bfloat16, device="cuda")
    for i in range(120):
        x[i * rows + i % rows, (7 * i) % cols] = -top[i] if i % 2 else top[i]
    q, scale = quantize(x, block, qt, pow2=True)
    assert torch.equal(scale.reshape(-1), want)
    back = q.float() * scale.repeat_interleave(rows, 0).repeat_interleave(cols, 1)[:, :cols]
    largest = back.abs().reshape(120, -1).amax(1)
    assert ((largest - top.float()).abs() <= torch.finfo(L.F8[qt]).eps / 2 * top.float()).all()
