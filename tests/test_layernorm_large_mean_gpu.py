"""GPU tests of layer norm's backward pass on rows whose mean * rstd is no 32-bit number although every xhat is one."""
import pytest
import torch

import composable_kernel_b200 as ck
from tests import llm_helpers as L

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("xt", [ck.CKB_F32, ck.CKB_BF16])
@pytest.mark.parametrize("N,ld", [(100, 100), (101, 101), (1032, 1032), (1030, 1040), (5000, 5000), (5001, 5001), (8203, 8203), (8200, 8200)])
@pytest.mark.parametrize("weights", [True, False])
def test_constant_rows_of_large_values(cuda_device, xt, N, ld, weights):
    """x = mean everywhere: xhat = 0, so dx = rstd (w - mean of w) and dgamma = 0, whatever the mean.  Row 1 is an
    ordinary one.  dx: the sum of N values of w in chains of 64 at most, half a step of 2^-24 each, of terms that add up
    to N * mean|w|, then five roundings and the output's; ordinary row: the same for the sum of w xhat, times |xhat|."""
    g = L.gen(N)
    M = 4
    x = torch.full((M, ld), float("nan"), dtype=L.WIDE[xt], device="cuda")[:, :N]
    x.copy_(torch.tensor([2.0e36, 0.0, -3.0e36, 1.0e38], device="cuda")[:, None].expand(M, N))
    x[1] = torch.randn((N,), generator=g, device="cuda").to(x.dtype)
    dy = torch.full((M, ld), float("nan"), dtype=L.WIDE[xt], device="cuda")[:, :N]
    dy.copy_(torch.randn((M, N), generator=g, device="cuda"))
    gamma = torch.rand((N,), generator=g, device="cuda") + 0.5 if weights else None
    mean = x.double().mean(1).float()
    mean[[0, 2, 3]] = x[[0, 2, 3], 0].float()
    rstd = torch.full((M,), 316.22775, device="cuda")
    rstd[1] = 1.0
    dx = torch.full((M, N), float("nan"), dtype=x.dtype, device="cuda")
    dg, db = (torch.full((N,), float("nan"), device="cuda") for _ in range(2))
    op = ck.DeviceLayernormBwd(xt, ck.CKB_F32)
    arg = op.MakeArgument(dy.data_ptr(), x.data_ptr(), gamma.data_ptr() if weights else None, mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(),
                          dg.data_ptr(), db.data_ptr(), M, N, ld, ld, N)
    L.run(op, arg, workspace=True)
    hat = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    w = dy.double() * (gamma.double() if weights else 1.0)
    r = rstd.double()[:, None]
    want = r * (w - w.mean(1, keepdim=True) - hat * (w * hat).mean(1, keepdim=True))
    # |xhat| with its own rounding: half a step of x and of the mean for the distance, one of the product
    chain = (64 + 5) * 2.0 ** -24
    hat_off = (x[1].double().abs() + mean[1].double().abs()) * r[1] * 2.0 ** -24 + hat[1].abs() * 2.0 ** -24
    sums = r * chain * (w.abs() + w.abs().mean(1, keepdim=True) + hat.abs() * (w * hat).abs().mean(1, keepdim=True))
    sums[1] += r[1] * (hat_off * (w[1] * hat[1]).mean().abs() + hat[1].abs() * (w[1].abs() * hat_off).mean())
    bound = sums + L.HALF[x.dtype] * (want.abs() + sums)
    assert ((dx.double() - want).abs() <= bound).all()
    # dgamma: only row 1 counts; four terms in any order
    dg_want = (dy.double() * hat).sum(0)
    dg_off = dy[1].double().abs() * (hat_off + 4 * 2.0 ** -24 * hat[1].abs())
    assert ((dg.double() - dg_want).abs() <= dg_off + 2.0 ** -24 * dg_want.abs()).all()
    assert ((db.double() - dy.double().sum(0)).abs() <= 4 * 2.0 ** -24 * dy.double().abs().sum(0)).all()
