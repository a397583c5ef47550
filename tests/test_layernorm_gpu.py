"""GPU tests of layer norm, forward and backward, against the formulas in 64 bits and against differences."""
import pytest
import torch

import composable_kernel_b200 as ck
from composable_kernel_b200 import capi
from tests import llm_helpers as L

pytestmark = pytest.mark.gpu

TYPES = [(ck.CKB_BF16, ck.CKB_BF16), (ck.CKB_BF16, ck.CKB_F32), (ck.CKB_F16, ck.CKB_F32), (ck.CKB_F16, ck.CKB_F16), (ck.CKB_F32, ck.CKB_F32)]
SIZES = [(1, 1), (3, 7), (5, 128), (9, 256), (17, 500), (4, 1024), (6, 1025), (33, 2048), (3, 4096), (2, 5120), (5, 8192), (3, 8200), (2, 16384), (2, 16392), (1, 40001)]
EPS = 1e-5


def ptr(t):
    return t.data_ptr() if t is not None else None


def inputs(M, N, xt, wt, seed, ld=None, start=0, mean=0.0):
    g = L.gen(seed)
    ld = ld or N
    x = torch.full((M * ld + start,), float("nan"), dtype=L.WIDE[xt], device="cuda")[start:].view(M, ld)[:, :N]
    x.copy_(torch.randn((M, N), generator=g, device="cuda") * 2 + mean)
    gamma = (1 + 0.3 * torch.randn((N,), generator=g, device="cuda")).to(L.WIDE[wt])
    beta = (0.5 * torch.randn((N,), generator=g, device="cuda")).to(L.WIDE[wt])
    return x, gamma, beta


def forward(x, gamma, beta, xt, wt, qt=None, y_on=True, stats=True, ldy=None, ldq=None, eps=EPS, y_start=0):
    M, N = x.shape
    ldy, ldq = ldy or N, ldq or N
    y = torch.full((M * ldy + y_start,), float("nan"), dtype=x.dtype, device="cuda")[y_start:].view(M, ldy) if y_on else None
    q = torch.full((M, ldq), 0xAA, dtype=torch.uint8, device="cuda") if qt is not None else None
    sc = torch.full((M, -(-N // 128)), -1.0, device="cuda") if qt is not None else None
    mean, rstd = (torch.full((M,), float("nan"), device="cuda") for _ in range(2)) if stats else (None, None)
    op = ck.DeviceLayernormFwd(xt, wt, qt if qt is not None else ck.CKB_F8_E4M3)
    arg = op.MakeArgument(x.data_ptr(), ptr(gamma), ptr(beta), ptr(y), ptr(mean), ptr(rstd), M, N, x.stride(0), ldy, eps, ptr(q), ptr(sc), ldq,
                          sc.stride() if sc is not None else (0, 0))
    assert op.IsSupportedArgument(arg), capi.last_error()
    L.run(op, arg)
    if y_on:
        assert torch.isnan(y[:, N:]).all()
        y = y[:, :N]
    if q is not None:
        assert (q[:, N:] == 0xAA).all()
        q = q[:, :N].contiguous().view(L.F8[qt])
    return y, q, sc, mean, rstd


def norm64(x, gamma, beta, eps=EPS):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    hat = (x - mean) * rstd
    y = hat * (gamma.double() if gamma is not None else 1) + (beta.double() if beta is not None else 0)
    return y, mean, rstd, hat


def stat_bounds(x, rstd, N):
    """What 32-bit statistics may be off.  A row's sum: pairwise or in chains of up to 32 + 20 terms (56 for rows of 40001:
    5 vectors of 8 and 10 steps of shuffles), half a step each, of terms that add up to N * mean|x|; the second pass takes
    out the first mean's rounding, so half a step of the mean itself and that chain over |x - mean| remain.
    rstd: the same chain over squares, halved by the square root, and four roundings."""
    chain = 64 * 2.0 ** -24
    mean_abs = x.double().abs().mean(1, keepdim=True)
    dev = (x.double() - x.double().mean(1, keepdim=True)).abs().mean(1, keepdim=True)
    mean_off = mean_abs * 4 * 2.0 ** -24 + dev * chain
    return mean_off, rstd * (chain / 2 + 4 * 2.0 ** -24) + 1e-30


def y_bound(x, y, gamma, beta, rstd, hat, mean_off, rstd_off, dtype):
    """x - mean is formed as (x - first mean) - correction: half a step of |x - mean| and of the first mean's own error,
    then the product with rstd, gamma and the sum with beta, half a step each, and the output's rounding."""
    g = gamma.double().abs() if gamma is not None else 1.0
    b = beta.double().abs() if beta is not None else 0.0
    inner = g * (hat.abs() * (rstd_off / rstd + 5 * 2.0 ** -24) + rstd * mean_off) + 2.0 ** -24 * (g * hat.abs() + b)
    return inner + L.HALF[dtype] * (y.abs() + inner) + torch.finfo(dtype).smallest_normal * L.HALF[dtype]


@pytest.mark.parametrize("xt,wt", TYPES)
@pytest.mark.parametrize("M,N", SIZES)
def test_forward(cuda_device, xt, wt, M, N):
    x, gamma, beta = inputs(M, N, xt, wt, M + N)
    y, _, _, mean, rstd = forward(x, gamma, beta, xt, wt)
    want, m, r, hat = norm64(x, gamma, beta)
    mean_off, rstd_off = stat_bounds(x, r, N)
    assert ((mean[:, None].double() - m).abs() <= mean_off + 1e-30).all()
    assert ((rstd[:, None].double() - r).abs() <= rstd_off).all()
    assert ((y.double() - want).abs() <= y_bound(x, want, gamma, beta, r, hat, mean_off, rstd_off, x.dtype)).all()


@pytest.mark.parametrize("mean", [1000.0, -1e5])
def test_mean_much_larger_than_the_deviation(cuda_device, mean):
    for N in (200, 3000, 20000):
        x, gamma, beta = inputs(5, N, ck.CKB_F32, ck.CKB_F32, N, mean=mean)
        y, _, _, m32, r32 = forward(x, gamma, beta, ck.CKB_F32, ck.CKB_F32)
        want, m, r, hat = norm64(x, gamma, beta)
        mean_off, rstd_off = stat_bounds(x, r, N)
        assert ((m32[:, None].double() - m).abs() <= mean_off).all()
        assert ((r32[:, None].double() - r).abs() <= rstd_off + r * 1e-6).all()
        # the kernel's own mean keeps more bits than the 32 it returns: only rounding of the distances remains
        inner = L.HALF[torch.float32] * abs(mean) * 2 * r * gamma.double().abs()
        assert ((y.double() - want).abs() <= y_bound(x, want, gamma, beta, r, hat, mean_off, rstd_off, x.dtype) + inner).all()


@pytest.mark.parametrize("ld,start", [(1001, 0), (1008, 0), (1008, 1), (1003, 3)])
def test_strides_and_alignment(cuda_device, ld, start):
    for xt, wt in TYPES:
        x, gamma, beta = inputs(7, 1000, xt, wt, 3, ld, start)
        gamma = torch.cat([gamma[:1], gamma])[1:] if start else gamma  # weights that do not start on 16 bytes
        y, _, _, _, _ = forward(x, gamma, beta, xt, wt, ldy=ld + 5, y_start=start)
        want, m, r, hat = norm64(x, gamma, beta)
        mean_off, rstd_off = stat_bounds(x, r, 1000)
        assert ((y.double() - want).abs() <= y_bound(x, want, gamma, beta, r, hat, mean_off, rstd_off, x.dtype)).all()


@pytest.mark.parametrize("xt,wt", TYPES)
@pytest.mark.parametrize("qt", [ck.CKB_F8_E4M3, ck.CKB_F8_E5M2])
@pytest.mark.parametrize("M,N", [(1, 1), (3, 100), (9, 640), (5, 1024), (7, 1500), (4, 4096), (3, 5000), (2, 9000), (2, 17000)])
def test_forward_to_8_bit_blocks(cuda_device, xt, wt, qt, M, N):
    x, gamma, beta = inputs(M, N, xt, wt, M + N, (N + 15) // 16 * 16)
    if M > 1:  # a row of equal values: y = beta; with beta zero in one block its scale is one
        x[1] = 3.0
        beta[:min(N, 128)] = 0
    for y_on in (False, True):
        y, q, sc, _, _ = forward(x, gamma, beta, xt, wt, qt, y_on=y_on, ldq=N + (8 if y_on else 1))
        want, m, r, hat = norm64(x, gamma, beta)
        mean_off, rstd_off = stat_bounds(x, r, N)
        off = y_bound(x, want, gamma, beta, r, hat, mean_off, rstd_off, torch.float32)
        block = torch.arange(N, device="cuda") // 128
        _, scale = L.quantize64(want.float(), 1, 128, qt)
        # a scale is off by what the largest value of its block may be off
        far = torch.zeros_like(scale, dtype=torch.float64).scatter_reduce_(1, block.expand(M, N), off, "amax") / L.QMAX[qt] + scale.double() * 2.0 ** -23
        plain = scale != 1.0
        assert ((sc.double() - scale.double()).abs() <= far)[plain].all()
        # q * scale: half an 8-bit step of the value (of the smallest step below the smallest normal value)
        back = q.double() * sc.double()[:, block]
        half = torch.finfo(L.F8[qt]).eps / 2
        assert ((back - want).abs() <= off + half * (want.abs() + off) + sc.double()[:, block] * torch.finfo(L.F8[qt]).smallest_normal * half).all()
        if M > 1:
            assert sc[1, 0] == 1.0 and (q[1, :min(N, 128)].float() == 0).all()
        if y_on:
            assert ((y.double() - want).abs() <= y_bound(x, want, gamma, beta, r, hat, mean_off, rstd_off, x.dtype)).all()


def test_without_weights_and_statistics(cuda_device):
    x, gamma, beta = inputs(6, 700, ck.CKB_BF16, ck.CKB_F32, 8)
    for ga, be in ((None, None), (gamma, None), (None, beta)):
        y, _, _, _, _ = forward(x, ga, be, ck.CKB_BF16, ck.CKB_F32, stats=False)
        want, m, r, hat = norm64(x, ga, be)
        mean_off, rstd_off = stat_bounds(x, r, 700)
        assert ((y.double() - want).abs() <= y_bound(x, want, ga, be, r, hat, mean_off, rstd_off, x.dtype)).all()


def test_bad_rows_stay_alone(cuda_device):
    for N in (300, 3000, 20000):
        x, gamma, beta = inputs(9, N, ck.CKB_F32, ck.CKB_F32, 1)
        good, _, _, _, _ = forward(x, gamma, beta, ck.CKB_F32, ck.CKB_F32)
        x[2, 5], x[4, 7] = float("nan"), float("inf")
        y, q, sc, mean, rstd = forward(x, gamma, beta, ck.CKB_F32, ck.CKB_F32, ck.CKB_F8_E4M3)
        keep = [i for i in range(9) if i not in (2, 4)]
        assert torch.equal(y[keep], good[keep])
        assert torch.isnan(y[2]).all() and torch.isnan(rstd[2]) and torch.isnan(sc[2]).all()
        assert torch.isnan(rstd[4]) or rstd[4] == 0


def test_eps_zero_and_equal_values(cuda_device):
    x = torch.full((3, 500), 2.5, device="cuda")
    y, _, _, mean, rstd = forward(x, None, None, ck.CKB_F32, ck.CKB_F32, eps=EPS)
    assert (y == 0).all() and (mean == 2.5).all()
    y, _, _, mean, rstd = forward(x, None, None, ck.CKB_F32, ck.CKB_F32, eps=0.0)
    assert torch.isinf(rstd).all() and torch.isnan(y).all()  # 0 * infinity, as the formula says


# ---- backward -------------------------------------------------------------------------------------
def backward(dy, x, gamma, mean, rstd, xt, wt, dx_on=True, dw_on=True, lddx=None):
    M, N = x.shape
    lddx = lddx or N
    dx = torch.full((M, lddx), float("nan"), dtype=x.dtype, device="cuda") if dx_on else None
    dg, db = (torch.full((N + 4,), float("nan"), dtype=L.WIDE[wt], device="cuda") if dw_on else None for _ in range(2))
    op = ck.DeviceLayernormBwd(xt, wt)
    arg = op.MakeArgument(dy.data_ptr(), x.data_ptr(), ptr(gamma), mean.data_ptr(), rstd.data_ptr(), ptr(dx), ptr(dg), ptr(db), M, N, dy.stride(0),
                          x.stride(0), lddx)
    assert op.IsSupportedArgument(arg), capi.last_error()
    size = op.GetWorkSpaceSize(arg)
    ws = torch.full((size + 256,), 0xFF, dtype=torch.uint8, device="cuda")
    op.SetWorkSpacePointer(arg, ws.data_ptr(), size)
    op.MakeInvoker().Run(arg, ck.StreamConfig(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert (ws[size:] == 0xFF).all()
    if dx_on:
        assert torch.isnan(dx[:, N:]).all()
        dx = dx[:, :N]
    if dw_on:
        assert torch.isnan(dg[N:]).all() and torch.isnan(db[N:]).all()
        dg, db = dg[:N], db[:N]
    return dx, dg, db


def check_backward(dy, x, gamma, xt, wt, **kw):
    M, N = x.shape
    _, m, r, _ = norm64(x, gamma, None)
    mean, rstd = m[:, 0].float(), r[:, 0].float()
    dx, dg, db = backward(dy, x, gamma, mean, rstd, xt, wt, **kw)
    # the formula on the statistics as they are given, in 64 bits
    hat = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    w = dy.double() * (gamma.double() if gamma is not None else 1)
    c1, c2 = w.mean(1, keepdim=True), (w * hat).mean(1, keepdim=True)
    # xhat: a difference (half a step of x and mean's difference) and a product; chains of up to 64 additions in a row's
    # sums; chains of M / parts + parts / 8 + 12 additions in a column's
    u = 2.0 ** -24
    hat_off = hat.abs() * 2 * u
    s1_off = w.abs().mean(1, keepdim=True) * 66 * u
    s2_off = (w * hat).abs().mean(1, keepdim=True) * 70 * u
    if dx is not None:
        want = rstd.double()[:, None] * (w - c1 - hat * c2)
        size = w.abs() + c1.abs() + (hat * c2).abs()
        inner = rstd.double()[:, None] * (5 * u * size + s1_off + hat.abs() * s2_off + hat_off * c2.abs())
        assert ((dx.double() - want).abs() <= inner + L.HALF[x.dtype] * (want.abs() + inner) + torch.finfo(x.dtype).smallest_normal * L.HALF[x.dtype]).all()
    if dg is not None:
        chain = (M + 40) * u
        for got, terms in ((dg, dy.double() * hat), (db, dy.double())):
            want = terms.sum(0)
            inner = terms.abs().sum(0) * (min(chain, 400 * u) + 3 * u)
            # below the smallest normal number the steps are smallest_normal * eps (binary16: 2^-24): off by half of one
            least = torch.finfo(got.dtype).smallest_normal * L.HALF[got.dtype]
            assert ((got.double() - want).abs() <= inner + L.HALF[got.dtype] * (want.abs() + inner) + least).all()


@pytest.mark.parametrize("xt,wt", TYPES)
@pytest.mark.parametrize("M,N", SIZES + [(700, 96), (1500, 1000), (400, 2050), (350, 8192), (180, 9000)])
def test_backward(cuda_device, xt, wt, M, N):
    x, gamma, _ = inputs(M, N, xt, wt, M + 3 * N)
    dy = torch.randn((M, N), generator=L.gen(N), device="cuda").to(x.dtype)
    check_backward(dy, x, gamma, xt, wt)


@pytest.mark.parametrize("ld,start", [(1001, 0), (1008, 0), (1008, 1)])
def test_backward_strides(cuda_device, ld, start):
    for xt, wt in TYPES:
        x, gamma, _ = inputs(40, 1000, xt, wt, 5, ld, start)
        dy, _, _ = inputs(40, 1000, xt, wt, 6, ld + 8, start)
        check_backward(dy, x, gamma, xt, wt, lddx=ld + 16)


def test_backward_parts_alone(cuda_device):
    for N in (500, 3000, 9000):
        x, gamma, _ = inputs(30, N, ck.CKB_BF16, ck.CKB_F32, 5)
        dy = torch.randn((30, N), generator=L.gen(2), device="cuda").to(x.dtype)
        check_backward(dy, x, gamma, ck.CKB_BF16, ck.CKB_F32, dw_on=False)
        check_backward(dy, x, gamma, ck.CKB_BF16, ck.CKB_F32, dx_on=False)
        check_backward(dy, x, None, ck.CKB_BF16, ck.CKB_F32)


def test_backward_gives_the_same_bits_twice(cuda_device):
    for N in (1000, 9000):
        x, gamma, _ = inputs(900, N, ck.CKB_F32, ck.CKB_F32, 5)
        dy = torch.randn((900, N), generator=L.gen(2), device="cuda")
        _, m, r, _ = norm64(x, gamma, None)
        one, two = (backward(dy, x, gamma, m[:, 0].float(), r[:, 0].float(), ck.CKB_F32, ck.CKB_F32) for _ in range(2))
        assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_gradients_against_differences(cuda_device):
    """f(x, gamma, beta) = sum of v * y through the forward kernel in 32 bits; central differences with a step of 2^-6.
    Truncation is (2^-6)^2 / 6 times the third derivative, of the order of |v| rstd^3: 1e-4; rounding of y, 2^-22, over
    the step of 2^-5 between the two sides: 2^-17 per value of the sum, 32 of them: 1e-3."""
    M, N, h = 2, 32, 2.0 ** -6
    x, gamma, beta = inputs(M, N, ck.CKB_F32, ck.CKB_F32, 21)
    v = torch.randn((M, N), generator=L.gen(22), device="cuda")
    _, _, _, mean, rstd = forward(x, gamma, beta, ck.CKB_F32, ck.CKB_F32)
    dx, dg, db = backward(v, x, gamma, mean, rstd, ck.CKB_F32, ck.CKB_F32)

    def f():
        return (forward(x, gamma, beta, ck.CKB_F32, ck.CKB_F32)[0].double() * v.double()).sum().item()

    for t, d, places in ((x, dx, [(0, 0), (0, 31), (1, 5)]), (gamma, dg, [(0,), (17,)]), (beta, db, [(3,), (31,)])):
        for at in places:
            keep = t[at].item()
            t[at] = keep + h
            up = f()
            t[at] = keep - h
            down = f()
            t[at] = keep
            assert abs((up - down) / (2 * h) - d[at].item()) <= 2e-3


# More rows than CTAs, so that a CTA works on several rows side by side and one after the other, at every alignment of rows.
@pytest.mark.parametrize("xt,wt", TYPES)
@pytest.mark.parametrize("M,N", [(300, 1025), (1000, 1037), (700, 2050), (450, 4097), (333, 5120), (310, 8191), (300, 8192), (1300, 200), (310, 9001)])
def test_many_rows_forward(cuda_device, xt, wt, M, N):
    x, gamma, beta = inputs(M, N, xt, wt, M + N)
    y, q, sc, mean, rstd = forward(x, gamma, beta, xt, wt, ck.CKB_F8_E4M3, ldy=N + 1 - N % 2, ldq=N + 1)
    want, m, r, hat = norm64(x, gamma, beta)
    mean_off, rstd_off = stat_bounds(x, r, N)
    assert ((mean[:, None].double() - m).abs() <= mean_off + 1e-30).all() and ((rstd[:, None].double() - r).abs() <= rstd_off).all()
    assert ((y.double() - want).abs() <= y_bound(x, want, gamma, beta, r, hat, mean_off, rstd_off, x.dtype)).all()
    off = y_bound(x, want, gamma, beta, r, hat, mean_off, rstd_off, torch.float32)
    s = sc.double()[:, torch.arange(N, device="cuda") // 128]
    half = torch.finfo(torch.float8_e4m3fn).eps / 2
    assert ((q.double() * s - want).abs() <= off + half * (want.abs() + off) + s * torch.finfo(torch.float8_e4m3fn).smallest_normal * half).all()


@pytest.mark.parametrize("xt,wt", TYPES)
@pytest.mark.parametrize("M,N", [(700, 5121), (500, 4104), (320, 6144), (400, 6145), (5000, 100), (6000, 257), (900, 513), (400, 12289), (1000, 16400)])
def test_many_rows_backward(cuda_device, xt, wt, M, N):
    x, gamma, _ = inputs(M, N, xt, wt, M + N)
    dy = torch.randn((M, N), generator=L.gen(N), device="cuda").to(x.dtype)
    check_backward(dy, x, gamma, xt, wt, lddx=N + 1 - N % 2)
