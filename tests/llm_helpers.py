"""Plain 64-bit forms and error bounds of the 8-bit products, the block quantizer and layer norm.

Half a step of a type is torch.finfo(t).eps / 2 relative to the value (bf16 2^-8, f16 2^-11, f32 2^-24, e4m3 2^-4,
e5m2 2^-3)."""
from __future__ import annotations

import torch

import composable_kernel_b200 as ck

F8 = {ck.CKB_F8_E4M3: torch.float8_e4m3fn, ck.CKB_F8_E5M2: torch.float8_e5m2}
WIDE = {ck.CKB_BF16: torch.bfloat16, ck.CKB_F16: torch.float16, ck.CKB_F32: torch.float32}
QMAX = {ck.CKB_F8_E4M3: 448.0, ck.CKB_F8_E5M2: 57344.0}
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def eight_bit(g, shape, dtype, pitch=None, integers=False):
    """8-bit values [rows, pitch] of which [rows, cols] are the matrix; the padding holds NaN."""
    rows, cols = shape[-2:]
    pitch = pitch or cols
    full = torch.full(shape[:-1] + (pitch,), float("nan"), device="cuda").to(F8[dtype])
    if integers:
        v = torch.randint(-3, 4, shape, generator=g, device="cuda").float()
    else:
        v = (torch.randn(shape, generator=g, device="cuda") * (QMAX[dtype] / 4)).clamp(-QMAX[dtype], QMAX[dtype])
    full[..., :cols] = v.to(F8[dtype])
    return full


def scales(g, shape, pow2=False):
    if pow2:
        return torch.exp2(torch.randint(-3, 3, shape, generator=g, device="cuda").float())
    return torch.exp(torch.randn(shape, generator=g, device="cuda")) * 1e-3


def product64(a, sa, b, sb, block_m, block_n):
    """a [M, K] and b [K, N] of 8-bit values, sa [M blocks, K blocks], sb [K blocks, N blocks] -> (E, sum of magnitudes)."""
    kb = torch.arange(a.shape[1], device="cuda") // 128
    x = a.double() * sa.double()[torch.arange(a.shape[0], device="cuda") // block_m][:, kb]
    y = b.double() * sb.double()[kb][:, torch.arange(b.shape[1], device="cuda") // block_n]
    return x @ y, x.abs() @ y.abs()


def product_bound(ref, size, k, dtype):
    """What E may be off: its own rounding, and 32-bit sums - 128 terms in a block on the tensor core (taken as a whole
    step of 2^-23 each, it may truncate), then the two scales' product, the scaling and an addition per block, half a
    step each - of terms whose magnitudes add up to `size`."""
    blocks = -(-k // 128)
    sums = size * (128 * 2.0 ** -23 + (blocks + 4) * 2.0 ** -24)
    return HALF[dtype] * (ref.abs() + sums) + sums + torch.finfo(dtype).smallest_normal * HALF[dtype]


def check_product(e, ref, size, k):
    off = (e.double() - ref).abs()
    worst = (off / product_bound(ref, size, k, e.dtype)).max().item() if e.numel() else 0.0
    assert torch.isfinite(e).all(), "values that are not finite"
    assert worst <= 1.0, f"{worst:.2f} times the bound"


def quantize64(x, block_m, block_n, dtype, pow2=False):
    """The formula: scales in 32 bits as they are kept, x / scale in 64 bits and its 8-bit rounding."""
    m, n = x.shape
    bm, bn = -(-m // block_m), -(-n // block_n)
    t = torch.zeros((bm * block_m, bn * block_n), dtype=torch.float64, device=x.device)
    t[:m, :n] = x.double()
    t = t.view(bm, block_m, bn, block_n)
    amax = t.abs().amax((1, 3))
    # (a 64-bit quotient by 7 * 2^n is never near a tie of 32 bits, so rounding it again is the 32-bit division)
    scale = (amax / QMAX[dtype]).float().clamp_min(2.0 ** -126)
    scale = torch.where(amax == 0, torch.ones_like(scale), scale)
    if pow2:
        up = torch.exp2(torch.ceil(torch.log2(scale.double()))).float()
        scale = torch.where(torch.isfinite(scale), up, scale)
    q = t / scale.double()[:, None, :, None]
    q = q.reshape(bm * block_m, bn * block_n)[:m, :n]
    return q, scale


def run(op, arg, workspace=False):
    ws = None
    if workspace:
        ws = torch.empty(max(16, op.GetWorkSpaceSize(arg)), dtype=torch.uint8, device="cuda")
        op.SetWorkSpacePointer(arg, ws.data_ptr())
    op.MakeInvoker().Run(arg, ck.StreamConfig(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert ck.device_status() == 0
    return ws
