"""Cases of the 8-bit block-scaled operators and of layer norm: inputs, plain forms, exact values, work.

Every operator exists twice here: in elementary torch operations in 32 bits (``own`` false), and as the calls a user
makes of this package (``own`` true).  Sizes are those of this repository's GEMM and grouped-GEMM configurations
(rows 3840, N = K = 4096, 64 groups of 256 * (1 + g mod 16) rows) or generic ones next to them.

Operators
  quantize   blocks of 1 x 128, 128 x 1 or 128 x 128 values -> 8-bit floats and one 32-bit scale per block
  gemm       E = (A * scale) (B * scale), A and B 8-bit with block scales, contraction length K
  grouped_m  the same for the experts of a layer: group g owns rows offsets[g] .. offsets[g + 1] of A and E
  grouped_k  the experts' weight gradients: group g owns the 128-row blocks offsets[g] .. offsets[g + 1] of A and B
  ln_fwd     layer norm, to 16 / 32 bits and (or) straight to 8-bit blocks of 1 x 128
  ln_bwd     its backward pass: dx, dgamma, dbeta
"""
import math

import torch

own = False

BLOCK = 128
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
F8_MAX = {"e4m3": 448.0, "e5m2": 57344.0}
WIDE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
WIDE_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # the activations of 16 sequences that decode one token each, on their way into an 8-bit product
        {"name": "quantize decode", "op": "quantize", "rows": 16, "cols": 4096, "block": "1x128", "x": "bf16", "q": "e4m3"},
        # master weights of a projection into 8-bit tiles; neither extent a multiple of the block
        {"name": "quantize weights", "op": "quantize", "rows": 14347, "cols": 5000, "block": "128x128", "x": "f32", "q": "e4m3"},
        # one projection while four sequences decode
        {"name": "gemm decode", "op": "gemm", "M": 4, "N": 4096, "K": 4096, "form": "forward", "e": "bf16"},
        # a prompt through a projection (the repository's own GEMM size)
        {"name": "gemm prompt", "op": "gemm", "M": 3840, "N": 4096, "K": 4096, "form": "forward", "e": "bf16"},
        # a weight gradient over a ragged number of tokens, added up in 32 bits
        {"name": "gemm weight gradient", "op": "gemm", "M": 11008, "N": 4096, "K": 8190, "form": "wgrad", "e": "f32"},
        # 64 experts, a handful of decoded tokens for each, some experts idle, the batch padded behind its end
        {"name": "grouped decode", "op": "grouped_m", "groups": 64, "rows": 256, "tail": 9, "N": 4096, "K": 4096, "spread": "random", "form": "forward"},
        # the repository's grouped-GEMM configuration: 64 groups of 256 to 4096 rows
        {"name": "grouped prompt", "op": "grouped_m", "groups": 64, "rows": 139264, "tail": 0, "N": 4096, "K": 4096, "spread": "steps", "form": "forward"},
        # weight gradients of 16 experts
        {"name": "grouped weight gradient", "op": "grouped_k", "groups": 16, "blocks": 100, "M": 2048, "N": 1408, "e": "f32"},
        # a few decoded tokens
        {"name": "layer norm decode", "op": "ln_fwd", "rows": 7, "cols": 4096, "x": "bf16", "w": "bf16", "out": "y"},
        # a prompt, normalised straight into the operand of the next 8-bit product; mean and rstd kept for training
        {"name": "layer norm quantized", "op": "ln_fwd", "rows": 8192, "cols": 5120, "x": "bf16", "w": "f32", "out": "q"},
        # a training step's backward pass
        {"name": "layer norm backward", "op": "ln_bwd", "rows": 16384, "cols": 4096, "x": "bf16", "w": "f32"},
        # odd sizes in 32 bits
        {"name": "layer norm backward odd", "op": "ln_bwd", "rows": 1023, "cols": 2561, "x": "f32", "w": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "gemm", "gemm", "grouped_m", "grouped_k", "ln_fwd", "ln_bwd"])
    if op == "quantize":
        cols = _log(rng, 128, 16384)
        return {"op": op, "rows": _log(rng, 1, min(32768, (1 << 26) // cols)), "cols": cols, "block": rng.choice(["1x128", "128x1", "128x128"]),
                "x": rng.choice(["bf16", "f16", "f32"]), "q": rng.choice(["e4m3", "e4m3", "e5m2"])}
    if op == "gemm":
        # N, K and the pitches of the 8-bit operands stay multiples of 16 (their rows start on 16-byte boundaries)
        n, k = 16 * _log(rng, 16, 1024), 16 * _log(rng, 8, 512)
        form = rng.choice(["forward", "forward", "dgrad", "wgrad"])
        m = _log(rng, 1, min(8192, (1 << 37) // (n * k)))
        if form == "wgrad":
            m, k = 16 * max(8, m // 16), k + rng.randrange(16)
        return {"op": op, "M": m, "N": n, "K": k, "form": form, "e": "f32" if form == "wgrad" else rng.choice(["bf16", "f16"])}
    if op == "grouped_m":
        n, k, rows = 16 * _log(rng, 32, 256), 16 * _log(rng, 32, 256), _log(rng, 16, 8192)
        return {"op": op, "groups": _log(rng, 2, 128), "rows": rows, "tail": rng.randrange(rows // 4 + 1), "N": n, "K": k, "spread": "random", "form": rng.choice(["forward", "dgrad"])}
    if op == "grouped_k":
        return {"op": op, "groups": _log(rng, 2, 32), "blocks": _log(rng, 4, 128), "M": 16 * _log(rng, 32, 160), "N": 16 * _log(rng, 32, 160), "e": rng.choice(["f32", "bf16"])}
    cols = _log(rng, 64, 16384)
    rows = _log(rng, 1, min(32768, (1 << 26) // cols))
    x = rng.choice(["bf16", "bf16", "f16", "f32"])
    w = rng.choice([x, "f32"])
    if op == "ln_fwd":
        return {"op": op, "rows": rows, "cols": cols, "x": x, "w": w, "out": rng.choice(["y", "q", "yq"])}
    return {"op": op, "rows": rows, "cols": cols, "x": x, "w": w}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _blocks(n):
    return -(-n // BLOCK)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(g, rows, cols, dtype):
    # hidden states: a few channels are much larger than the rest
    x = torch.randn((rows, cols), generator=g, device="cuda")
    return x.mul_(torch.exp(torch.randn((cols,), generator=g, device="cuda"))).to(WIDE[dtype])


def _eight_bit(g, shape, kind):
    # what a quantizer leaves: the largest value of a block near the type's largest
    x = torch.randn(shape, generator=g, device="cuda")
    return x.mul_(F8_MAX[kind] / 4).clamp_(-F8_MAX[kind], F8_MAX[kind]).to(F8[kind])


def _scales(g, shape, size):
    return torch.exp(torch.randn(shape, generator=g, device="cuda") * 0.5) * size


def _group_sizes(case, seed, total, n):
    if case.get("spread") == "steps":
        return [256 * (1 + i % 16) for i in range(n)]
    g = torch.Generator().manual_seed(seed)
    share = torch.rand((n,), generator=g).square()  # uneven, as a router's choices are
    pick = torch.multinomial(share + 1e-6, total, replacement=True, generator=g)
    return torch.bincount(pick, minlength=n).tolist()


def _inputs(case, seed):
    g, op = _gen(seed), case["op"]
    s = {"case": case}
    if op == "quantize":
        s["x"] = _activations(g, case["rows"], case["cols"], case["x"])
    elif op == "gemm":
        m, n, k, kb, form = case["M"], case["N"], case["K"], _blocks(case["K"]), case["form"]
        # forward: activations [M, K], weights [N, K].  dgrad: output gradients [M, K] in e5m2, weights [K, N].
        # wgrad: both operands lie token by token ([K, M] and [K, N]) and carry a scale per column and 128 tokens.
        wg = form == "wgrad"
        s["a"] = _eight_bit(g, (k, m) if wg else (m, k), "e4m3" if form == "forward" else "e5m2")
        s["b"] = _eight_bit(g, (n, k) if form == "forward" else (k, n), "e4m3")
        s["sa"] = _scales(g, (kb, m) if wg else (m, kb), 1e-3)
        s["sb"] = _scales(g, (kb, n) if wg or form == "dgrad" else (n, kb), 1e-4) if wg else _scales(
            g, (_blocks(n), kb) if form == "forward" else (kb, _blocks(n)), 1e-4)
    elif op == "grouped_m":
        n, k, kb, rows, form = case["N"], case["K"], _blocks(case["K"]), case["rows"], case["form"]
        s["sizes"] = _group_sizes(case, seed, rows - case["tail"], case["groups"])
        s["offsets"] = torch.tensor([0] + s["sizes"], device="cuda").cumsum(0).to(torch.int32)
        s["a"] = _eight_bit(g, (rows, k), "e4m3" if form == "forward" else "e5m2")
        s["b"] = _eight_bit(g, (case["groups"], n, k) if form == "forward" else (case["groups"], k, n), "e4m3")
        s["sa"] = _scales(g, (rows, kb), 1e-3)
        s["sb"] = _scales(g, (case["groups"], _blocks(n), kb) if form == "forward" else (case["groups"], kb, _blocks(n)), 1e-4)
    elif op == "grouped_k":
        m, n, blocks = case["M"], case["N"], case["blocks"]
        s["sizes"] = _group_sizes(case, seed, blocks, case["groups"])
        s["offsets"] = torch.tensor([0] + s["sizes"], device="cuda").cumsum(0).to(torch.int32)
        s["a"] = _eight_bit(g, (blocks * BLOCK, m), "e5m2")
        s["b"] = _eight_bit(g, (blocks * BLOCK, n), "e4m3")
        s["sa"] = _scales(g, (blocks, m), 1e-3)
        s["sb"] = _scales(g, (blocks, n), 1e-4)
    else:
        rows, cols = case["rows"], case["cols"]
        s["x"] = (_activations(g, rows, cols, "f32") + torch.randn((rows, 1), generator=g, device="cuda")).to(WIDE[case["x"]])
        s["gamma"] = (1 + 0.1 * torch.randn((cols,), generator=g, device="cuda")).to(WIDE[case["w"]])
        s["beta"] = (0.1 * torch.randn((cols,), generator=g, device="cuda")).to(WIDE[case["w"]])
        s["eps"] = 1e-5
        if op == "ln_bwd":
            s["dy"] = torch.randn((rows, cols), generator=g, device="cuda").mul_(1e-2).to(WIDE[case["x"]])
            x = s["x"].double()  # statistics that the forward pass kept
            mean = x.mean(1)
            s["mean"] = mean.float()
            s["rstd"] = (x.sub_(mean[:, None]).square_().mean(1) + s["eps"]).rsqrt().float()
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        _plan(s)
    return s


# ---- the calls of this package --------------------------------------------------------------------------------------
def _plan(s):
    """What a user's program keeps: output buffers and the argument of the device operation."""
    import composable_kernel_b200 as ck
    case, op = s["case"], s["case"]["op"]
    f8 = {"e4m3": ck.CKB_F8_E4M3, "e5m2": ck.CKB_F8_E5M2}
    wide = {"bf16": ck.CKB_BF16, "f16": ck.CKB_F16, "f32": ck.CKB_F32}
    row, col = ck.CKB_ROW_MAJOR, ck.CKB_COL_MAJOR

    def empty(shape, dtype):
        return torch.empty(shape, dtype=dtype, device="cuda")

    if op == "quantize":
        rows, cols = case["rows"], case["cols"]
        br, bc = (int(v) for v in case["block"].split("x"))
        s["q"], s["scale"] = empty((rows, cols), F8[case["q"]]), empty((-(-rows // br), -(-cols // bc)), torch.float32)
        o = ck.DeviceBlockQuantize(wide[case["x"]], f8[case["q"]], br, bc)
        arg = o.MakeArgument(s["x"].data_ptr(), s["q"].data_ptr(), s["scale"].data_ptr(), rows, cols, cols, cols, s["scale"].stride())
        s["out"] = (s["q"], s["scale"])
    elif op == "gemm":
        m, n, k, form = case["M"], case["N"], case["K"], case["form"]
        s["e"] = empty((m, n), WIDE[case["e"]])
        o = ck.DeviceGemmABScale(f8["e4m3" if form == "forward" else "e5m2"], f8["e4m3"], wide[case["e"]], col if form == "wgrad" else row,
                                 col if form == "forward" else row, 1, 1 if form == "wgrad" else BLOCK)
        # scale strides: (from one row of A or column of B to the next block of them, from one K block to the next)
        sa = s["sa"].stride()[::-1] if form == "wgrad" else s["sa"].stride()
        sb = s["sb"].stride() if form == "forward" else s["sb"].stride()[::-1]
        arg = o.MakeArgument(s["a"].data_ptr(), s["b"].data_ptr(), s["sa"].data_ptr(), s["sb"].data_ptr(), s["e"].data_ptr(), m, n, k,
                             s["a"].stride(0), s["b"].stride(0), n, sa, sb)
        s["out"] = s["e"]
    elif op == "grouped_m":
        n, k, form = case["N"], case["K"], case["form"]
        s["e"] = torch.zeros((case["rows"], n), dtype=torch.bfloat16, device="cuda")  # rows behind the last group stay zero
        o = ck.DeviceGroupedGemmABScale(ck.CKB_GROUP_ROWS, f8["e4m3" if form == "forward" else "e5m2"], f8["e4m3"], wide["bf16"], row,
                                        col if form == "forward" else row, 1, BLOCK)
        sb = s["sb"].stride()[1:] if form == "forward" else s["sb"].stride()[:0:-1]
        arg = o.MakeArgument(s["a"].data_ptr(), s["b"].data_ptr(), s["sa"].data_ptr(), s["sb"].data_ptr(), s["e"].data_ptr(), s["offsets"].data_ptr(),
                             case["groups"], case["rows"], n, k, s["a"].stride(0), s["b"].stride(1), n, s["sa"].stride(), sb,
                             s["b"].stride(0), s["sb"].stride(0), 0)
        s["out"] = s["e"]
    elif op == "grouped_k":
        m, n, groups = case["M"], case["N"], case["groups"]
        s["e"] = empty((groups, m, n), WIDE[case["e"]])
        o = ck.DeviceGroupedGemmABScale(ck.CKB_GROUP_K_BLOCKS, f8["e5m2"], f8["e4m3"], wide[case["e"]], col, row, 1, 1)
        arg = o.MakeArgument(s["a"].data_ptr(), s["b"].data_ptr(), s["sa"].data_ptr(), s["sb"].data_ptr(), s["e"].data_ptr(), s["offsets"].data_ptr(),
                             groups, m, n, case["blocks"] * BLOCK, m, n, n, s["sa"].stride()[::-1], s["sb"].stride()[::-1], 0, 0, m * n)
        s["out"] = s["e"]
    elif op == "ln_fwd":
        rows, cols, x = case["rows"], case["cols"], case["x"]
        y = empty((rows, cols), WIDE[x]) if "y" in case["out"] else None
        q = empty((rows, cols), F8["e4m3"]) if "q" in case["out"] else None
        sc = empty((rows, _blocks(cols)), torch.float32) if "q" in case["out"] else None
        mean, rstd = empty((rows,), torch.float32), empty((rows,), torch.float32)
        o = ck.DeviceLayernormFwd(wide[x], wide[case["w"]], f8["e4m3"])
        arg = o.MakeArgument(s["x"].data_ptr(), s["gamma"].data_ptr(), s["beta"].data_ptr(), y.data_ptr() if y is not None else None, mean.data_ptr(),
                             rstd.data_ptr(), rows, cols, cols, cols, s["eps"], q.data_ptr() if q is not None else None,
                             sc.data_ptr() if sc is not None else None, cols, sc.stride() if sc is not None else (0, 0))
        s["out"] = [t for t in (y, q, sc, mean, rstd) if t is not None]
    else:
        rows, cols = case["rows"], case["cols"]
        dx, dg, db = empty((rows, cols), WIDE[case["x"]]), empty((cols,), WIDE[case["w"]]), empty((cols,), WIDE[case["w"]])
        o = ck.DeviceLayernormBwd(wide[case["x"]], wide[case["w"]])
        arg = o.MakeArgument(s["dy"].data_ptr(), s["x"].data_ptr(), s["gamma"].data_ptr(), s["mean"].data_ptr(), s["rstd"].data_ptr(), dx.data_ptr(),
                             dg.data_ptr(), db.data_ptr(), rows, cols, cols, cols, cols)
        s["workspace"] = empty((max(1, o.GetWorkSpaceSize(arg)),), torch.uint8)
        o.SetWorkSpacePointer(arg, s["workspace"].data_ptr())
        s["out"] = [dx, dg, db]
    s["arg"], s["invoker"] = arg, o.MakeInvoker()
    s["stream"] = ck.StreamConfig(torch.cuda.current_stream().cuda_stream)


# ---- plain forms, in 32 bits ----------------------------------------------------------------------------------------
def _quantize(x, block, kind):
    """x in 32 bits -> (8-bit values, scales)."""
    (r, c), (br, bc) = x.shape, (int(v) for v in block.split("x"))
    nr, nc = -(-r // br), -(-c // bc)
    t = torch.nn.functional.pad(x, (0, nc * bc - c, 0, nr * br - r)).view(nr, br, nc, bc)
    amax = t.abs().amax((1, 3))
    scale = torch.where(amax == 0, torch.ones_like(amax), (amax / F8_MAX[kind]).clamp_min(2.0 ** -126))
    q = (t / scale[:, None, :, None]).clamp(-F8_MAX[kind], F8_MAX[kind]).to(F8[kind])
    return q.view(nr * br, nc * bc)[:r, :c].contiguous(), scale


def _spread(scale, rows, cols, per_row, per_col):
    """One scale for each value: each is repeated over its block of per_row x per_col values."""
    return scale.repeat_interleave(per_row, 0)[:rows].repeat_interleave(per_col, 1)[:, :cols]


def _operand(q, scale, per_row, per_col):
    return q.float().mul_(_spread(scale, q.shape[0], q.shape[1], per_row, per_col))


def _ln_fwd(s):
    case, x = s["case"], s["x"].float()
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = (d.square().mean(1) + s["eps"]).rsqrt()
    y = d * rstd[:, None] * s["gamma"].float() + s["beta"].float()
    out = [y.to(WIDE[case["x"]])] if "y" in case["out"] else []
    if "q" in case["out"]:
        out += _quantize(y, "1x128", "e4m3")
    return out + [mean, rstd]


def _ln_bwd(s):
    xhat = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
    dy = s["dy"].float()
    dg, db = (dy * xhat).sum(0), dy.sum(0)
    w = dy * s["gamma"].float()
    dx = s["rstd"][:, None] * (w - w.mean(1, keepdim=True) - xhat * (w * xhat).mean(1, keepdim=True))
    return [dx.to(s["x"].dtype), dg.to(s["gamma"].dtype), db.to(s["gamma"].dtype)]


def _plain(s):
    case, op = s["case"], s["case"]["op"]
    if op == "quantize":
        return _quantize(s["x"].float(), case["block"], case["q"])
    if op == "gemm":
        form, out = case["form"], WIDE[case["e"]]
        if form == "wgrad":
            return (_operand(s["a"], s["sa"], BLOCK, 1).t() @ _operand(s["b"], s["sb"], BLOCK, 1)).to(out)
        b = _operand(s["b"], s["sb"], BLOCK, BLOCK)
        return (_operand(s["a"], s["sa"], 1, BLOCK) @ (b.t() if form == "forward" else b)).to(out)
    if op == "grouped_m":
        t = case["form"] == "forward"
        parts = s["sizes"] + [case["rows"] - sum(s["sizes"])]
        a, b = _operand(s["a"], s["sa"], 1, BLOCK).split(parts), zip(s["b"], s["sb"])
        w = (_operand(q, sc, BLOCK, BLOCK) for q, sc in b)
        done = [x @ (v.t() if t else v) for x, v in zip(a[:-1], w)]
        return torch.cat(done + [torch.zeros((parts[-1], case["N"]), device="cuda")]).bfloat16()
    if op == "grouped_k":
        rows = [v * BLOCK for v in s["sizes"]]
        a, b = _operand(s["a"], s["sa"], BLOCK, 1).split(rows), _operand(s["b"], s["sb"], BLOCK, 1).split(rows)
        return torch.stack([x.t() @ y for x, y in zip(a, b)]).to(WIDE[case["e"]])
    return _ln_fwd(s) if op == "ln_fwd" else _ln_bwd(s)


def run(state):
    if own:
        state["invoker"].Run(state["arg"], state["stream"])
        return state["out"]
    return _plain(state)


# ---- work -----------------------------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "quantize":
        r, c, (br, bc) = case["rows"], case["cols"], (int(v) for v in case["block"].split("x"))
        return {"bytes": r * c * (WIDE_BYTES[case["x"]] + 1) + 4 * -(-r // br) * -(-c // bc), "flops": 2 * r * c}
    if op == "gemm":
        m, n, k, kb = case["M"], case["N"], case["K"], _blocks(case["K"])
        scales = (m + n) * kb if case["form"] == "wgrad" else (m + _blocks(n)) * kb
        return {"bytes": m * k + n * k + 4 * scales + m * n * WIDE_BYTES[case["e"]], "flops": 2 * m * n * k}
    if op == "grouped_m":
        # every expert that has a row reads its weights; with random sizes about groups * (1 - exp(-rows / groups)) have one
        n, k, kb, used, groups = case["N"], case["K"], _blocks(case["K"]), case["rows"] - case["tail"], case["groups"]
        busy = groups if case["spread"] == "steps" else min(groups * (1 - math.exp(-0.5 * used / groups)), used)
        return {"bytes": used * (k + 4 * kb + 2 * n) + busy * (n * k + 4 * _blocks(n) * kb), "flops": 2 * used * n * k}
    if op == "grouped_k":
        m, n, blocks = case["M"], case["N"], case["blocks"]
        return {"bytes": blocks * (m + n) * (BLOCK + 4) + case["groups"] * m * n * WIDE_BYTES[case["e"]], "flops": 2 * m * n * blocks * BLOCK}
    r, c, x, w = case["rows"], case["cols"], WIDE_BYTES[case["x"]], WIDE_BYTES[case["w"]]
    if op == "ln_fwd":
        out = (x if "y" in case["out"] else 0) + (1 if "q" in case["out"] else 0)
        return {"bytes": r * c * (x + out) + 2 * c * w + 8 * r + (4 * r * _blocks(c) if "q" in case["out"] else 0), "flops": 8 * r * c}
    return {"bytes": 3 * r * c * x + 3 * c * w + 8 * r, "flops": 13 * r * c}


# ---- the operators' definitions in 64 bits --------------------------------------------------------------------------
def _exact_quantize(x, block, kind):
    r, c = x.shape
    br, bc = (int(v) for v in block.split("x"))
    row, col = torch.arange(r, device="cuda") // br, torch.arange(c, device="cuda") // bc
    nr, nc = int(row[-1]) + 1, int(col[-1]) + 1
    by_col = torch.zeros((r, nc), dtype=torch.float64, device="cuda").scatter_reduce_(1, col.expand(r, c), x.abs(), "amax")
    amax = torch.zeros((nr, nc), dtype=torch.float64, device="cuda").scatter_reduce_(0, row[:, None].expand(r, nc), by_col, "amax")
    scale = torch.where(amax == 0, 1.0, torch.clamp(amax / F8_MAX[kind], min=2.0 ** -126))
    # an 8-bit value counts in units of the scale as it is kept, in 32 bits
    q = x / scale.float().double()[row][:, col]
    return torch.clamp(q, -F8_MAX[kind], F8_MAX[kind]).to(F8[kind]), scale


def _exact_gemm(a, sa, b, sb, a_rows, b_cols):
    """a [M, K] with scales [M blocks, K blocks], b [K, N] with scales [K blocks, N blocks]."""
    kk = torch.arange(a.shape[1], device="cuda") // BLOCK
    m, n = torch.arange(a.shape[0], device="cuda") // a_rows, torch.arange(b.shape[1], device="cuda") // b_cols
    return (a.double() * sa.double()[m][:, kk]) @ (b.double() * sb.double()[kk][:, n])


def exact(case, seed):
    s, op = _inputs(case, seed), case["op"]
    if op == "quantize":
        return _exact_quantize(s["x"].double(), case["block"], case["q"])
    if op == "gemm":
        if case["form"] == "forward":
            return _exact_gemm(s["a"], s["sa"], s["b"].t(), s["sb"].t(), 1, BLOCK)
        if case["form"] == "dgrad":
            return _exact_gemm(s["a"], s["sa"], s["b"], s["sb"], 1, BLOCK)
        return _exact_gemm(s["a"].t(), s["sa"].t(), s["b"], s["sb"], 1, 1)
    if op == "grouped_m":
        e, at = torch.zeros((case["rows"], case["N"]), dtype=torch.float64, device="cuda"), 0
        for i, n in enumerate(s["sizes"]):
            b, sb = (s["b"][i].t(), s["sb"][i].t()) if case["form"] == "forward" else (s["b"][i], s["sb"][i])
            e[at:at + n] = _exact_gemm(s["a"][at:at + n], s["sa"][at:at + n], b, sb, 1, BLOCK)
            at += n
        return e
    if op == "grouped_k":
        e, at = torch.zeros((case["groups"], case["M"], case["N"]), dtype=torch.float64, device="cuda"), 0
        for i, n in enumerate(s["sizes"]):
            r, t = slice(at * BLOCK, (at + n) * BLOCK), slice(at, at + n)
            e[i] = _exact_gemm(s["a"][r].t(), s["sa"][t].t(), s["b"][r], s["sb"][t], 1, 1)
            at += n
        return e
    x, gamma, beta = s["x"].double(), s["gamma"].double(), s["beta"].double()
    if op == "ln_fwd":
        var, mean = torch.var_mean(x, 1, correction=0)
        rstd = 1 / torch.sqrt(var + s["eps"])
        y = (x - mean[:, None]) * rstd[:, None] * gamma + beta
        out = [y] if "y" in case["out"] else []
        if "q" in case["out"]:
            out += _exact_quantize(y, "1x128", "e4m3")
        return out + [mean, rstd]
    dy, mean, rstd, n = s["dy"].double(), s["mean"].double(), s["rstd"].double(), case["cols"]
    # dx = rstd (dxhat - sum(dxhat) / n - xhat sum(dxhat xhat) / n), dxhat = dy gamma, xhat = (x - mean) rstd
    xhat = (x - mean[:, None]) * rstd[:, None]
    dxhat = dy * gamma
    c1, c2 = dxhat.sum(1) / n, torch.einsum("rc,rc->r", dxhat, xhat) / n
    return [rstd[:, None] * (dxhat - c1[:, None] - c2[:, None] * xhat), torch.einsum("rc,rc->c", dy, xhat), dy.sum(0)]
