"""GPU tests of the 8-bit products, the block quantizer and layer norm as a model uses them together: a layer forward and
backward, experts, captured graphs, several streams, rows that lie far apart.

Every product is compared with the 64-bit product of the very 8-bit values and scales that went into it; the whole chain
with the 64-bit chain on the unrounded inputs, within what the 8-bit roundings may cost."""
import pytest
import torch

import composable_kernel_b200 as ck
from composable_kernel_b200 import capi
from tests import llm_helpers as L

pytestmark = pytest.mark.gpu

ROW, COL = ck.CKB_ROW_MAJOR, ck.CKB_COL_MAJOR
E4, BF, F32 = ck.CKB_F8_E4M3, ck.CKB_BF16, ck.CKB_F32
EPS = 1e-5


def up16(n):
    return (n + 15) // 16 * 16


def stream_config():
    return ck.StreamConfig(torch.cuda.current_stream().cuda_stream)


def go(op, arg):
    assert op.IsSupportedArgument(arg), capi.last_error()
    op.MakeInvoker().Run(arg, stream_config())


def quantize(x, block, q=None, s=None):
    """[M, N] -> 8-bit rows on a pitch of 16 bytes and the scales [row blocks, column blocks]."""
    M, N = x.shape
    q = torch.zeros((M, up16(N)), dtype=torch.uint8, device="cuda") if q is None else q
    s = torch.zeros((-(-M // block[0]), -(-N // block[1])), device="cuda") if s is None else s
    op = ck.DeviceBlockQuantize(BF, E4, *block)
    go(op, op.MakeArgument(x.data_ptr(), q.data_ptr(), s.data_ptr(), M, N, x.stride(0), q.stride(0), s.stride()))
    return q, s


def value(q, s, block, n):
    """What 8-bit values and scales stand for, in 64 bits."""
    m = q.shape[0]
    v = q[:, :n].contiguous().view(torch.float8_e4m3fn).double()
    return v * s.double()[torch.arange(m, device="cuda") // block[0]][:, torch.arange(n, device="cuda") // block[1]]


def norm(x, gamma, beta, y, mean, rstd, q=None, qs=None):
    M, N = x.shape
    op = ck.DeviceLayernormFwd(BF, F32, E4)
    go(op, op.MakeArgument(x.data_ptr(), gamma.data_ptr(), beta.data_ptr(), y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), M, N, x.stride(0),
                           y.stride(0), EPS, q.data_ptr() if q is not None else None, qs.data_ptr() if qs is not None else None,
                           q.stride(0) if q is not None else 0, qs.stride() if qs is not None else (0, 0)))


def product(te, la, lb, bm, bn, a, sa, b, sb, e, M, N, K):
    """sa: strides (row block, K block), sb: strides (column block, K block), each as a tensor with these two dimensions."""
    op = ck.DeviceGemmABScale(E4, E4, te, la, lb, bm, bn)
    go(op, op.MakeArgument(a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(), e.data_ptr(), M, N, K, a.stride(0), b.stride(0), e.stride(0),
                           sa.stride(), sb.stride()))


class Layer:
    """out = layer_norm(x) W^T and its gradients; every buffer made once, so that a pass can be captured."""

    def __init__(self, tokens, width, out, seed):
        g = L.gen(seed)
        T, H, O = self.size = tokens, width, out
        t = lambda *s, dtype=torch.bfloat16: torch.zeros(s, dtype=dtype, device="cuda")
        self.x, self.dout = t(T, H), t(T, O)
        self.w = (torch.randn((O, H), generator=g, device="cuda") / H ** 0.5).bfloat16()
        self.gamma = torch.rand(H, generator=g, device="cuda") + 0.5
        self.beta = torch.randn(H, generator=g, device="cuda") * 0.1
        self.fill(seed + 1)
        f = torch.float32
        self.y, self.mean, self.rstd = t(T, H), t(T, dtype=f), t(T, dtype=f)
        self.y8, self.ys = t(T, up16(H), dtype=torch.uint8), t(T, -(-H // 128), dtype=f)
        self.yt8, self.yts = t(T, up16(H), dtype=torch.uint8), t(-(-T // 128), H, dtype=f)
        self.d8, self.ds = t(T, up16(O), dtype=torch.uint8), t(T, -(-O // 128), dtype=f)
        self.dt8, self.dts = t(T, up16(O), dtype=torch.uint8), t(-(-T // 128), O, dtype=f)
        self.w8, self.ws = quantize(self.w, (128, 128))
        self.o, self.dy, self.dw, self.dx = t(T, O), t(T, H), t(O, H, dtype=f), t(T, H)
        self.dgamma, self.dbeta = t(H, dtype=f), t(H, dtype=f)
        self.bwd = ck.DeviceLayernormBwd(BF, F32)
        self.bwd_arg = self.bwd.MakeArgument(self.dy.data_ptr(), self.x.data_ptr(), self.gamma.data_ptr(), self.mean.data_ptr(), self.rstd.data_ptr(),
                                             self.dx.data_ptr(), self.dgamma.data_ptr(), self.dbeta.data_ptr(), T, H, H, H, H)
        n = self.bwd.GetWorkSpaceSize(self.bwd_arg)
        self.workspace = torch.empty(n, dtype=torch.uint8, device="cuda")
        self.bwd.SetWorkSpacePointer(self.bwd_arg, self.workspace.data_ptr(), n)

    def fill(self, seed):
        g = L.gen(seed)
        T, H, O = self.size
        self.x.copy_(torch.randn((T, H), generator=g, device="cuda") * 2 + 0.5)
        self.dout.copy_(torch.randn((T, O), generator=g, device="cuda"))

    def step(self):
        T, H, O = self.size
        norm(self.x, self.gamma, self.beta, self.y, self.mean, self.rstd, self.y8, self.ys)
        product(BF, ROW, COL, 1, 128, self.y8, self.ys, self.w8, self.ws, self.o, T, O, H)
        quantize(self.dout, (1, 128), self.d8, self.ds)
        product(BF, ROW, ROW, 1, 128, self.d8, self.ds, self.w8, self.ws.t(), self.dy, T, H, O)
        quantize(self.dout, (128, 1), self.dt8, self.dts)
        quantize(self.y, (128, 1), self.yt8, self.yts)
        product(F32, COL, ROW, 1, 1, self.dt8, self.dts.t(), self.yt8, self.yts.t(), self.dw, O, H, T)
        go(self.bwd, self.bwd_arg)

    def outputs(self):
        return [t.clone() for t in (self.o, self.dy, self.dw, self.dx, self.dgamma, self.dbeta, self.y8, self.ys)]

    def check(self):
        T, H, O = self.size
        y, w, d = value(self.y8, self.ys, (1, 128), H), value(self.w8, self.ws, (128, 128), H), value(self.d8, self.ds, (1, 128), O)
        dt, yt = value(self.dt8, self.dts, (128, 1), O), value(self.yt8, self.yts, (128, 1), H)
        for got, a, b, k in ((self.o, y, w.t(), H), (self.dy, d, w, O), (self.dw, dt.t(), yt, T)):
            L.check_product(got, a @ b, a.abs() @ b.abs(), k)
        # the whole chain: an 8-bit value is off by half a step, 2^-4 of the value or 2^-10 of its scale among the subnormals,
        # and what layer norm writes by its own 32-bit arithmetic besides (2^-14 of the row's largest value is far above it)
        x = self.x.double()
        mu = x.mean(1, keepdim=True)
        rstd = 1 / (((x - mu) ** 2).mean(1, keepdim=True) + EPS).sqrt()
        y64 = (x - mu) * rstd * self.gamma.double() + self.beta.double()
        wd, dd = self.w.double(), self.dout.double()

        def off(v, s, block, extra=0.0):
            m, n = v.shape
            sc = s.double()[torch.arange(m, device="cuda") // block[0]][:, torch.arange(n, device="cuda") // block[1]]
            return v.abs() * 2.0 ** -4 + sc * 2.0 ** -10 + (1 + 2.0 ** -4) * extra

        small = y64.abs().amax(1, keepdim=True) * 2.0 ** -14
        oy, ow, od = off(y64, self.ys, (1, 128), small), off(wd, self.ws, (128, 128)), off(dd, self.ds, (1, 128))
        odt, oyt = off(dd, self.dts, (128, 1)), off(y64, self.yts, (128, 1), small + y64.abs() * 2.0 ** -8)
        for got, a, oa, b, ob in ((self.o, y64, oy, wd.t(), ow.t()), (self.dy, dd, od, wd, ow), (self.dw, dd.t(), odt.t(), y64, oyt)):
            want = a @ b
            rounding = oa @ b.abs() + (a.abs() + oa) @ ob
            rounding += (want.abs() + rounding) * 2.0 ** -8 + (a.abs() @ b.abs()) * 2.0 ** -14
            assert ((got.double() - want).abs() <= rounding).all()
        # layer norm's gradients from the dy that the product wrote: the formula, as 64-bit autograd gives it
        xg, gg, bg = (t.clone().requires_grad_() for t in (x, self.gamma.double(), self.beta.double()))
        m = xg.mean(1, keepdim=True)
        out = (xg - m) / (((xg - m) ** 2).mean(1, keepdim=True) + EPS).sqrt() * gg + bg
        out.backward(self.dy.double())
        # 32-bit sums over H or T terms of at most the largest magnitudes, a step each
        top = self.dy.double().abs().amax() * (x - mu).abs().amax() * rstd.amax()
        hat = ((x - mu) * rstd).abs().amax()
        lead = rstd.amax() * self.gamma.double().amax() * self.dy.double().abs().amax() * (2 + hat ** 2)
        assert ((self.dx.double() - xg.grad).abs() <= 2.0 ** -8 * xg.grad.abs() + lead * 80 * 2.0 ** -24 * 2).all()
        assert ((self.dgamma.double() - gg.grad).abs() <= top * T * 40 * 2.0 ** -24).all()
        assert ((self.dbeta.double() - bg.grad).abs() <= self.dy.double().abs().amax() * T * 40 * 2.0 ** -24).all()


@pytest.mark.parametrize("T,H,O", [(1, 128, 128), (7, 264, 130), (300, 520, 392), (1025, 1024, 2048)])
def test_a_layer_forward_and_backward(cuda_device, T, H, O):
    layer = Layer(T, H, O, seed=T)
    layer.step()
    torch.cuda.synchronize()
    assert ck.device_status() == 0
    layer.check()


def test_a_step_gives_the_same_bits_again(cuda_device):
    layer = Layer(260, 1160, 640, seed=1)
    layer.step()
    first = layer.outputs()
    for _ in range(3):
        layer.step()
        for a, b in zip(first, layer.outputs()):
            assert torch.equal(a, b)


def test_captured_steps_replay_on_new_inputs(cuda_device):
    layer, side = Layer(130, 520, 264, seed=2), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.step()  # first-use initialisation outside the capture
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    before = ck.launch_count()
    with torch.cuda.graph(graph, stream=side):
        layer.step()
    assert ck.launch_count() == before + 9  # layer norm, 3 products, 3 quantizers, 2 of the backward pass
    for seed in (11, 12):
        layer.fill(seed)
        for t in (layer.o, layer.dy, layer.dw, layer.dx, layer.dgamma, layer.dbeta):
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        got = layer.outputs()
        layer.check()
        layer.step()
        for a, b in zip(got, layer.outputs()):
            assert torch.equal(a, b)


def test_two_graphs_and_an_eager_stream_at_once(cuda_device):
    """Each with its own buffers; nothing of the library's own is shared between them."""
    layers = [Layer(129, 392, 264, seed=3), Layer(64, 1160, 136, seed=4), Layer(300, 136, 520, seed=5)]
    streams = [torch.cuda.Stream() for _ in layers]
    want = []
    for layer in layers:
        layer.step()
        torch.cuda.synchronize()
        want.append(layer.outputs())
    graphs = []
    for layer, s in zip(layers[:2], streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            layer.step()
        graphs.append(graph)
    for _ in range(20):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            layers[2].step()
    torch.cuda.synchronize()
    for layer, outputs in zip(layers, want):
        for a, b in zip(outputs, layer.outputs()):
            assert torch.equal(a, b)


def test_k_split_products_on_two_streams(cuda_device):
    """Clusters that hand parts over through shared memory, two launches in flight."""
    g = L.gen(6)
    tile = capi.scaled_tile(32, 1, 8)
    runs = []
    for i in range(2):
        a, b = L.eight_bit(g, (20 + i, 4096), E4), L.eight_bit(g, (1000, 4096), E4)
        sa, sb = L.scales(g, (20 + i, 32)), L.scales(g, (8, 32))
        e = torch.zeros((20 + i, 1000), dtype=torch.bfloat16, device="cuda")
        op = ck.DeviceGemmABScale(E4, E4, BF, ROW, COL, 1, 128, tile_config=tile)
        arg = op.MakeArgument(a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(), e.data_ptr(), 20 + i, 1000, 4096, 4096, 4096, 1000,
                              sa.stride(), sb.stride())
        runs.append((op, arg, e, a, b, sa, sb, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(30):
        for op, arg, *_, s in runs:
            op.MakeInvoker().Run(arg, ck.StreamConfig(s.cuda_stream))
    torch.cuda.synchronize()
    assert ck.device_status() == 0
    for op, arg, e, a, b, sa, sb, s in runs:
        L.check_product(e, *L.product64(a.float(), sa, b.t().float(), sb.t(), 1, 128), 4096)


@pytest.mark.parametrize("rows", [[3, 0, 130, 1, 57], [0, 0, 5], [128, 256, 0, 128]])
def test_experts_forward_and_weight_gradient(cuda_device, rows):
    """Tokens of each expert in rows of their own, each expert's rows padded to whole K blocks for the weights' gradient."""
    g = L.gen(len(rows))
    G, H, O = len(rows), 264, 392
    padded = [-(-r // 128) * 128 for r in rows]
    starts = [sum(padded[:i]) for i in range(G + 1)]
    T = starts[-1] + 128  # a block behind the last expert
    x, d = torch.zeros((T, H), dtype=torch.bfloat16, device="cuda"), torch.zeros((T, O), dtype=torch.bfloat16, device="cuda")
    for i, r in enumerate(rows):
        x[starts[i]:starts[i] + r] = torch.randn((r, H), generator=g, device="cuda").bfloat16()
        d[starts[i]:starts[i] + r] = torch.randn((r, O), generator=g, device="cuda").bfloat16()
    w = torch.randn((G * O, H), generator=g, device="cuda").bfloat16()
    # each expert's weights quantized on their own: O is no multiple of 128
    w8 = torch.zeros((G, O, up16(H)), dtype=torch.uint8, device="cuda")
    ws = torch.zeros((G, -(-O // 128), -(-H // 128)), device="cuda")
    for i in range(G):
        quantize(w[i * O:(i + 1) * O], (128, 128), w8[i], ws[i])
    x8, xs = quantize(x, (1, 128))
    e = torch.full((T, O), float("nan"), dtype=torch.bfloat16, device="cuda")
    offsets = torch.tensor(starts, dtype=torch.int32, device="cuda")
    op = ck.DeviceGroupedGemmABScale(ck.CKB_GROUP_ROWS, E4, E4, BF, ROW, COL, 1, 128)
    go(op, op.MakeArgument(x8.data_ptr(), w8.data_ptr(), xs.data_ptr(), ws.data_ptr(), e.data_ptr(), offsets.data_ptr(), G, T, O, H, x8.stride(0),
                           w8.stride(1), O, xs.stride(), ws.stride()[1:], w8.stride(0), ws.stride(0)))
    # weights' gradient: scales along the tokens
    xt8, xts = quantize(x, (128, 1))
    dt8, dts = quantize(d, (128, 1))
    dw = torch.full((G, O, H), float("nan"), device="cuda")
    blocks = torch.tensor([s // 128 for s in starts], dtype=torch.int32, device="cuda")
    opk = ck.DeviceGroupedGemmABScale(ck.CKB_GROUP_K_BLOCKS, E4, E4, F32, COL, ROW, 1, 1)
    go(opk, opk.MakeArgument(dt8.data_ptr(), xt8.data_ptr(), dts.data_ptr(), xts.data_ptr(), dw.data_ptr(), blocks.data_ptr(), G, O, H, T, dt8.stride(0),
                             xt8.stride(0), H, dts.t().stride(), xts.t().stride(), GroupStrideE=O * H))
    torch.cuda.synchronize()
    assert ck.device_status() == 0
    xv, xtv, dtv = value(x8, xs, (1, 128), H), value(xt8, xts, (128, 1), H), value(dt8, dts, (128, 1), O)
    for i in range(G):
        s = slice(starts[i], starts[i + 1])
        wv = value(w8[i], ws[i], (128, 128), H)
        L.check_product(e[s], xv[s] @ wv.t(), xv[s].abs() @ wv.abs().t(), H)
        assert (e[starts[i] + rows[i]:starts[i + 1]] == 0).all()  # padded rows are rows of zeros
        L.check_product(dw[i], dtv[s].t() @ xtv[s], dtv[s].abs().t() @ xtv[s].abs(), max(padded[i], 1))
    assert torch.isnan(e[starts[-1]:]).all()


FAR = 1 << 28  # elements between rows: from row 16 on, offsets pass 32 bits


def far(rows, cols, dtype):
    """[rows, cols] on a pitch of FAR elements; only these rows of the buffer are ever touched."""
    return torch.empty((rows * FAR,), dtype=dtype, device="cuda").view(rows, FAR)[:, :cols]


def test_rows_that_lie_far_apart(cuda_device):
    g = L.gen(8)
    M, N = 20, 264
    x = far(M, N, torch.bfloat16)
    x.copy_(torch.randn((M, N), generator=g, device="cuda"))
    near = x.contiguous()
    for block in ((1, 128), (128, 1), (128, 128)):
        q = far(M, N, torch.uint8)
        _, s = quantize(x, block, q)
        want, ws = quantize(near, block)
        assert torch.equal(q, want[:, :N]) and torch.equal(s, ws)
        del q
    gamma, beta = torch.rand(N, device="cuda"), torch.rand(N, device="cuda")
    stats = [torch.zeros(M, device="cuda") for _ in range(4)]
    y, near_y = far(M, N, torch.bfloat16), torch.zeros_like(near)
    norm(x, gamma, beta, y, *stats[:2])
    norm(near, gamma, beta, near_y, *stats[2:])
    assert torch.equal(y, near_y) and torch.equal(stats[0], stats[2]) and torch.equal(stats[1], stats[3])
    outs = []
    for dy, xx, dx in ((y, x, far(M, N, torch.bfloat16)), (near_y, near, torch.zeros_like(near))):
        dg, db = torch.zeros(N, device="cuda"), torch.zeros(N, device="cuda")
        op = ck.DeviceLayernormBwd(BF, F32)
        L.run(op, op.MakeArgument(dy.data_ptr(), xx.data_ptr(), gamma.data_ptr(), stats[0].data_ptr(), stats[1].data_ptr(), dx.data_ptr(), dg.data_ptr(),
                                  db.data_ptr(), M, N, dy.stride(0), xx.stride(0), dx.stride(0)), workspace=True)
        outs.append((dx.clone(), dg, db))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_products_of_rows_that_lie_far_apart(cuda_device):
    g = L.gen(9)
    M, N, K = 20, 24, 264
    a, b, e = far(M, K, torch.uint8), far(N, K, torch.uint8), far(M, N, torch.bfloat16)
    a.copy_(L.eight_bit(g, (M, K), E4).view(torch.uint8))
    b.copy_(L.eight_bit(g, (N, K), E4).view(torch.uint8))
    sa, sb = L.scales(g, (M, 3)), L.scales(g, (1, 3))
    av, bv = a.contiguous().view(torch.float8_e4m3fn).float(), b.contiguous().view(torch.float8_e4m3fn).float()
    ref, mag = L.product64(av, sa, bv.t(), sb.t(), 1, 128)
    for tile in (0, capi.scaled_tile(128, 2), capi.scaled_tile(128, 1)):
        e.fill_(float("nan"))
        op = ck.DeviceGemmABScale(E4, E4, BF, ROW, COL, 1, 128, tile_config=tile)
        L.run(op, op.MakeArgument(a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(), e.data_ptr(), M, N, K, FAR, FAR, FAR, sa.stride(), sb.stride()))
        L.check_product(e, ref, mag, K)


def test_host_pointers_are_refused(cuda_device):
    h = torch.zeros(128 * 128, dtype=torch.float32)
    d = torch.zeros(128 * 128, dtype=torch.float32, device="cuda")
    p, r = h.data_ptr(), d.data_ptr()
    gemm, quant = ck.DeviceGemmABScale(), ck.DeviceBlockQuantize(F32, E4)
    fwd, bwd = ck.DeviceLayernormFwd(F32, F32), ck.DeviceLayernormBwd(F32, F32)
    for i in range(5):
        v = [r] * 5
        v[i] = p
        calls = [(gemm, gemm.MakeArgument(*v, 16, 16, 128, 128, 128, 16, (1, 16), (1, 1)))]
        if i < 3:
            calls.append((quant, quant.MakeArgument(*v[:3], 4, 128, 128, 128, (1, 1))))
        calls.append((fwd, fwd.MakeArgument(*v, None, 4, 128, 128, 128, EPS)))
        calls.append((bwd, bwd.MakeArgument(*v, r, None, None, 4, 128, 128, 128, 128)))
        for op, arg in calls:
            with pytest.raises(capi.CkbError, match="not a device pointer"):
                op.MakeInvoker().Run(arg, stream_config())
    torch.cuda.synchronize()
