"""GPU tests of the 8-bit products with block scales (plain and grouped) against 64-bit products."""
import itertools

import pytest
import torch

import composable_kernel_b200 as ck
from composable_kernel_b200 import capi
from tests import llm_helpers as L

pytestmark = pytest.mark.gpu

ROW, COL = ck.CKB_ROW_MAJOR, ck.CKB_COL_MAJOR
E4, E5 = ck.CKB_F8_E4M3, ck.CKB_F8_E5M2


def pad16(n, more=0):
    return (n + 15) // 16 * 16 + more


class Problem:
    """Operands of one product as they lie in memory, and its 64-bit result."""

    def __init__(self, M, N, K, la=ROW, lb=COL, bm=1, bn=128, ta=E4, tb=E4, te=ck.CKB_BF16, seed=0, integers=False, pad=0, k_first=False):
        g = L.gen(seed)
        self.size, self.types, self.layouts, self.blocks = (M, N, K), (ta, tb, te), (la, lb), (bm, bn)
        kb = -(-K // 128)
        a_shape, b_shape = (M, K) if la == ROW else (K, M), (N, K) if lb == COL else (K, N)
        self.a = L.eight_bit(g, a_shape, ta, pad16(a_shape[1], pad), integers)
        self.b = L.eight_bit(g, b_shape, tb, pad16(b_shape[1], pad), integers)
        self.sa, self.sb = L.scales(g, (-(-M // bm), kb), integers), L.scales(g, (kb, -(-N // bn)), integers)
        if k_first:  # the same scales, the other index contiguous
            self.sa, self.sb = self.sa.t().contiguous().t(), self.sb.t().contiguous().t()
        am = self.a[:, :a_shape[1]] if la == ROW else self.a[:, :a_shape[1]].t()
        bm_ = self.b[:, :b_shape[1]].t() if lb == COL else self.b[:, :b_shape[1]]
        self.ref, self.mag = L.product64(am.float(), self.sa, bm_.float(), self.sb, bm, bn)

    def run(self, tile=0, lde=None, offset=0):
        M, N, K = self.size
        lde = lde or N
        dtype = L.WIDE[self.types[2]]
        buf = torch.full((M * lde + offset + 64,), float("nan"), dtype=dtype, device="cuda")
        e = buf[offset:offset + M * lde].view(M, lde)
        op = ck.DeviceGemmABScale(*self.types, *self.layouts, *self.blocks, tile_config=tile)
        arg = op.MakeArgument(self.a.data_ptr(), self.b.data_ptr(), self.sa.data_ptr(), self.sb.data_ptr(), e.data_ptr(), M, N, K,
                              self.a.stride(0), self.b.stride(0), lde, self.sa.stride(), self.sb.stride()[::-1])
        assert op.IsSupportedArgument(arg), capi.last_error()
        L.run(op, arg)
        assert torch.isnan(e[:, N:]).all() and torch.isnan(buf[:offset]).all() and torch.isnan(buf[offset + M * lde:]).all()
        return e[:, :N]

    def check(self, **kw):
        L.check_product(self.run(**kw), self.ref, self.mag, self.size[2])


PAIR = [capi.scaled_tile(c, 2) for c in (128, 192, 224, 256)]
SINGLE = [capi.scaled_tile(c, 1) for c in (16, 32, 64, 128)]


@pytest.mark.parametrize("tile", PAIR + SINGLE)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (5, 130, 128), (300, 520, 400), (513, 257, 1000)])
def test_every_tile(cuda_device, tile, M, N, K):
    Problem(M, N, K, seed=M).check(tile=tile)


@pytest.mark.parametrize("la,lb", list(itertools.product((ROW, COL), (ROW, COL))))
@pytest.mark.parametrize("bm,bn", list(itertools.product((1, 128), (1, 128))))
@pytest.mark.parametrize("tile", [0] + PAIR + [capi.scaled_tile(128, 1)])
def test_layouts_and_scale_blocks(cuda_device, la, lb, bm, bn, tile):
    Problem(391, 464, 700, la, lb, bm, bn, seed=7).check(tile=tile)


@pytest.mark.parametrize("ta,tb", list(itertools.product((E4, E5), (E4, E5))))
@pytest.mark.parametrize("te", [ck.CKB_BF16, ck.CKB_F16, ck.CKB_F32])
@pytest.mark.parametrize("tile", [capi.scaled_tile(256, 2), capi.scaled_tile(128, 2), capi.scaled_tile(32, 1)])
def test_types(cuda_device, ta, tb, te, tile):
    p = Problem(200, 384, 512, ta=ta, tb=tb, te=te, seed=3)
    if te == ck.CKB_F16:  # keep the results inside binary16
        f = 2.0 ** -6 if ta == tb == E4 else 2.0 ** -20 if ta == tb == E5 else 2.0 ** -13
        p.sa *= f
        p.ref, p.mag = p.ref * f, p.mag * f
    p.check(tile=tile)


@pytest.mark.parametrize("M", [1, 2, 7, 16, 17, 33, 64, 100, 128, 129, 255])
def test_few_rows(cuda_device, M):
    Problem(M, 4096, 2048, seed=M).check()


@pytest.mark.parametrize("ks", [2, 4, 8])
@pytest.mark.parametrize("cols", [16, 32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(1, 128, 2048), (37, 300, 2100), (130, 640, 4000)])
def test_k_split_over_a_cluster(cuda_device, ks, cols, M, N, K):
    Problem(M, N, K, seed=ks).check(tile=capi.scaled_tile(cols, 1, ks))


@pytest.mark.parametrize("bm,bn", list(itertools.product((1, 128), (1, 128))))
def test_k_split_scale_blocks(cuda_device, bm, bn):
    Problem(60, 400, 1500, bm=bm, bn=bn, seed=5).check(tile=capi.scaled_tile(64, 1, 4))


@pytest.mark.parametrize("tile", [0] + PAIR + SINGLE[:2] + [capi.scaled_tile(64, 1, 2)])
def test_integers_are_exact(cuda_device, tile):
    """Integers up to 3, scales that are powers of two between 1/8 and 4: every sum is a multiple of 2^-6 and at most
    9 * 512 * 16 < 2^17, so 24 bits hold it and any order of summation gives the same bits."""
    p = Problem(270, 600, 512, te=ck.CKB_F32, seed=11, integers=True)
    assert torch.equal(p.run(tile=tile).double(), p.ref)


def test_strides_and_unaligned_output(cuda_device):
    p = Problem(70, 330, 600, pad=48, k_first=True, seed=13)
    for tile in (capi.scaled_tile(256, 2), capi.scaled_tile(192, 2), capi.scaled_tile(224, 2), capi.scaled_tile(64, 1)):
        p.check(tile=tile, lde=333, offset=1)
        p.check(tile=tile, lde=344, offset=8)


def test_one_scale_for_a_whole_tensor(cuda_device):
    """Scale strides of zero."""
    p = Problem(150, 200, 300, seed=17)
    p.sa = torch.full((1, 1), 0.5, device="cuda").expand(p.sa.shape)
    p.sb = torch.full((1, 1), 0.25, device="cuda").expand(p.sb.shape)
    p.ref, p.mag = L.product64(p.a[:, :300].float(), p.sa, p.b[:, :300].float().t(), p.sb, 1, 128)
    p.check()


def test_infinities_nans_and_zero_scales_stay_in_their_rows(cuda_device):
    """A NaN in A, an infinite or zero scale reach their row (column) of E only."""
    for tile in (capi.scaled_tile(256, 2), capi.scaled_tile(64, 1)):
        p = Problem(140, 260, 384, te=ck.CKB_F32, seed=19)
        want = p.ref.clone()
        p.a[3, 5] = float("nan")
        p.sa[9, 1] = float("inf")
        p.sa[11] = 0.0
        e = p.run(tile=tile)
        assert torch.isnan(e[3]).all() and not torch.isfinite(e[9]).any()
        assert (e[11] == 0).all()
        keep = [i for i in range(140) if i not in (3, 9, 11)]
        L.check_product(e[keep], want[keep], p.mag[keep], 384)


def test_larger_shapes_in_one_launch_of_many_tiles(cuda_device):
    for M, N, K in ((3000, 2500, 640), (1025, 8200, 256)):
        Problem(M, N, K, seed=23).check()


# ---- groups of rows ------------------------------------------------------------------------------
class Rows:
    def __init__(self, sizes, N, K, rows=None, lb=COL, te=ck.CKB_BF16, bn=128, seed=0, offsets=None):
        g = L.gen(seed)
        self.groups, self.rows, self.N, self.K, self.lb, self.bn, self.te = len(sizes), rows or max(1, sum(sizes)), N, K, lb, bn, te
        kb = -(-K // 128)
        self.a = L.eight_bit(g, (self.rows, K), E4, pad16(K))
        shape = (self.groups, N, K) if lb == COL else (self.groups, K, N)
        self.b = L.eight_bit(g, shape, E4, pad16(shape[2]))
        self.sa, self.sb = L.scales(g, (self.rows, kb)), L.scales(g, (self.groups, kb, -(-N // bn)))
        self.offsets = offsets if offsets is not None else [0] + list(itertools.accumulate(sizes))

    def run(self, tile=0, offsets=None):
        off = torch.tensor(offsets or self.offsets, dtype=torch.int32, device="cuda")
        dtype = L.WIDE[self.te]
        e = torch.full((self.rows, self.N), float("nan"), dtype=dtype, device="cuda")
        op = ck.DeviceGroupedGemmABScale(ck.CKB_GROUP_ROWS, E4, E4, self.te, ROW, self.lb, 1, self.bn, tile_config=tile)
        arg = op.MakeArgument(self.a.data_ptr(), self.b.data_ptr(), self.sa.data_ptr(), self.sb.data_ptr(), e.data_ptr(), off.data_ptr(),
                              self.groups, self.rows, self.N, self.K, self.a.stride(0), self.b.stride(1), self.N, self.sa.stride(),
                              self.sb.stride()[:0:-1], self.b.stride(0), self.sb.stride(0))
        assert op.IsSupportedArgument(arg), capi.last_error()
        L.run(op, arg)
        return e

    def check(self, tile=0):
        e = self.run(tile)
        at = torch.zeros(self.rows, dtype=torch.bool, device="cuda")
        for g in range(self.groups):
            lo, hi = self.offsets[g], self.offsets[g + 1]
            at[lo:hi] = True
            if hi > lo:
                b = self.b[g][:, :self.K].t() if self.lb == COL else self.b[g][:, :self.N]
                ref, mag = L.product64(self.a[lo:hi, :self.K].float(), self.sa[lo:hi], b.float(), self.sb[g], 1, self.bn)
                L.check_product(e[lo:hi], ref, mag, self.K)
        assert torch.isnan(e[~at]).all(), "rows outside every group were written"


GROUP_TILES = [0, capi.scaled_tile(256, 2), capi.scaled_tile(192, 2), capi.scaled_tile(16, 1), capi.scaled_tile(128, 1)]


@pytest.mark.parametrize("tile", GROUP_TILES)
@pytest.mark.parametrize("sizes", [[1], [0, 5, 0, 0, 131, 1, 0], [300, 17, 260], [0, 0, 0], [0, 700]])
def test_groups_of_rows(cuda_device, tile, sizes):
    Rows(sizes, 300, 400, rows=sum(sizes) + 5, seed=len(sizes)).check(tile)


@pytest.mark.parametrize("lb,bn", list(itertools.product((ROW, COL), (1, 128))))
@pytest.mark.parametrize("tile", GROUP_TILES)
def test_groups_of_rows_layouts(cuda_device, lb, bn, tile):
    Rows([70, 0, 200, 3], 272, 384, rows=300, lb=lb, bn=bn, seed=2).check(tile)


@pytest.mark.parametrize("groups", [64, 1000, 1024])
def test_many_groups(cuda_device, groups):
    sizes = [(7 * g) % 4 for g in range(groups)]
    Rows(sizes, 128, 128, rows=sum(sizes) + 1, seed=groups).check()


def test_groups_that_do_not_start_at_row_zero(cuda_device):
    Rows([10, 20], 256, 256, rows=64, seed=4, offsets=[17, 27, 47]).check()


def test_wild_offsets_stay_inside_the_tensors(cuda_device):
    """Offsets out of range or decreasing are clipped: rows that no clipped group covers keep their values."""
    p = Rows([20, 20, 20], 256, 256, rows=64, seed=6)
    for off in ([-5, 10, 1 << 30, 1 << 30], [64, 64, 64, 64], [-(1 << 31), -7, -1, 0], [40, 20, 10, 30], [(1 << 31) - 1, -1, 5, 5]):
        e = p.run(offsets=off)
        clip = lambda v, lo: min(max(v, lo), 64)
        covered = torch.zeros(64, dtype=torch.bool, device="cuda")
        for g in range(3):
            lo = clip(off[g], 0)
            covered[lo:clip(off[g + 1], lo)] = True
        assert torch.isnan(e[~covered]).all() and torch.isfinite(e[covered]).all()


# ---- groups of K blocks --------------------------------------------------------------------------
@pytest.mark.parametrize("tile", [0, capi.scaled_tile(256, 2), capi.scaled_tile(128, 2), capi.scaled_tile(128, 1)])
@pytest.mark.parametrize("blocks", [[1], [0, 2, 0, 3, 1], [0, 0], [5, 0]])
@pytest.mark.parametrize("te", [ck.CKB_F32, ck.CKB_BF16])
def test_groups_of_k_blocks(cuda_device, tile, blocks, te):
    M, N, groups, total = 272, 336, len(blocks), sum(blocks) + 1
    g = L.gen(9)
    a, b = L.eight_bit(g, (total * 128, M), E5), L.eight_bit(g, (total * 128, N), E4)
    sa, sb = L.scales(g, (total, M)), L.scales(g, (total, N))
    off = torch.tensor([0] + list(itertools.accumulate(blocks)), dtype=torch.int32, device="cuda")
    e = torch.full((groups, M, N), float("nan"), dtype=L.WIDE[te], device="cuda")
    op = ck.DeviceGroupedGemmABScale(ck.CKB_GROUP_K_BLOCKS, E5, E4, te, COL, ROW, 1, 1, tile_config=tile)
    arg = op.MakeArgument(a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(), e.data_ptr(), off.data_ptr(), groups, M, N,
                          total * 128, M, N, N, sa.stride()[::-1], sb.stride()[::-1], 0, 0, M * N)
    assert op.IsSupportedArgument(arg), capi.last_error()
    L.run(op, arg)
    for i, n in enumerate(blocks):
        lo = int(off[i])
        r, t = slice(lo * 128, (lo + n) * 128), slice(lo, lo + n)
        if n == 0:
            assert (e[i] == 0).all()
        else:
            ref, mag = L.product64(a[r].float().t(), sa[t].t(), b[r].float(), sb[t], 1, 1)
            L.check_product(e[i], ref, mag, n * 128)
