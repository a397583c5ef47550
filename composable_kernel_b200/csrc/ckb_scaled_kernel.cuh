// The 8-bit product with block scales:
//   E[m,n] = sum over K blocks kb of 128:  sa[m,kb] * sb[n,kb] * sum over k in kb of A[m,k] * B[k,n]
//
// The scales are arbitrary 32-bit numbers, so they cannot ride in the tensor core: every K block is multiplied into a
// fresh accumulator in tensor memory, and the epilogue warps add it, scaled, to 32-bit sums that they keep in
// registers for the whole tile.
//   warp 0     TMA producer: a ring of stages, each one K block (128 bytes of K) of the U tile (128 rows per CTA) and
//              the V tile (BN / CG rows per CTA), 128-byte swizzle, K-major or MN-major as the operand lies
//   warp 1     one thread issues four tcgen05.mma (kind::f8f6f4, 32 bytes of K each) per K block into one of two
//              tensor-memory accumulators and ONE commit per K block: its barrier tells the producer that the stage is
//              free and the epilogue warps that the accumulator is complete
//   warps 4-11 two per lane quarter, each half of the columns: load the accumulator, release it, fused multiply-add
//              into the sums (two values per instruction).  The scales of the next two K blocks are on their way
//              while one is added.
// Per 256 x 256 tile of a CTA pair and K block the tensor pipe needs 512 cycles; an epilogue warp needs four loads of
// 32 columns and 64 packed multiply-adds, about 350, so the tensor pipe stays the limit while loads come in time
// (32 KB per CTA and K block = 64 bytes per cycle, just under what L2 delivers to all SMs at once).
//
// Where the scales come from (VMODE).  A scale of the U side is one number per lane or per tile; on the V side:
//   VMODE 0  one scale per 128 columns: a chunk of 16 columns has one factor per lane, in a register
//   VMODE 1  one scale per column, U scale uniform over the tile: their products are staged in shared memory
//   VMODE 2  one scale per column and one per lane: two packed operations per pair of values
//
// CTA pairs (CG = 2, BN = 256): as in ckb_kernel.cuh - the leader issues tcgen05.mma.cta_group::2 for both CTAs, each
// CTA loads its own 128 U rows and its own half of the V rows (no load has more than one destination), all bytes are
// counted on the leader's barrier, the commit fans out to both.
// Single CTAs (CG = 1, BN = 16 .. 128): U = columns of B, V = rows of A; few rows then cost few columns instead of a
// padded 128-row tile.  With ksplit = 2, 4 or 8 a cluster of as many CTAs shares the K blocks of one tile: each CTA
// pushes its sums to the CTA that owns the columns (st.shared::cluster), a cluster barrier, and the owners add the
// slices in slice order (deterministic) and store.
//
// Every wait is bounded as in ckb_kernel.cuh; after a wait gave up all roles drain and leave.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ckb_kernel.cuh"
#include "ckb_scaled_plan.h"

namespace ckb {

struct ScaledParams
{
    CUtensorMap tm_u, tm_v;
    ScaledTiles tiles;
    const float *su, *sv;
    int64_t su_row, su_kb, su_group; // elements from one scale to the next: row block, K block, group
    int64_t sv_row, sv_kb, sv_group;
    int32_t u_shift, v_shift;        // log2 of the rows per scale: 0 or 7
    void* e;
    int64_t lde, e_group;
    int32_t e_dtype;                 // CKB_F16 / CKB_BF16 / CKB_F32
    int32_t e_vec;                   // rows of E may be written 16 bytes at a time
    int32_t num_tiles;               // GROUP_ROWS: taken from the offsets
    int32_t num_units;               // CTAs (pairs, clusters) of the grid
    int32_t u_mn, v_mn;              // operand is MN-major
    int32_t u_batched, v_batched;    // operand has a third dimension: the group
    int32_t v_box_rows;              // rows of a K-major V box
    uint32_t idesc;
    const int32_t* offsets;
    uint64_t wait_limit_ns;
    uint32_t* status;
};

// Warps 0-3 (producer, MMA issuer, two that only take part in the barriers) form one warpgroup, the epilogue warps two
// more, so that registers can be dealt out unevenly: 128 sums per lane (BN = 256) next to a chunk of 32 accumulator
// columns, addresses and scales do not fit the 168 that twelve warps get at launch.  72 + 216 + 216 = 3 x 168.
constexpr int SCALED_EPI_WARP0 = 4;
constexpr int SCALED_THREADS   = 32 * (SCALED_EPI_WARP0 + NUM_EPI_WARPS);
constexpr int SCALED_REGS_LOW = 72, SCALED_REGS_HIGH = 216;
static_assert(SCALED_REGS_LOW + 2 * SCALED_REGS_HIGH == 3 * 168, "the shares add up to what the block is launched with");

template <int BN, int CG>
struct ScaledSmem
{
    static constexpr int U_BYTES     = 128 * BK_BYTES;
    static constexpr int V_BYTES     = (BN / CG) * BK_BYTES;
    static constexpr int STAGE_BYTES = U_BYTES + V_BYTES;
    // CG = 2: 4 KB per epilogue warp through which rows of E leave in whole lines.
    // CG = 1: the slices of a K split, BN columns x 128 rows of 32 bits.
    static constexpr int OUT_BYTES = CG == 2 ? NUM_EPI_WARPS * 4096 : BN * 512;
    static constexpr int STAGES    = CG == 2 ? 5 : BN == 128 ? 4 : BN == 64 ? 6 : 8;
    static constexpr int OUT_OFFSET = STAGES * STAGE_BYTES;
    static constexpr int HALF       = BN / 2; // columns of an epilogue warp
    static constexpr int COL_OFFSET = OUT_OFFSET + OUT_BYTES; // column scales: two buffers per epilogue warp
    static constexpr int GRP_OFFSET = COL_OFFSET + NUM_EPI_WARPS * 2 * (HALF < 32 ? 32 : HALF) * 4;
    static constexpr int BAR_OFFSET = GRP_OFFSET + (3 * CKB_SCALED_MAX_GROUPS + 4) * 4;
    // full[STAGES], done[STAGES], acc_empty[2], drain
    static constexpr int NUM_BARS    = 2 * STAGES + 3;
    static constexpr int MISC_OFFSET = BAR_OFFSET + NUM_BARS * 8;
    static constexpr int TOTAL       = MISC_OFFSET + 16;
    static constexpr int DYN_BYTES   = TOTAL + 1024; // slack to align the base to 1024 B
};

template <typename T>
__device__ __forceinline__ T scaled_out(float v);
template <>
__device__ __forceinline__ float scaled_out<float>(float v)
{
    return v;
}
template <>
__device__ __forceinline__ __half scaled_out<__half>(float v)
{
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 scaled_out<__nv_bfloat16>(float v)
{
    return __float2bfloat16_rn(v);
}

// Rows of E of one warp (32 rows x ncols columns, one row per lane in `acc`) through the warp's 4 KB of shared memory,
// so that a store instruction writes four runs of 128 contiguous bytes instead of 32 pieces of 16 a pitch apart.
template <typename T, int HALF>
__device__ __forceinline__ void store_rows(const uint64_t (&acc)[HALF / 2], uint8_t* tile, T* e, int64_t lde, int row0,
                                           int row_end, int col0, int col_end, int ncols, bool vec, int lane)
{
    constexpr int PER  = 16 / sizeof(T);  // values of a 16-byte piece
    constexpr int PASS = 8 * PER;         // columns of a pass: 128 bytes
    static_assert(HALF % PASS == 0, "a pass is 128 bytes wide");
#pragma unroll
    for(int p = 0; p < HALF / PASS; ++p)
    {
        if(p * PASS >= ncols)
            break;
        __syncwarp();
#pragma unroll
        for(int c = 0; c < 8; ++c)
        {
            alignas(16) T piece[PER];
#pragma unroll
            for(int i = 0; i < PER; i += 2)
            {
                float lo, hi;
                unpack_f32x2(acc[(p * PASS + c * PER + i) / 2], lo, hi);
                piece[i]     = scaled_out<T>(lo);
                piece[i + 1] = scaled_out<T>(hi);
            }
            *reinterpret_cast<uint4*>(tile + lane * 128 + ((c ^ (lane & 7)) * 16)) = *reinterpret_cast<const uint4*>(piece);
        }
        __syncwarp();
        const int c = lane & 7;
        const int n = p * PASS + c * PER; // first column of this lane's pieces
        if(n < ncols)
        {
#pragma unroll
            for(int i = 0; i < 8; ++i)
            {
                const int r = i * 4 + (lane >> 3);
                if(row0 + r >= row_end)
                    continue;
                const uint4 v = *reinterpret_cast<const uint4*>(tile + r * 128 + ((c ^ (r & 7)) * 16));
                T* dst        = e + static_cast<int64_t>(row0 + r) * lde + col0 + n;
                if(vec && col0 + n + PER <= col_end)
                    *reinterpret_cast<uint4*>(dst) = v;
                else
                {
                    const T* w = reinterpret_cast<const T*>(&v);
#pragma unroll
                    for(int j = 0; j < PER; ++j)
                        if(col0 + n + j < col_end)
                            dst[j] = w[j];
                }
            }
        }
    }
}

// The sums of a lane are a column of E (U = columns of B): for every row of E the lanes write neighbouring columns.
template <typename T, int HALF>
__device__ __forceinline__ void store_cols(const uint64_t (&acc)[HALF / 2], T* e, int64_t lde, int u, int u_end, int v0,
                                           int v_end, int ncols)
{
    if(u >= u_end)
        return;
#pragma unroll
    for(int c = 0; c < HALF; c += 2)
    {
        float lo, hi;
        unpack_f32x2(acc[c / 2], lo, hi);
        if(c < ncols && v0 + c < v_end)
            e[static_cast<int64_t>(v0 + c) * lde + u] = scaled_out<T>(lo);
        if(c + 1 < ncols && v0 + c + 1 < v_end)
            e[static_cast<int64_t>(v0 + c + 1) * lde + u] = scaled_out<T>(hi);
    }
}

// Owner side of a K split: sums column part `rank` over the slices, in slice order, and stores it.
template <typename T>
__device__ __forceinline__ void store_slices(const float* part, int pw, int slices, T* e, int64_t lde, int u, int u_end,
                                             int v0, int v_end, int row, int first)
{
    if(u >= u_end)
        return;
    for(int c = first; c < pw; c += 2)
    {
        if(v0 + c >= v_end)
            break;
        float sum = part[c * 128 + row];
        for(int s = 1; s < slices; ++s)
            sum += part[(s * pw + c) * 128 + row];
        e[static_cast<int64_t>(v0 + c) * lde + u] = scaled_out<T>(sum);
    }
}

template <int BN, int CG, int VMODE>
__global__ void __launch_bounds__(SCALED_THREADS, 1) scaled_kernel(const __grid_constant__ ScaledParams P)
{
    using L                     = ScaledSmem<BN, CG>;
    constexpr int STAGES        = L::STAGES;
    constexpr int HALF          = L::HALF;
    constexpr uint32_t ACC_COLS = 2 * BN; // 32 .. 512, a power of two
    constexpr int CHUNK         = HALF < 32 ? HALF : 32;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr  = smem_u32(smem_raw);
    const uint32_t base_addr = (raw_addr + 1023u) & ~1023u;
    uint8_t* smem            = smem_raw + (base_addr - raw_addr);

    const uint32_t bar_base  = base_addr + L::BAR_OFFSET;
    auto full_bar            = [&](int s) { return bar_base + 8u * s; };
    auto done_bar            = [&](int s) { return bar_base + 8u * (STAGES + s); };
    auto acc_empty_bar       = [&](int a) { return bar_base + 8u * (2 * STAGES + a); };
    const uint32_t drain_bar = bar_base + 8u * (2 * STAGES + 2);
    volatile uint32_t* misc  = reinterpret_cast<volatile uint32_t*>(smem + L::MISC_OFFSET);
    // misc[0] = TMEM base address, misc[1] = abort flag, misc[2] = constant 0, misc[3] = number of tiles (GROUP_ROWS)
    int32_t* grp_start = reinterpret_cast<int32_t*>(smem + L::GRP_OFFSET);
    int32_t* grp_row0  = grp_start + CKB_SCALED_MAX_GROUPS + 4;
    int32_t* grp_row1  = grp_row0 + CKB_SCALED_MAX_GROUPS;

    const int warp           = threadIdx.x >> 5;
    const int lane           = threadIdx.x & 31;
    const int ksplit         = CG == 1 ? P.tiles.ksplit : 1;
    const uint32_t cta_rank  = (CG == 2 || ksplit > 1) ? cluster_ctarank() : 0u;
    const bool is_leader     = CG == 1 || cta_rank == 0;
    const int unit           = static_cast<int>(blockIdx.x) / (CG == 2 ? 2 : ksplit);

    if(threadIdx.x == 0)
    {
        for(int s = 0; s < STAGES; ++s)
        {
            mbar_init(full_bar(s), 1); // the (leader's) producer arrival + all bytes of the stage
            mbar_init(done_bar(s), 1); // one tcgen05.commit arrival
        }
        for(int a = 0; a < 2; ++a)
            mbar_init(acc_empty_bar(a), NUM_EPI_WARPS * CG);
        mbar_init(drain_bar, 1);
        misc[1] = 0;
        misc[2] = 0;
        misc[3] = 0;
        fence_mbar_init();
    }
    if(warp == 1)
    {
        if constexpr(CG == 2)
        {
            tmem_alloc_pair(smem_u32(const_cast<uint32_t*>(&misc[0])), ACC_COLS);
            tmem_relinquish_pair();
        }
        else
        {
            tmem_alloc(smem_u32(const_cast<uint32_t*>(&misc[0])), ACC_COLS);
            tmem_relinquish();
        }
    }
    tc_fence_before_sync();
    if(CG == 2 || ksplit > 1)
        cluster_sync_all(); // the peers' barriers and shared memory must exist before anything is sent there
    else
        __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = misc[0];
    grid_dependency_wait();
    grid_launch_dependents();

    int num_tiles = P.num_tiles;
    if(P.tiles.mode == SCALED_GROUP_ROWS)
    {
        // tiles of every group, then their running sum (one warp, 32 groups at a time)
        for(int g = threadIdx.x; g < P.tiles.groups; g += SCALED_THREADS)
            scaled_group_span(P.offsets, g, P.tiles.swapped ? P.tiles.ext_v : P.tiles.ext_u, &grp_row0[g], &grp_row1[g]);
        __syncthreads();
        if(warp == 0)
        {
            const int other = P.tiles.swapped ? P.tiles.tiles_u : P.tiles.tiles_v;
            int total       = 0;
            for(int g0 = 0; g0 < P.tiles.groups; g0 += 32)
            {
                const int g = g0 + lane;
                int n       = g < P.tiles.groups ? scaled_group_tiles(P.tiles, grp_row1[g] - grp_row0[g]) * other : 0;
                const int own = n;
#pragma unroll
                for(int d = 1; d < 32; d <<= 1)
                {
                    const int up = __shfl_up_sync(0xffffffffu, n, d);
                    if(lane >= d)
                        n += up;
                }
                if(g < P.tiles.groups)
                    grp_start[g] = total + n - own;
                total += __shfl_sync(0xffffffffu, n, 31);
            }
            if(lane == 0)
            {
                grp_start[P.tiles.groups] = total;
                misc[3]                   = static_cast<uint32_t>(total);
            }
        }
        __syncthreads();
        num_tiles = static_cast<int>(misc[3]);
    }
    auto item_of = [&](int t) -> ScaledItem {
        if(P.tiles.mode == SCALED_GROUP_ROWS)
            return scaled_group_item(P.tiles, t, grp_start, grp_row0, grp_row1);
        ScaledItem it = scaled_item(P.tiles, t, P.offsets);
        if(CG == 1 && ksplit > 1)
        {
            // slice `rank` of the K blocks, lengths differing by one at most
            const int n = it.kb1 - it.kb0, r = static_cast<int>(cta_rank);
            const int a = it.kb0 + static_cast<int>(static_cast<int64_t>(n) * r / ksplit);
            it.kb1      = it.kb0 + static_cast<int>(static_cast<int64_t>(n) * (r + 1) / ksplit);
            it.kb0      = a;
        }
        return it;
    };

    WaitCtx wc{&misc[1], P.wait_limit_ns, P.status};
    const int half_cols = CG == 2 ? P.tiles.width >> 1 : HALF; // columns of an epilogue warp in this launch

    if(warp < SCALED_EPI_WARP0)
    {
    if constexpr(BN >= 128)
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(SCALED_REGS_LOW));
    if(warp == 0)
    {
        // ------------------------------------------------------------------ TMA producer
        if(lane < 2)
            tma_prefetch_desc(lane == 0 ? &P.tm_u : &P.tm_v);
        int stage           = 0;
        uint32_t phase      = 0;
        int loads           = 0;
        bool ok             = true;
        const uint32_t bar0 = (CG == 2) ? mapa_shared(full_bar(0), 0) : full_bar(0);
        // lane 0 loads the U box, lane 1 the V box
        const bool is_v      = lane == 1;
        const bool mn        = is_v ? P.v_mn != 0 : P.u_mn != 0;
        const bool batched   = is_v ? P.v_batched != 0 : P.u_batched != 0;
        const CUtensorMap* m = is_v ? &P.tm_v : &P.tm_u;
        // an MN-major V box always spans 128 columns (its smem tile has room for them: BN / CG = 128)
        const uint32_t stage_tx = CG * (L::U_BYTES + (P.v_mn ? 128 : P.v_box_rows) * BK_BYTES);
        for(int t = unit; ok && t < num_tiles; t += P.num_units)
        {
            const ScaledItem it = item_of(t);
            const int row       = is_v ? it.v0 + static_cast<int>(CG == 2 ? cta_rank : 0) * half_cols
                                       : it.u0 + static_cast<int>(CG == 2 ? cta_rank : 0) * 128;
            for(int kb = it.kb0; kb < it.kb1; ++kb)
            {
                ok = bounded_wait(done_bar(stage), phase ^ 1u, wc, WAIT_EMPTY);
                ok = __all_sync(0xffffffffu, ok);
                if(!ok)
                    break;
                if(is_leader && lane == 0)
                    mbar_arrive_expect_tx(full_bar(stage), stage_tx);
                if(lane < 2)
                {
                    const uint32_t dst = base_addr + stage * L::STAGE_BYTES + (is_v ? L::U_BYTES : 0);
                    const uint32_t bar = bar0 + 8u * stage;
                    const int c0 = mn ? row : kb * SCALED_BLOCK, c1 = mn ? kb * SCALED_BLOCK : row;
                    if(batched)
                    {
                        if constexpr(CG == 2)
                            tma_load_3d_pair(dst, m, bar, c0, c1, it.group);
                        else
                            tma_load_3d(dst, m, bar, c0, c1, it.group);
                    }
                    else
                    {
                        if constexpr(CG == 2)
                            tma_load_2d_pair(dst, m, bar, c0, c1);
                        else
                            tma_load_2d(dst, m, bar, c0, c1);
                    }
                }
                __syncwarp();
                ++loads;
                if(++stage == STAGES)
                {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        // Do not leave while a bulk copy may still write shared memory (see ckb_kernel.cuh).
        if(is_leader && lane == 0)
            for(int s = 0; s < STAGES && s < loads; ++s)
            {
                const int last_fill = ((loads - 1 - s) / STAGES) * STAGES + s;
                WaitCtx drain{&misc[2], kDrainLimitNs, P.status};
                bounded_wait(full_bar(s), static_cast<uint32_t>(last_fill / STAGES) & 1u, drain, WAIT_DRAIN);
            }
        __syncwarp();
    }
    else if(warp == 1)
    {
        // ------------------------------------------------------------------ MMA issuer
        if(lane == 0 && is_leader)
        {
            int stage       = 0;
            uint32_t phase  = 0;
            uint32_t iter   = 0; // K blocks so far
            bool ok         = true;
            bool issued_any = false;
            const uint64_t u_const = P.u_mn ? make_smem_desc_mn_sw128(0, 128 * BK_BYTES) : make_smem_desc_k_sw128(0);
            const uint64_t v_const = P.v_mn ? make_smem_desc_mn_sw128(0, 128 * BK_BYTES) : make_smem_desc_k_sw128(0);
            const uint32_t u_hi = static_cast<uint32_t>(u_const >> 32), v_hi = static_cast<uint32_t>(v_const >> 32);
            const uint32_t u_step = P.u_mn ? (32 * BK_BYTES) >> 4 : 32 >> 4;
            const uint32_t v_step = P.v_mn ? (32 * BK_BYTES) >> 4 : 32 >> 4;
            for(int t = unit; ok && t < num_tiles; t += P.num_units)
            {
                const ScaledItem it = item_of(t);
                for(int kb = it.kb0; kb < it.kb1; ++kb, ++iter)
                {
                    const int acc = iter & 1;
                    ok = bounded_wait(acc_empty_bar(acc), ((iter >> 1) & 1u) ^ 1u, wc, WAIT_TMEM_EMPTY) &&
                         bounded_wait(full_bar(stage), phase, wc, WAIT_FULL);
                    if(!ok)
                        break;
                    tc_fence_after_sync();
                    const uint32_t u_addr = base_addr + stage * L::STAGE_BYTES;
                    uint32_t u_lo         = static_cast<uint32_t>(u_const) | ((u_addr & 0x3FFFFu) >> 4);
                    uint32_t v_lo         = static_cast<uint32_t>(v_const) | (((u_addr + L::U_BYTES) & 0x3FFFFu) >> 4);
                    const uint32_t d      = tmem_base + acc * BN;
#pragma unroll
                    for(int k = 0; k < 4; ++k)
                    {
                        if constexpr(CG == 2)
                            mma_f8_ss_pair_split(d, u_lo, u_hi, v_lo, v_hi, P.idesc, k != 0);
                        else
                            mma_f8_ss_split(d, u_lo, u_hi, v_lo, v_hi, P.idesc, k != 0);
                        u_lo += u_step;
                        v_lo += v_step;
                    }
                    issued_any = true;
                    if constexpr(CG == 2)
                        mma_commit_pair_mc(done_bar(stage), 3);
                    else
                        mma_commit(done_bar(stage));
                    if(++stage == STAGES)
                    {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            // Every MMA issued must be finished before the tensor memory is freed.
            if(issued_any)
            {
                if constexpr(CG == 2)
                    mma_commit_pair(drain_bar);
                else
                    mma_commit(drain_bar);
                WaitCtx drain{&misc[2], kDrainLimitNs, P.status};
                bounded_wait(drain_bar, 0, drain, WAIT_DRAIN);
            }
        }
        __syncwarp();
    }
    }
    else
    {
        if constexpr(BN >= 128)
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SCALED_REGS_HIGH));
        // ------------------------------------------------------------------ epilogue warps
        const int quarter = warp & 3, half = (warp - SCALED_EPI_WARP0) >> 2;
        const int row     = quarter * 32 + lane; // lane of the accumulator
        const int col     = half * half_cols;    // first column of this warp
        const uint32_t taddr0  = tmem_base + col + (static_cast<uint32_t>(quarter * 32) << 16);
        const uint32_t empty0  = (CG == 2) ? mapa_shared(acc_empty_bar(0), 0) : acc_empty_bar(0);
        constexpr int CV       = (HALF + 31) / 32;
        constexpr int CBUF     = HALF < 32 ? 32 : HALF;
        float* colbuf          = reinterpret_cast<float*>(smem + L::COL_OFFSET) + (warp - SCALED_EPI_WARP0) * 2 * CBUF;
        uint8_t* out_tile      = smem + L::OUT_OFFSET + (warp - SCALED_EPI_WARP0) * 4096;
        uint64_t acc[HALF / 2];
        float su_r[2], lo_r[2], hi_r[2], cv_r[2][CV];
        const float *su_p = nullptr, *sv_p = nullptr, *sv_hi_p = nullptr;
        bool su_on = false;
        uint32_t cv_on = 0;
        int hi_from = 0; // VMODE 0: columns (of the warp) from here on belong to the second scale block
        ScaledItem it{};

        // scales of K block `kb` into slot j (zeros beyond the item or outside the matrix: never used or never stored)
        auto load_scales = [&](int j, int kb) {
            const bool in = kb < it.kb1;
            su_r[j]       = in && su_on ? __ldg(su_p + kb * P.su_kb) : 0.f;
            if constexpr(VMODE == 0)
            {
                lo_r[j] = in && cv_on != 0 ? __ldg(sv_p + kb * P.sv_kb) : 0.f;
                hi_r[j] = in && cv_on > 1 ? __ldg(sv_hi_p + kb * P.sv_kb) : lo_r[j];
            }
            else
            {
#pragma unroll
                for(int q = 0; q < CV; ++q)
                    cv_r[j][q] = in && (cv_on >> q & 1u) ? __ldg(sv_p + q * 32 * P.sv_row + kb * P.sv_kb) : 0.f;
            }
        };
        auto open_item = [&](int t) {
            it          = item_of(t);
            const int u = it.u0 + static_cast<int>(CG == 2 ? cta_rank : 0) * 128 + (VMODE == 1 ? 0 : row);
            su_on       = u < it.u_end;
            su_p        = P.su + it.group * P.su_group + static_cast<int64_t>(u >> P.u_shift) * P.su_row;
            const int v = it.v0 + col;
            if constexpr(VMODE == 0)
            {
                const int b0 = v >> 7;
                sv_p         = P.sv + it.group * P.sv_group + static_cast<int64_t>(b0) * P.sv_row;
                sv_hi_p      = sv_p + P.sv_row;
                hi_from      = ((b0 + 1) << 7) - v;
                cv_on        = v < it.v_end ? (hi_from < half_cols && v + hi_from < it.v_end ? 2u : 1u) : 0u;
            }
            else
            {
                sv_p  = P.sv + it.group * P.sv_group + static_cast<int64_t>(v + lane) * P.sv_row;
                cv_on = 0;
#pragma unroll
                for(int q = 0; q < CV; ++q)
                    if(v + q * 32 + lane < it.v_end && q * 32 + lane < half_cols)
                        cv_on |= 1u << q;
            }
            load_scales(0, it.kb0);
            load_scales(1, it.kb0 + 1);
        };

        int stage      = 0;
        uint32_t phase = 0, iter = 0;
        bool ok        = true;
        if(unit < num_tiles)
            open_item(unit);
        for(int t = unit; ok && t < num_tiles;)
        {
#pragma unroll
            for(int i = 0; i < HALF / 2; ++i)
                acc[i] = 0;
            auto step = [&](int j, int kb) {
                ok = bounded_wait(done_bar(stage), phase, wc, WAIT_TMEM_FULL);
                ok = __all_sync(0xffffffffu, ok);
                if(!ok)
                    return;
                tc_fence_after_sync();
                const float su = su_r[j];
                float s_lo = 0.f, s_hi = 0.f;
                float* cb = colbuf + (iter & 1u) * CBUF;
                if constexpr(VMODE == 0)
                {
                    s_lo = su * lo_r[j];
                    s_hi = su * hi_r[j];
                }
                else
                {
                    // the other buffer was last read two K blocks ago, a __syncwarp in between
#pragma unroll
                    for(int q = 0; q < CV; ++q)
                        cb[q * 32 + lane] = VMODE == 1 ? cv_r[j][q] * su : cv_r[j][q];
                    __syncwarp();
                }
                load_scales(j, kb + 2);
                const uint32_t taddr = taddr0 + (iter & 1u) * BN;
#pragma unroll
                for(int c = 0; c < HALF; c += CHUNK)
                {
                    if(CG == 2 && c >= half_cols)
                        break;
                    const bool whole = CG == 1 || c + 32 <= half_cols; // else 16 columns of the chunk
                    uint32_t v[32];
                    if constexpr(CHUNK == 32)
                    {
                        tmem_ld_32x32b_x16(taddr + c, v);
                        if(whole)
                            tmem_ld_32x32b_x16(taddr + c + 16, v + 16);
                        tmem_ld_wait_regs16(v);
                        if(whole)
                            keep_regs16(v + 16);
                    }
                    else if constexpr(CHUNK == 16)
                    {
                        tmem_ld_32x32b_x16(taddr + c, v);
                        tmem_ld_wait_regs16(v);
                    }
                    else
                    {
                        tmem_ld_32x32b_x8(taddr + c, v);
                        tmem_ld_wait_regs8(v);
                    }
                    if(c + CHUNK >= half_cols)
                    {
                        // everything is in registers: the next but one K block may overwrite the accumulator
                        tc_fence_before_sync();
                        __syncwarp();
                        if(lane == 0)
                        {
                            if constexpr(CG == 2)
                                mbar_arrive_cluster(empty0 + 8u * (iter & 1u));
                            else
                                mbar_arrive(empty0 + 8u * (iter & 1u));
                        }
                    }
#pragma unroll
                    for(int h = 0; h < CHUNK; h += 16)
                    {
                        if(h == 16 && !whole)
                            break;
                        constexpr int N = CHUNK < 16 ? CHUNK : 16;
                        if constexpr(VMODE == 0)
                        {
                            const float s     = c + h >= hi_from ? s_hi : s_lo;
                            const uint64_t s2 = pack_f32x2(s, s);
#pragma unroll
                            for(int i = 0; i < N; i += 2)
                                acc[(c + h + i) / 2] = fma_f32x2(
                                    pack_f32x2(__uint_as_float(v[h + i]), __uint_as_float(v[h + i + 1])), s2, acc[(c + h + i) / 2]);
                        }
                        else
                        {
                            const uint64_t su2 = pack_f32x2(su, su);
#pragma unroll
                            for(int i = 0; i < N; i += 4)
                            {
                                const float4 s4 = *reinterpret_cast<const float4*>(cb + c + h + i);
                                uint64_t p0 = pack_f32x2(__uint_as_float(v[h + i]), __uint_as_float(v[h + i + 1]));
                                uint64_t p1 = pack_f32x2(__uint_as_float(v[h + i + 2]), __uint_as_float(v[h + i + 3]));
                                if constexpr(VMODE == 2)
                                {
                                    p0 = mul_f32x2(p0, su2);
                                    p1 = mul_f32x2(p1, su2);
                                }
                                acc[(c + h + i) / 2]     = fma_f32x2(p0, pack_f32x2(s4.x, s4.y), acc[(c + h + i) / 2]);
                                acc[(c + h + i) / 2 + 1] = fma_f32x2(p1, pack_f32x2(s4.z, s4.w), acc[(c + h + i) / 2 + 1]);
                            }
                        }
                    }
                }
                ++iter;
                if(++stage == STAGES)
                {
                    stage = 0;
                    phase ^= 1u;
                }
            };
            const int kb1 = it.kb1;
            for(int kb = it.kb0; ok && kb < kb1; kb += 2)
            {
                step(0, kb);
                if(ok && kb + 1 < kb1)
                    step(1, kb + 1);
            }
            if(!ok)
                break;
            const ScaledItem cur = it;
            t += P.num_units;
            if(t < num_tiles)
                open_item(t); // the next tile's first scales arrive while this one is stored
            if(CG == 1 && ksplit > 1)
            {
                // hand the sums to the CTAs that own the columns: [slice][column of the part][row]
                const int pw        = BN / ksplit;
                const uint32_t part = base_addr + L::OUT_OFFSET + static_cast<uint32_t>(cta_rank) * pw * 512u + row * 4u;
#pragma unroll
                for(int c = 0; c < HALF; ++c)
                {
                    float lo, hi;
                    unpack_f32x2(acc[c / 2], lo, hi);
                    const int n     = col + c;
                    const int owner = n / pw;
                    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(
                                     mapa_shared(part + static_cast<uint32_t>(n - owner * pw) * 512u, static_cast<uint32_t>(owner))),
                                 "f"(c & 1 ? hi : lo)
                                 : "memory");
                }
                continue; // one tile per cluster: summed below, behind the cluster barrier
            }
            const int64_t e_off = cur.group * P.e_group;
            const int u_row     = cur.u0 + static_cast<int>(CG == 2 ? cta_rank : 0) * 128 + quarter * 32;
            auto store = [&](auto* e) {
                using T = typename std::remove_pointer<decltype(e)>::type;
                if(CG == 1 || P.tiles.swapped)
                    store_cols<T, HALF>(acc, e + e_off, P.lde, u_row + lane, cur.u_end, cur.v0 + col, cur.v_end, half_cols);
                else if constexpr(CG == 2)
                    store_rows<T, HALF>(acc, out_tile, e + e_off, P.lde, u_row, cur.u_end, cur.v0 + col, cur.v_end, half_cols,
                                        P.e_vec != 0, lane);
            };
            if(P.e_dtype == CKB_BF16)
                store(static_cast<__nv_bfloat16*>(P.e));
            else if(P.e_dtype == CKB_F16)
                store(static_cast<__half*>(P.e));
            else
                store(static_cast<float*>(P.e));
        }
    }

    if(CG == 1 && ksplit > 1)
    {
        cluster_sync_all(); // every slice is at its owner (release / acquire at cluster scope)
        if(warp >= SCALED_EPI_WARP0 && misc[1] == 0 && unit < num_tiles)
        {
            const ScaledItem it = item_of(unit);
            const int t = static_cast<int>(threadIdx.x) - 32 * SCALED_EPI_WARP0, row = t & 127;
            const int pw      = BN / ksplit;
            const float* part = reinterpret_cast<const float*>(smem + L::OUT_OFFSET);
            const int v0      = it.v0 + static_cast<int>(cta_rank) * pw;
            auto sum = [&](auto* e) { store_slices(part, pw, ksplit, e, P.lde, it.u0 + row, it.u_end, v0, it.v_end, row, t >> 7); };
            if(P.e_dtype == CKB_BF16)
                sum(static_cast<__nv_bfloat16*>(P.e));
            else if(P.e_dtype == CKB_F16)
                sum(static_cast<__half*>(P.e));
            else
                sum(static_cast<float*>(P.e));
        }
    }

    // ---------------------------------------------------------------------- common exit
    tc_fence_before_sync();
    if constexpr(CG == 2)
        cluster_sync_all(); // the leader's MMAs read the peer's shared memory until the very end
    else
        __syncthreads();
    tc_fence_after_sync();
    if(warp == 1)
    {
        if constexpr(CG == 2)
            tmem_dealloc_pair(tmem_base, ACC_COLS);
        else
            tmem_dealloc(tmem_base, ACC_COLS);
    }
}

} // namespace ckb
