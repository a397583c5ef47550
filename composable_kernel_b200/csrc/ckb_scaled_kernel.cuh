// The 8-bit product with block scales:
//   E[m,n] = sum over K blocks kb of 128:  sa[m,kb] * sb[n,kb] * sum over k in kb of A[m,k] * B[k,n]
//
// The scales are arbitrary 32-bit numbers, so they cannot ride in the tensor core: every K block is multiplied into a
// fresh accumulator in tensor memory, and the epilogue warps add it, scaled, to 32-bit sums that they keep in
// registers for the whole tile.
//   warp 0     TMA producer: a ring of stages, each one K block (128 bytes of K) of the U tile (128 rows per CTA) and
//              the V tile (BN / CG rows per CTA), 128-byte swizzle, K-major or MN-major as the operand lies
//   warp 1     one thread issues four tcgen05.mma (kind::f8f6f4, 32 bytes of K each) per K block into one of two to four
//              tensor-memory accumulators, with ONE wait (data there, accumulator free) and ONE commit per K block: the
//              commit's barrier tells the producer that the stage is free and the epilogue warps that the accumulator is
//              complete.  A wait costs this thread about 80 cycles even if nothing is waited for
//   warps 2, 3 bring the scales into a ring in shared memory
//   warps 4-11 two per lane quarter, each half of the columns: load the accumulator, release it, fused multiply-add
//              into the sums (two values per instruction).  They issue no global loads: a hand-over behind one would
//              wait for it (the first version, which loaded its scales itself and released the accumulator with a
//              cluster-scope release, took 2300 cycles per K block).
// Per 256 x 256 tile of a CTA pair and K block the tensor pipe needs 512 cycles, the copies 32 KB per CTA.
//
// Where the scales come from (VMODE).  A scale of the U side is one number per lane or per tile; on the V side:
//   VMODE 0  one scale per 128 columns: a chunk of 16 columns has one factor per lane, in a register
//   VMODE 1  one scale per column: two packed operations per pair of values, the second on the product of the scales
//
// CTA pairs (CG = 2, BN = 128 .. 256): as in ckb_kernel.cuh - the leader issues tcgen05.mma.cta_group::2 for both CTAs, each
// CTA loads its own 128 U rows and its own half of the V rows (no load has more than one destination), all bytes are
// counted on the leader's barrier, the commit fans out to both.
// Single CTAs (CG = 1, BN = 16 .. 128): U = columns of B, V = rows of A; few rows then cost few columns instead of a
// padded 128-row tile.  With ksplit = 2, 4 or 8 a cluster of as many CTAs shares the K blocks of one tile: each CTA
// pushes its sums to the CTA that owns the columns (st.shared::cluster), a cluster barrier, and the owners add the
// slices in slice order (deterministic) and store.
//
// Measured: 3840 x 4096 x 4096 to bf16 69-76 us back to back (1.7-1.87 PFLOP/s, SM clock 1.8-1.965 GHz; the fp16 product of the
// same size in the same run 74-79 us on small whole numbers, 90-93 on normal ones), 84 us among other passes; 11008 x 4096 x 8190 with a scale per column on
// both sides to f32 480-555 us, the longer the hotter; 4 x 4096 x 4096 8.5 us; 64 groups of 4 rows each with 4096 x 4096
// weights 170 us (6.3 TB/s), 247 rows spread over 64 groups at random 124-150 us (41 to 57 groups have rows, and the weights of
// the others are not read).  The large products are bound by the chain that each epilogue warp goes through per K block (wait,
// scales, tensor-memory load, wait, release): tensor pipe 46 % and issue slots 44 % active, neither full.  The decode forms are
// bound by launch, fill and hand-over, the grouped ones of few rows by the bytes of the weights.
//
// Every wait is bounded as in ckb_kernel.cuh; after a wait gave up all roles leave their loops, and what is still on its way is
// waited for behind the barrier of the exit.
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
    int32_t u_shift;                 // log2 of the rows per scale of U: 0 or 7 (V: an instance each)
    void* e;
    int64_t lde, e_group;
    int32_t e_dtype;                 // CKB_F16 / CKB_BF16 / CKB_F32
    int32_t e_vec;                   // rows of E may be written 16 bytes at a time
    int32_t num_tiles;               // GROUP_ROWS: taken from the offsets
    int32_t num_units;               // CTAs (pairs, clusters) of the grid
    int32_t u_mn, v_mn;              // operand is MN-major
    int32_t u_batched, v_batched;    // operand has a third dimension: the group
    int32_t v_box_rows;              // rows of a K-major V box
    uint32_t test_wait;              // test hook, 0 in use (see scaled_test_wait)
    uint32_t idesc;
    const int32_t* offsets;
    uint64_t wait_limit_ns;
    uint32_t* status;
};

// Warps 0-3 (producer, MMA issuer, two for the scales) form one warpgroup, the epilogue warps two more, so that registers
// can be dealt out unevenly: 128 sums per lane (BN = 256) next to a chunk of 32 accumulator columns, addresses and scales
// do not fit the 168 that twelve warps get at launch, and spills in the first warpgroup cost as much as in the others.
// What the K loop of an epilogue warp costs is its chain of hand-overs, about 190 instructions per K block around 64 packed
// multiply-adds, in which every warp goes through every K block.  Sixteen warps with a quarter of the columns each repeat the
// hand-overs of eight (511 against 436 ns per K block of a 256 x 256 tile), and groups of four K blocks unrolled with fixed
// stages save instructions but not time (424; the loops no longer fit the instruction caches: 365 against 282 at BN = 16).
// Fewer hand-overs per warp (sets of warps that take K blocks in turn) were not tried.
constexpr int SCALED_EPI_WARP0 = 4;

// Words of shared memory beside the barriers
enum
{
    MISC_TMEM,       // base address of the tensor memory
    MISC_ABORT,      // a wait of this CTA gave up
    MISC_COPY_DRAIN, // the wait for copies at the exit gave up
    MISC_TILES,      // number of tiles (GROUP_ROWS)
    MISC_MMA_DRAIN,  // the wait for MMAs at the exit gave up
    MISC_PEER_ABORT, // a wait of the pair's other CTA gave up
    MISC_LOADS,      // [CTA of the pair] stages that its producer filled
    MISC_RELEASES = MISC_LOADS + 2, // [CTA of the pair][epilogue warp] accumulators that it released (~0: for every stage)
    MISC_WORDS    = MISC_RELEASES + 2 * 8
};

template <int BN, int CG>
struct ScaledSmem
{
    static constexpr int EPI_WARPS   = 8;
    static constexpr int THREADS     = 32 * (SCALED_EPI_WARP0 + EPI_WARPS);
    static constexpr bool SPLIT_REGS = BN >= 128;
    // (224 columns with a scale each: 2048 x 2688 x 4096 takes 59 us with 224 registers, which spill, 52.5 with 232; 256 columns
    // spill with 40 registers in the first warpgroup)
    static constexpr int REGS_LOW = BN == 128 ? 72 : BN == 224 ? 40 : 56, REGS_HIGH = BN == 128 ? 216 : BN == 224 ? 232 : 224;
    static_assert(REGS_LOW + 2 * REGS_HIGH == 3 * 168, "the shares add up to what the block is launched with");
    static constexpr int U_BYTES     = 128 * BK_BYTES;
    // (a pair's CTA always has room for 128 rows: an MN-major box is that wide whatever the tile)
    static constexpr int V_BYTES     = (CG == 2 ? 128 : BN) * BK_BYTES;
    static constexpr int STAGE_BYTES = U_BYTES + V_BYTES;
    // CG = 2: 2 KB per epilogue warp through which rows of E leave in whole sectors.
    // CG = 1: the slices of a K split, BN columns x 128 rows of 32 bits.
    static constexpr int OUT_BYTES = CG == 2 ? EPI_WARPS * 2048 : BN * 512;
    static constexpr int STAGES    = CG == 2 ? 5 : BN == 128 ? 4 : BN == 64 ? 6 : 8;
    static constexpr int OUT_OFFSET = STAGES * STAGE_BYTES;
    static constexpr int COLS       = BN / (EPI_WARPS / 4); // columns of an epilogue warp
    // scales: a ring of SLOTS batches of SCALE_BATCH K blocks, 128 of U and up to BN of V for each of them
    static constexpr int SLOTS        = 2;
    static constexpr int SCALE_BATCH  = CG == 2 ? 4 : 8; // K blocks whose scales are handed over together
    static constexpr int V_SCALES     = BN < 32 ? 32 : BN;
    static constexpr int SCALE_WORDS  = 128 + V_SCALES;
    static constexpr int SCALE_OFFSET = OUT_OFFSET + OUT_BYTES;
    static constexpr int GRP_OFFSET   = SCALE_OFFSET + SLOTS * SCALE_BATCH * SCALE_WORDS * 4;
    static constexpr int BAR_OFFSET = GRP_OFFSET + (3 * CKB_SCALED_MAX_GROUPS + 4) * 4;
    // accumulators in tensor memory: as many as fit, four at most
    static constexpr int NUM_ACC     = 4 * BN <= 512 ? 4 : 2;
    static constexpr int ACC_COLS    = NUM_ACC * BN <= 64 ? 64 : NUM_ACC * BN <= 128 ? 128 : NUM_ACC * BN <= 256 ? 256 : 512;
    static_assert(STAGES >= NUM_ACC, "see full_bar");
    // full[STAGES], done[STAGES], scale_full[SLOTS], scale_empty[SLOTS], drain
    static constexpr int NUM_BARS    = 2 * STAGES + 2 * SLOTS + 1;
    static constexpr int MISC_OFFSET = BAR_OFFSET + NUM_BARS * 8;
    static constexpr int TOTAL       = MISC_OFFSET + MISC_WORDS * 4;
    static constexpr int DYN_BYTES   = TOTAL + 1024; // slack to align the base to 1024 B
};

// bounded_wait for the hand-overs of every K block: less code in the loops of the roles (their instructions have to
// stay in the cache together), and the clock, which takes longer to read than most of these waits, only every 1024 polls.
__device__ __forceinline__ bool block_wait(uint32_t bar, uint32_t parity, const WaitCtx& w, uint32_t code)
{
    uint32_t polls = 0;
    uint64_t t0    = 0;
    while(!mbar_try_wait(bar, parity))
    {
        if((++polls & 1023u) != 0)
            continue;
        const uint64_t now = global_timer_ns();
        if(polls == 1024)
            t0 = now;
        if(*w.abort_flag != 0)
            return false;
        if(now - t0 > w.limit_ns || polls > (1u << 30))
        {
            atomicCAS(w.status, 0u, (code << 24) | (blockIdx.x & 0xFFFFFFu));
            *w.abort_flag = 1;
            return false;
        }
    }
    return true;
}

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

// Rows of E leave a warp through its 2 KB of shared memory, 32 rows x 64 bytes at a time, so that a store instruction
// writes eight runs of 64 contiguous bytes instead of pieces a pitch apart.  The 16-byte pieces of a row are permuted so
// that neither side has bank conflicts.
__device__ __forceinline__ uint32_t out_piece(int row, int c) { return row * 64 + ((c ^ ((row >> 1) & 3)) * 16); }

// Writes one pass (columns n0 .. n0 + 64 bytes of the warp's COLS columns) to E.  `dst` is this lane's first piece: row
// lane / 4, columns n0 + (lane % 4) * PER; rows: how many of the warp's 32 rows exist, cols: columns from n0 on that do.
// `whole`: all of them, in 16-byte pieces.
template <typename T>
__device__ __forceinline__ void store_pass(const uint8_t* tile, T* dst, int64_t lde8, int rows, int cols, bool vec, bool whole, int lane)
{
    constexpr int PER = 16 / sizeof(T); // values of a piece
    const int c = lane & 3, n = c * PER;
#pragma unroll
    for(int i = 0; i < 4; ++i, dst += lde8)
    {
        const int r   = i * 8 + (lane >> 2);
        const uint4 v = *reinterpret_cast<const uint4*>(tile + out_piece(r, c));
        if(whole)
            *reinterpret_cast<uint4*>(dst) = v;
        else if(r < rows)
        {
            if(vec && n + PER <= cols)
                *reinterpret_cast<uint4*>(dst) = v;
            else
            {
                const T* w = reinterpret_cast<const T*>(&v);
#pragma unroll
                for(int j = 0; j < PER; ++j)
                    if(n + j < cols)
                        dst[j] = w[j];
            }
        }
    }
}

// FRAG = false: a lane holds its row, columns in order.  FRAG = true: fragments of 8 columns (tmem_ld_16x256b): pair
// 4 g + 2 h + k of a lane = row 16 h + 8 k + lane / 4, columns 8 g + 2 (lane % 4) and the next one.
template <typename T, int COLS, bool FRAG>
__device__ __forceinline__ void store_rows(const uint64_t (&acc)[COLS / 2], uint8_t* tile, T* e, int64_t lde, int row0,
                                           int row_end, int col0, int col_end, bool vec, int lane)
{
    constexpr int PER  = 16 / sizeof(T);
    constexpr int PASS = 4 * PER; // columns of a pass
    static_assert(COLS % 8 == 0, "whole pieces and fragments");
    const int rows     = row_end - row0, cols = col_end - col0;
    const bool whole   = vec && rows >= 32 && cols >= COLS;
    const int64_t lde8 = 8 * lde;
    T* dst             = e + static_cast<int64_t>(row0 + (lane >> 2)) * lde + col0 + (lane & 3) * PER;
#pragma unroll
    for(int n0 = 0; n0 < COLS; n0 += PASS)
    {
        __syncwarp();
        if constexpr(!FRAG)
        {
#pragma unroll
            for(int c = 0; c < 4 && n0 + c * PER < COLS; ++c)
            {
                alignas(16) T piece[PER];
#pragma unroll
                for(int i = 0; i < PER; i += 2)
                {
                    float lo, hi;
                    unpack_f32x2(acc[(n0 + c * PER + i) / 2], lo, hi);
                    piece[i]     = scaled_out<T>(lo);
                    piece[i + 1] = scaled_out<T>(hi);
                }
                *reinterpret_cast<uint4*>(tile + out_piece(lane, c)) = *reinterpret_cast<const uint4*>(piece);
            }
        }
        else
        {
#pragma unroll
            for(int g = n0 / 8; g < (n0 + PASS) / 8 && g < COLS / 8; ++g)
#pragma unroll
                for(int k = 0; k < 4; ++k) // rows 8 k + lane / 4
                {
                    float lo, hi;
                    unpack_f32x2(acc[g * 4 + k], lo, hi);
                    alignas(8) T pair[2] = {scaled_out<T>(lo), scaled_out<T>(hi)};
                    const int byte = ((g * 8 - n0) + 2 * (lane & 3)) * static_cast<int>(sizeof(T));
                    uint8_t* dst   = tile + out_piece(k * 8 + (lane >> 2), byte >> 4) + (byte & 15);
                    if constexpr(sizeof(T) == 4)
                        *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(pair);
                    else
                        *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(pair);
                }
        }
        __syncwarp();
        store_pass<T>(tile, dst + n0, lde8, rows, cols - n0 < COLS - n0 ? cols - n0 : COLS - n0, vec, whole && n0 + PASS <= COLS, lane);
    }
}

// The sums of a lane are a column of E (U = columns of B): for every row of E the lanes write neighbouring columns.
template <typename T, int COLS>
__device__ __forceinline__ void store_cols(const uint64_t (&acc)[COLS / 2], T* e, int64_t lde, int u, int u_end, int v0,
                                           int v_end)
{
    if(u >= u_end)
        return;
    const int rows = v_end - v0;
    T* dst         = e + static_cast<int64_t>(v0) * lde + u;
#pragma unroll
    for(int c = 0; c < COLS; c += 2, dst += 2 * lde)
    {
        float lo, hi;
        unpack_f32x2(acc[c / 2], lo, hi);
        if(c < rows)
            dst[0] = scaled_out<T>(lo);
        if(c + 1 < rows)
            dst[lde] = scaled_out<T>(hi);
    }
}

// Owner side of a K split: sums column part `rank` over the slices, in slice order, and stores it.
template <typename T>
__device__ __forceinline__ void store_slices(const float* part, int pw, int slices, T* e, int64_t lde, int u, int u_end,
                                             int v0, int v_end, int row, int first, int step)
{
    if(u >= u_end)
        return;
    for(int c = first; c < pw; c += step)
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
__global__ void __launch_bounds__(ScaledSmem<BN, CG>::THREADS, 1) scaled_kernel(const __grid_constant__ ScaledParams P)
{
    using L                     = ScaledSmem<BN, CG>;
    constexpr int STAGES        = L::STAGES;
    constexpr int COLS          = L::COLS;
    constexpr int EPI_WARPS     = L::EPI_WARPS;
    constexpr uint32_t ACC_COLS = L::ACC_COLS;
    constexpr int SLOTS         = L::SLOTS;
    constexpr int SCALE_BATCH   = L::SCALE_BATCH;
    constexpr int CHUNK         = COLS < 32 ? COLS : 32;
    constexpr bool STRADDLES    = 128 % COLS != 0; // a warp's columns may touch two blocks of 128
    // Scales per column: with a row per lane every lane reads every column's scale, 512 bytes per four columns and warp,
    // and shared memory takes twice as long as the sums (640 cycles for 128 columns, 365 with a scale per row); in
    // fragments a lane has a quarter of the columns and four rows.
    constexpr bool FRAG         = CG == 2 && VMODE != 0;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr  = smem_u32(smem_raw);
    const uint32_t base_addr = (raw_addr + 1023u) & ~1023u;
    uint8_t* smem            = smem_raw + (base_addr - raw_addr);

    const uint32_t bar_base  = base_addr + L::BAR_OFFSET;
    auto full_bar            = [&](int s) { return bar_base + 8u * s; };
    auto done_bar            = [&](int s) { return bar_base + 8u * (STAGES + s); };
    auto scale_full_bar      = [&](int s) { return bar_base + 8u * (2 * STAGES + s); };
    auto scale_empty_bar     = [&](int s) { return bar_base + 8u * (2 * STAGES + SLOTS + s); };
    const uint32_t drain_bar = bar_base + 8u * (2 * STAGES + 2 * SLOTS);
    float* scale_ring        = reinterpret_cast<float*>(smem + L::SCALE_OFFSET);
    volatile uint32_t* misc  = reinterpret_cast<volatile uint32_t*>(smem + L::MISC_OFFSET);
    int32_t* grp_start = reinterpret_cast<int32_t*>(smem + L::GRP_OFFSET);
    int32_t* grp_row0  = grp_start + CKB_SCALED_MAX_GROUPS + 4;
    int32_t* grp_row1  = grp_row0 + CKB_SCALED_MAX_GROUPS;

    const int warp           = threadIdx.x >> 5;
    const int lane           = threadIdx.x & 31;
    const int ksplit         = CG == 1 ? P.tiles.ksplit : 1;
    const uint32_t cta_rank  = (CG == 2 || ksplit > 1) ? cluster_ctarank() : 0u;
    const bool is_leader     = CG == 1 || cta_rank == 0;
    const int unit           = static_cast<int>(blockIdx.x) / (CG == 2 ? 2 : ksplit);

    // What the exit has to know about both CTAs of a pair goes to the leader.
    auto tell_leader = [&](int word, uint32_t v) {
        if constexpr(CG == 2)
            st_cluster_u32(mapa_shared(base_addr + L::MISC_OFFSET + 4u * word, 0), v);
        else
            misc[word] = v;
    };
    // Barrier of the whole CTA (pair: the leader's MMAs and both producers' copies reach into the other CTA until the end).
    auto exit_barrier = [&]() {
        __syncwarp();
        if constexpr(CG == 2)
            cluster_sync_all();
        else
            asm volatile("bar.sync 0;" ::: "memory"); // (warps come to it at two places)
    };
    // The barrier behind which no role is in its loop any more; true if a wait gave up (the same answer in both CTAs of a pair).
    auto roles_left = [&]() -> bool {
        tc_fence_before_sync();
        exit_barrier();
        return misc[MISC_ABORT] != 0 || (CG == 2 && misc[MISC_PEER_ABORT] != 0);
    };
    auto gave_up = [&]() { // by each role whose wait gave up; MISC_ABORT is set already
        if constexpr(CG == 2)
            if(lane == 0)
                st_cluster_u32(mapa_shared(base_addr + L::MISC_OFFSET + 4u * MISC_PEER_ABORT, cluster_ctarank() ^ 1u), 1u);
    };

    if(threadIdx.x == 0)
    {
        const uint32_t only = P.test_wait >> 2, hook = only == 0 || (only >> (blockIdx.x & 1) & 1) ? P.test_wait & 3u : 0u;
        for(int s = 0; s < STAGES; ++s)
        {
            // the (leader's) producer arrival, all bytes of the stage, and the release of the accumulator that the K block
            // will use: one arrival per epilogue warp (of both CTAs)
            mbar_init(full_bar(s), 1 + EPI_WARPS * CG);
            mbar_init(done_bar(s), 1 + (hook >> 1)); // one tcgen05.commit arrival
        }
        for(int s = 0; s < SLOTS; ++s)
        {
            mbar_init(scale_full_bar(s), 64 + (hook & 1u)); // one arrival per lane of the two scale warps
            mbar_init(scale_empty_bar(s), EPI_WARPS);
        }
        mbar_init(drain_bar, 1);
        fence_mbar_init();
    }
    if(threadIdx.x != MISC_TMEM && threadIdx.x < MISC_WORDS)
        misc[threadIdx.x] = threadIdx.x < MISC_RELEASES ? 0u : ~0u;
    if(warp == 1)
    {
        if constexpr(CG == 2)
        {
            tmem_alloc_pair(smem_u32(const_cast<uint32_t*>(&misc[MISC_TMEM])), ACC_COLS);
            tmem_relinquish_pair();
        }
        else
        {
            tmem_alloc(smem_u32(const_cast<uint32_t*>(&misc[MISC_TMEM])), ACC_COLS);
            tmem_relinquish();
        }
    }
    tc_fence_before_sync();
    if(CG == 2 || ksplit > 1)
        cluster_sync_all(); // the peers' barriers and shared memory must exist before anything is sent there
    else
        __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = misc[MISC_TMEM];
    grid_dependency_wait();
    grid_launch_dependents();

    int num_tiles = P.num_tiles;
    if(P.tiles.mode == SCALED_GROUP_ROWS)
    {
        // tiles of every group, then their running sum (one warp, 32 groups at a time)
        for(int g = threadIdx.x; g < P.tiles.groups; g += L::THREADS)
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
                misc[MISC_TILES]          = static_cast<uint32_t>(total);
            }
        }
        __syncthreads();
        num_tiles = static_cast<int>(misc[MISC_TILES]);
    }
    auto item_of = [&](int t) -> ScaledItem {
        if(P.tiles.mode == SCALED_GROUP_ROWS)
            return scaled_group_item(P.tiles, t, grp_start, grp_row0, grp_row1);
        ScaledItem it = scaled_item(P.tiles, t, P.offsets);
        if(CG == 1 && ksplit > 1)
            scaled_slice(&it, static_cast<int>(cta_rank), ksplit);
        return it;
    };

    WaitCtx wc{&misc[MISC_ABORT], P.wait_limit_ns, P.status};
    constexpr int NUM_ACC = L::NUM_ACC;

    if(warp < SCALED_EPI_WARP0)
    {
    if constexpr(L::SPLIT_REGS)
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::REGS_LOW));
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
        // an MN-major V box always spans 128 columns (its smem tile has room for them: BN / CG = 128)
        const uint32_t stage_tx = CG * (L::U_BYTES + (P.v_mn ? 128 : P.v_box_rows) * BK_BYTES);
        const int pair_rank     = CG == 2 ? static_cast<int>(cta_rank) : 0;
        auto load_box = [&](const CUtensorMap* m, uint32_t dst, uint32_t bar, int c0, int c1, bool batched, int group) {
            if(batched)
            {
                if constexpr(CG == 2)
                    tma_load_3d_pair(dst, m, bar, c0, c1, group);
                else
                    tma_load_3d(dst, m, bar, c0, c1, group);
            }
            else
            {
                if constexpr(CG == 2)
                    tma_load_2d_pair(dst, m, bar, c0, c1);
                else
                    tma_load_2d(dst, m, bar, c0, c1);
            }
        };
        // The loops of the two single-thread roles are run by the whole warp, one elected lane issues: the loop state then
        // lives in uniform registers, which the copy and MMA instructions take their operands from.
        for(int t = unit; ok && t < num_tiles; t += P.num_units)
        {
            const ScaledItem it = item_of(t);
            const int u = it.u0 + pair_rank * 128, v = it.v0 + pair_rank * (BN / 2);
            for(int kb = it.kb0; kb < it.kb1; ++kb)
            {
                ok = block_wait(done_bar(stage), phase ^ 1u, wc, WAIT_EMPTY);
                ok = __all_sync(0xffffffffu, ok);
                if(!ok)
                    break;
                const uint32_t dst = base_addr + stage * L::STAGE_BYTES, bar = bar0 + 8u * stage;
                const int k = kb * SCALED_BLOCK;
                if(elect_one_sync())
                {
                    if(is_leader)
                        mbar_arrive_expect_tx(full_bar(stage), stage_tx);
                    load_box(&P.tm_u, dst, bar, P.u_mn ? u : k, P.u_mn ? k : u, P.u_batched != 0, it.group);
                    load_box(&P.tm_v, dst + L::U_BYTES, bar, P.v_mn ? v : k, P.v_mn ? k : v, P.v_batched != 0, it.group);
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
        if(lane == 0)
            tell_leader(MISC_LOADS + pair_rank, static_cast<uint32_t>(loads));
        if(!ok)
            gave_up();
        __syncwarp();
        if(CG == 1 && ksplit > 1)
            cluster_sync_all(); // (the one before the slices are summed)
        // Do not leave while a bulk copy may still write shared memory.  Where no wait gave up, every stage has been
        // multiplied, so every byte has come.  Otherwise stages may be filled whose barriers lack more than bytes: releases of
        // epilogue warps that are gone, or the part of the CTA whose producer stopped first.  All roles have left their
        // loops, so what is missing is known: it is made up for here, and then the barriers depend on the copies alone.  A
        // stage is filled again only after its last K block was multiplied, so only the last STAGES fills can be
        // incomplete, each on a barrier of its own.
        // (Here and not in the common exit, where its registers would count in every role: 2 to 15 % of the time.)
        if(roles_left())
        {
            if(is_leader && lane == 0)
            {
                const uint32_t own = misc[MISC_LOADS], other = CG == 2 ? misc[MISC_LOADS + 1] : own;
                const uint32_t most = own > other ? own : other, first = most > STAGES ? most - STAGES : 0u;
#pragma unroll 1
                for(uint32_t i = first; i < most; ++i)
                {
                    const uint32_t bar = full_bar(i % STAGES);
                    if(i >= own)
                        mbar_arrive_expect_tx(bar, stage_tx / CG); // only the other CTA's copies are on their way
                    else if(i >= other)
                        mbar_complete_tx(bar, stage_tx / CG); // only this CTA's are
#pragma unroll 1
                    for(int w = 0; w < CG * EPI_WARPS; ++w)
                        if(misc[MISC_RELEASES + w] <= i)
                            mbar_arrive(bar);
                }
                WaitCtx drain{&misc[MISC_COPY_DRAIN], kDrainLimitNs, P.status};
#pragma unroll 1
                for(uint32_t i = first; i < most; ++i)
                    bounded_wait(full_bar(i % STAGES), (i / STAGES) & 1u, drain, WAIT_DRAIN);
            }
            exit_barrier();
        }
    }
    else if(warp == 1)
    {
        // ------------------------------------------------------------------ MMA issuer
        if(is_leader)
        {
            int stage          = 0;
            uint32_t phase     = 0;
            int acc            = 0;
            bool ok            = true;
            bool issued_any    = false;
            const uint64_t u_const = P.u_mn ? make_smem_desc_mn_sw128(0, 128 * BK_BYTES) : make_smem_desc_k_sw128(0);
            const uint64_t v_const = P.v_mn ? make_smem_desc_mn_sw128(0, 128 * BK_BYTES) : make_smem_desc_k_sw128(0);
            const uint32_t u_hi = static_cast<uint32_t>(u_const >> 32), v_hi = static_cast<uint32_t>(v_const >> 32);
            const uint32_t u_step = P.u_mn ? (32 * BK_BYTES) >> 4 : 32 >> 4;
            const uint32_t v_step = P.v_mn ? (32 * BK_BYTES) >> 4 : 32 >> 4;
            for(int t = unit; ok && t < num_tiles; t += P.num_units)
            {
                const ScaledItem it = item_of(t);
                for(int kb = it.kb0; kb < it.kb1; ++kb)
                {
                    ok = block_wait(full_bar(stage), phase, wc, WAIT_FULL);
                    ok = __all_sync(0xffffffffu, ok);
                    if(!ok)
                        break;
                    tc_fence_after_sync();
                    const uint32_t u_addr = base_addr + stage * L::STAGE_BYTES;
                    const uint32_t u_lo   = static_cast<uint32_t>(u_const) | ((u_addr & 0x3FFFFu) >> 4);
                    const uint32_t v_lo   = static_cast<uint32_t>(v_const) | (((u_addr + L::U_BYTES) & 0x3FFFFu) >> 4);
                    const uint32_t d      = tmem_base + acc * BN;
                    if(elect_one_sync())
                    {
#pragma unroll
                        for(int k = 0; k < 4; ++k)
                        {
                            if constexpr(CG == 2)
                                mma_f8_ss_pair_split(d, u_lo + k * u_step, u_hi, v_lo + k * v_step, v_hi, P.idesc, k != 0);
                            else
                                mma_f8_ss_split(d, u_lo + k * u_step, u_hi, v_lo + k * v_step, v_hi, P.idesc, k != 0);
                        }
                        if constexpr(CG == 2)
                            mma_commit_pair_mc(done_bar(stage), 3);
                        else
                            mma_commit(done_bar(stage));
                    }
                    __syncwarp();
                    issued_any = true;
                    if(++acc == NUM_ACC)
                        acc = 0;
                    if(++stage == STAGES)
                    {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if(!ok)
                gave_up();
            // Every MMA issued must be finished before the tensor memory is freed.
            if(issued_any)
            {
                if(elect_one_sync())
                {
                    if constexpr(CG == 2)
                        mma_commit_pair(drain_bar);
                    else
                        mma_commit(drain_bar);
                }
                __syncwarp();
                WaitCtx drain{&misc[MISC_MMA_DRAIN], kDrainLimitNs, P.status};
                bounded_wait(drain_bar, 0, drain, WAIT_DRAIN);
            }
        }
        __syncwarp();
    }
    else
    {
        // ------------------------------------------------------------------ scales
        // Warp 2 brings the scales of the U side, warp 3 those of the V side, as asynchronous copies into the ring in
        // shared memory (no registers, nothing waits for their latency).  A batch of SCALE_BATCH K blocks belongs to one
        // tile; the last one of a tile may be shorter.
        const bool is_v    = warp == 3;
        const int n_per    = is_v ? (VMODE == 0 ? 1 : L::V_SCALES / 32) : 4; // scales of a lane and K block
        const int64_t kbs  = is_v ? P.sv_kb : P.su_kb;
        const uint32_t ring = base_addr + L::SCALE_OFFSET + ((is_v ? 128 : 0) + lane) * 4;
        int slot           = 0;
        uint32_t phase     = 0;
        bool ok            = true;
        for(int t = unit; ok && t < num_tiles; t += P.num_units)
        {
            const ScaledItem it = item_of(t);
            const float* p      = is_v ? P.sv + it.group * P.sv_group : P.su + it.group * P.su_group;
            int64_t step        = 0; // from one of the lane's scales to the next
            int have;                // how many of them exist
            if(is_v && VMODE == 0)
            {
                // blocks of 128 columns that the tile touches: three at most
                const int b = (it.v0 >> 7) + lane;
                have        = lane < 3 && (static_cast<int64_t>(b) << 7) < it.v_end ? 1 : 0;
                p += b * P.sv_row;
            }
            else
            {
                const int x   = (is_v ? it.v0 : it.u0 + static_cast<int>(CG == 2 ? cta_rank : 0) * 128) + lane;
                const int end = is_v ? (it.v0 + BN < it.v_end ? it.v0 + BN : it.v_end) : it.u_end;
                have          = x < end ? (end - x + 31) / 32 : 0;
                const int sh  = is_v ? 0 : P.u_shift;
                step          = is_v ? 32 * P.sv_row : sh ? 0 : 32 * P.su_row; // (a U tile lies in one block of 128)
                p += static_cast<int64_t>(x >> sh) * (is_v ? P.sv_row : P.su_row);
            }
            if(have <= 0)
                p = P.su; // (a valid address, never read)
            p += it.kb0 * (have > 0 ? kbs : 0);
            for(int kb = it.kb0; kb < it.kb1; kb += SCALE_BATCH)
            {
                ok = block_wait(scale_empty_bar(slot), phase ^ 1u, wc, WAIT_EMPTY);
                ok = __all_sync(0xffffffffu, ok);
                if(!ok)
                    break;
                const int n_kb = it.kb1 - kb < SCALE_BATCH ? it.kb1 - kb : SCALE_BATCH;
                uint32_t dst   = ring + slot * SCALE_BATCH * L::SCALE_WORDS * 4;
                for(int j = 0; j < n_kb; ++j)
                {
                    const float* q = p;
                    for(int i = 0; i < n_per; ++i)
                    {
                        const bool in = i < have;
                        copy_async_4(dst + i * 128, in ? q : P.su, in ? 4u : 0u);
                        q += in ? step : 0;
                    }
                    p += have > 0 ? kbs : 0;
                    dst += L::SCALE_WORDS * 4;
                }
                copy_async_arrive(scale_full_bar(slot));
                if(++slot == SLOTS)
                {
                    slot = 0;
                    phase ^= 1u;
                }
            }
        }
        if(!ok)
            gave_up();
        copy_async_wait_all(); // nothing may land in shared memory after the exit
        __syncwarp();
    }
    }
    else
    {
        if constexpr(L::SPLIT_REGS)
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::REGS_HIGH));
        // ------------------------------------------------------------------ epilogue warps
        const int quarter = warp & 3, part = (warp - SCALED_EPI_WARP0) >> 2;
        const int row     = quarter * 32 + lane; // lane of the accumulator
        const int col     = part * COLS;    // first column of this warp
        const uint32_t taddr0 = tmem_base + col + (static_cast<uint32_t>(quarter * 32) << 16);
        // The MMA thread waits on one barrier per K block: releasing the accumulator of K block i is an arrival on the
        // barrier of the stage that K block i + NUM_ACC will fill (its last phase is over: K block i has been multiplied, and
        // with it every K block up to i + NUM_ACC - STAGES).  The first NUM_ACC find their accumulators free.
        const uint32_t ready0 = (CG == 2) ? mapa_shared(full_bar(0), 0) : full_bar(0);
        auto release_for = [&](int s) { // accumulator of the K block that stage s gets next
            if(lane == 0)
            {
                if constexpr(CG == 2)
                    mbar_arrive_cluster_relaxed(ready0 + 8u * s);
                else
                    mbar_arrive(ready0 + 8u * s);
            }
        };
        for(int s = 0; s < NUM_ACC; ++s)
            release_for(s);
        int next_stage = NUM_ACC % STAGES;
        uint8_t* out_tile     = smem + L::OUT_OFFSET + (warp - SCALED_EPI_WARP0) * 2048;
        uint64_t acc[COLS / 2];
        int stage = 0, slot = 0, buf = 0;
        uint32_t round = 0, slot_phase = 0; // round: of the ring of stages
        bool ok = true;
        for(int t = unit; ok && t < num_tiles; t += P.num_units)
        {
            const ScaledItem it = item_of(t);
            // VMODE 0: the warp's columns touch two blocks of 128 at most; from column hi_from on it is the second
            const int lo_i    = ((it.v0 + col) >> 7) - (it.v0 >> 7);
            const int hi_from = (((it.v0 + col) >> 7) + 1) * 128 - (it.v0 + col);
#pragma unroll
            for(int i = 0; i < COLS / 2; ++i)
                acc[i] = 0;
            const float* su_s = nullptr;
            int in_batch      = 0;
            for(int kb = it.kb0; kb < it.kb1; ++kb)
            {
                if(in_batch == 0)
                {
                    ok   = block_wait(scale_full_bar(slot), slot_phase, wc, WAIT_FULL);
                    su_s = scale_ring + slot * SCALE_BATCH * L::SCALE_WORDS;
                }
                else
                    su_s += L::SCALE_WORDS;
                const float* sv_s = su_s + 128 + (VMODE == 0 ? lo_i : col);
                uint64_t s_lo = 0, s_hi = 0, su2[4] = {};
                if constexpr(VMODE == 0)
                {
                    const float su = su_s[row], lo = su * sv_s[0];
                    s_lo = pack_f32x2(lo, lo);
                    if constexpr(STRADDLES)
                    {
                        const float hi = su * sv_s[1];
                        s_hi           = pack_f32x2(hi, hi);
                    }
                }
                else
                {
#pragma unroll
                    for(int k = 0; k < (FRAG ? 4 : 1); ++k)
                    {
                        const float su = su_s[FRAG ? quarter * 32 + k * 8 + (lane >> 2) : row];
                        su2[k]         = pack_f32x2(su, su);
                    }
                }
                ok = ok && block_wait(done_bar(stage), round & 1u, wc, WAIT_TMEM_FULL);
                ok = __all_sync(0xffffffffu, ok);
                if(!ok)
                    break;
                tc_fence_after_sync();
                const uint32_t taddr = taddr0 + buf * BN;
                // everything is in registers: a later K block may overwrite the accumulator
                auto release = [&]() {
                    tc_fence_before_sync();
                    __syncwarp();
                    release_for(next_stage);
                };
                // N columns from column c on, from tensor memory into v, and from v into the sums
                auto load = [&](auto width, int c, uint32_t* v) {
                    constexpr int N = decltype(width)::value;
                    if constexpr(FRAG && N == 32)
                    {
                        tmem_ld_16x256b_x4(taddr + c, v);
                        tmem_ld_16x256b_x4(taddr + c + (16u << 16), v + 16);
                    }
                    else if constexpr(N == 32)
                    {
                        tmem_ld_32x32b_x16(taddr + c, v);
                        tmem_ld_32x32b_x16(taddr + c + 16, v + 16);
                    }
                    else if constexpr(FRAG && N == 16)
                    {
                        tmem_ld_16x256b_x2(taddr + c, v);
                        tmem_ld_16x256b_x2(taddr + c + (16u << 16), v + 8);
                    }
                    else if constexpr(N == 16)
                        tmem_ld_32x32b_x16(taddr + c, v);
                    else
                        tmem_ld_32x32b_x8(taddr + c, v);
                };
                auto pair_of = [](const uint32_t* v) { return pack_f32x2(__uint_as_float(v[0]), __uint_as_float(v[1])); };
                auto add     = [&](auto width, int c, const uint32_t* v) {
                    constexpr int N = decltype(width)::value;
                    if constexpr(VMODE == 0)
                    {
#pragma unroll
                        for(int i = 0; i < N; i += 2)
                        {
                            const uint64_t s2 = STRADDLES && c + (i & ~7) >= hi_from ? s_hi : s_lo;
                            acc[(c + i) / 2]  = fma_f32x2(pair_of(v + i), s2, acc[(c + i) / 2]);
                        }
                    }
                    else if constexpr(FRAG)
                    {
#pragma unroll
                        for(int g = 0; g < N / 8; ++g)
                        {
                            const uint64_t s2 = *reinterpret_cast<const uint64_t*>(sv_s + c + g * 8 + 2 * (lane & 3));
#pragma unroll
                            for(int k = 0; k < 4; ++k) // rows 8 k + lane / 4
                            {
                                const uint64_t p = pair_of(v + (k >> 1) * (N / 2) + g * 4 + (k & 1) * 2);
                                uint64_t& a      = acc[(c / 8 + g) * 4 + k];
                                a                = fma_f32x2(p, mul_f32x2(s2, su2[k]), a);
                            }
                        }
                    }
                    else
                    {
#pragma unroll
                        for(int i = 0; i < N; i += 4)
                        {
                            const ulonglong2 s4 = *reinterpret_cast<const ulonglong2*>(sv_s + c + i);
                            acc[(c + i) / 2]     = fma_f32x2(pair_of(v + i), mul_f32x2(s4.x, su2[0]), acc[(c + i) / 2]);
                            acc[(c + i) / 2 + 1] = fma_f32x2(pair_of(v + i + 2), mul_f32x2(s4.y, su2[0]), acc[(c + i) / 2 + 1]);
                        }
                    }
                };
                // (a chunk in flight while another is added was slower: the warps of a scheduler hide each other's loads)
                constexpr int LAST = COLS % CHUNK == 0 ? CHUNK : COLS % CHUNK; // BN = 224: 16
#pragma unroll
                for(int c = 0; c + CHUNK <= COLS; c += CHUNK)
                {
                    uint32_t v[CHUNK];
                    load(std::integral_constant<int, CHUNK>{}, c, v);
                    tmem_ld_wait_regs<CHUNK>(v);
                    if(c + CHUNK == COLS)
                        release();
                    add(std::integral_constant<int, CHUNK>{}, c, v);
                }
                if constexpr(LAST != CHUNK)
                {
                    uint32_t v[LAST];
                    load(std::integral_constant<int, LAST>{}, COLS - LAST, v);
                    tmem_ld_wait_regs<LAST>(v);
                    release();
                    add(std::integral_constant<int, LAST>{}, COLS - LAST, v);
                }
                if(++in_batch == SCALE_BATCH || kb + 1 == it.kb1)
                {
                    in_batch = 0;
                    __syncwarp();
                    if(lane == 0)
                        mbar_arrive(scale_empty_bar(slot));
                    if(++slot == SLOTS)
                    {
                        slot = 0;
                        slot_phase ^= 1u;
                    }
                }
                if(++buf == NUM_ACC)
                    buf = 0;
                if(++next_stage == STAGES)
                    next_stage = 0;
                if(++stage == STAGES)
                {
                    stage = 0;
                    ++round;
                }
            }
            if(!ok)
                break;
            if(CG == 1 && ksplit > 1)
            {
                // hand the sums to the CTAs that own the columns: [slice][column of the part][row]
                const int pw        = BN / ksplit;
                const uint32_t part = base_addr + L::OUT_OFFSET + static_cast<uint32_t>(cta_rank) * pw * 512u + row * 4u;
#pragma unroll
                for(int c = 0; c < COLS; ++c)
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
            const int64_t e_off = it.group * P.e_group;
            const int u_row     = it.u0 + static_cast<int>(CG == 2 ? cta_rank : 0) * 128 + quarter * 32;
            auto store = [&](auto* e) {
                using T = typename std::remove_pointer<decltype(e)>::type;
                if constexpr(CG == 1)
                    store_cols<T, COLS>(acc, e + e_off, P.lde, u_row + lane, it.u_end, it.v0 + col, it.v_end);
                else
                    store_rows<T, COLS, FRAG>(acc, out_tile, e + e_off, P.lde, u_row, it.u_end, it.v0 + col, it.v_end, P.e_vec != 0, lane);
            };
            if(P.e_dtype == CKB_BF16)
                store(static_cast<__nv_bfloat16*>(P.e));
            else if(P.e_dtype == CKB_F16)
                store(static_cast<__half*>(P.e));
            else
                store(static_cast<float*>(P.e));
        }
        if(!ok)
        {
            if(lane == 0)
                tell_leader(MISC_RELEASES + (CG == 2 ? cluster_ctarank() * EPI_WARPS : 0) + warp - SCALED_EPI_WARP0, round * STAGES + stage + NUM_ACC);
            gave_up();
        }
        __syncwarp();
    }

    if(CG == 1 && ksplit > 1)
    {
        if(warp != 0) // (the producer has been there)
            cluster_sync_all(); // every slice is at its owner (release / acquire at cluster scope)
        if(warp >= SCALED_EPI_WARP0 && misc[MISC_ABORT] == 0 && unit < num_tiles)
        {
            const ScaledItem it = item_of(unit);
            const int t = static_cast<int>(threadIdx.x) - 32 * SCALED_EPI_WARP0, row = t & 127;
            const int pw      = BN / ksplit;
            const float* part = reinterpret_cast<const float*>(smem + L::OUT_OFFSET);
            const int v0      = it.v0 + static_cast<int>(cta_rank) * pw;
            auto sum = [&](auto* e) { store_slices(part, pw, ksplit, e, P.lde, it.u0 + row, it.u_end, v0, it.v_end, row, t >> 7, EPI_WARPS / 4); };
            if(P.e_dtype == CKB_BF16)
                sum(static_cast<__nv_bfloat16*>(P.e));
            else if(P.e_dtype == CKB_F16)
                sum(static_cast<__half*>(P.e));
            else
                sum(static_cast<float*>(P.e));
        }
    }

    // ---------------------------------------------------------------------- common exit
    if(warp != 0 && roles_left()) // (the producer has been there)
        exit_barrier();
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
