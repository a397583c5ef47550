// Work decomposition of the 8-bit products with block scales (plain C++: kernel, host and host-only test compile the
// same text).
//
// One operand of the product is the U side (the 128 rows a CTA's tensor core works on), the other the V side (the
// columns of the accumulator).  `swapped` = 0: U = A (rows of E), V = B (columns of E); `swapped` = 1: U = B, V = A.
// CTA pairs work unswapped, single CTAs swapped.
// A tile is u_rows = 128 x CTAs of U by `width` of V.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define CKB_SP_HD __host__ __device__ __forceinline__
#else
#define CKB_SP_HD inline
#endif

namespace ckb {

constexpr int SCALED_BLOCK = 128; // K values per scale

enum { SCALED_PLAIN = 0, SCALED_GROUP_ROWS = 1, SCALED_GROUP_K = 2 };

struct ScaledTiles
{
    int32_t mode;      // SCALED_*
    int32_t swapped;
    int32_t u_rows;    // 128 or 256
    int32_t width;     // columns of V per tile
    int32_t ext_u, ext_v; // extents of U and V (GROUP_ROWS: of the side of B; the other one comes from the offsets)
    int32_t tiles_u, tiles_v;
    int32_t num_kb;    // K blocks of the whole problem
    int32_t groups;
    int32_t band;      // U tiles walked side by side (tile_of)
    int32_t ksplit;    // CTAs of a cluster that share a tile's K blocks (1: no split)
};

// What a tile is: where it starts on both sides, where its side ends, and which K blocks it adds up.
struct ScaledItem
{
    int32_t u0, v0, u_end, v_end;
    int32_t kb0, kb1;
    int32_t group;
};

CKB_SP_HD int32_t scaled_div_up(int32_t a, int32_t b) { return (a + b - 1) / b; } // a + b < 2^31 (host check)
CKB_SP_HD int32_t scaled_clip(int32_t v, int32_t lo, int32_t hi) { return v < lo ? lo : v > hi ? hi : v; }

// Tiles are walked in bands of `band` U tiles: all V tiles of a band before the next band, the U tiles of the band
// fastest.  The operand tiles that units work on at the same time then form a block, whose two sides stay in L2.
CKB_SP_HD void scaled_tile_of(int32_t t, int32_t tiles_u, int32_t tiles_v, int32_t band, int32_t* u, int32_t* v)
{
    const int32_t per  = band * tiles_v; // host: fits 32 bits
    const int32_t b    = t / per, rest = t - b * per;
    const int32_t left = tiles_u - b * band;
    const int32_t high = left < band ? left : band;
    *v                 = rest / high;
    *u                 = b * band + (rest - *v * high);
}

// Rows of group g: offsets as they are clipped (see ckb_scaled_grouped_gemm_desc).
CKB_SP_HD void scaled_group_span(const int32_t* offsets, int g, int32_t extent, int32_t* lo, int32_t* hi)
{
    *lo = scaled_clip(offsets[g], 0, extent);
    *hi = scaled_clip(offsets[g + 1], *lo, extent);
}

// Tiles of the offsets' side for a group of n rows (GROUP_ROWS).
CKB_SP_HD int32_t scaled_group_tiles(const ScaledTiles& p, int32_t n)
{
    return scaled_div_up(n, p.swapped ? p.width : p.u_rows);
}

// Item of tile t (PLAIN, GROUP_K: t counts group by group).
CKB_SP_HD ScaledItem scaled_item(const ScaledTiles& p, int32_t t, const int32_t* offsets)
{
    ScaledItem it;
    it.group = 0;
    it.kb0   = 0;
    it.kb1   = p.num_kb;
    if(p.mode == SCALED_GROUP_K)
    {
        const int32_t per = p.tiles_u * p.tiles_v;
        it.group          = t / per;
        t -= it.group * per;
        scaled_group_span(offsets, it.group, p.num_kb, &it.kb0, &it.kb1);
    }
    int32_t u, v;
    scaled_tile_of(t, p.tiles_u, p.tiles_v, p.band, &u, &v);
    it.u0    = u * p.u_rows;
    it.v0    = v * p.width;
    it.u_end = p.ext_u;
    it.v_end = p.ext_v;
    return it;
}

// Slice `rank` of a tile's K blocks (of `ksplit`): in order, lengths that differ by one at most.
CKB_SP_HD void scaled_slice(ScaledItem* it, int rank, int ksplit)
{
    const int32_t first = it->kb0;
    const int64_t n     = it->kb1 - first;
    it->kb0             = first + static_cast<int32_t>(n * rank / ksplit);
    it->kb1             = first + static_cast<int32_t>(n * (rank + 1) / ksplit);
}

// Item of tile t of a GROUP_ROWS problem.  starts[g] = tiles before group g (starts[groups] = all of them),
// row0[g] / row1[g] = its rows.
CKB_SP_HD ScaledItem scaled_group_item(const ScaledTiles& p, int32_t t, const int32_t* starts, const int32_t* row0,
                                       const int32_t* row1)
{
    int32_t lo = 0, hi = p.groups; // the last group that starts at or before t (empty groups share a start with the next)
    while(hi - lo > 1)
    {
        const int32_t mid = (lo + hi) >> 1;
        if(starts[mid] <= t)
            lo = mid;
        else
            hi = mid;
    }
    ScaledItem it;
    it.group            = lo;
    it.kb0              = 0;
    it.kb1              = p.num_kb;
    const int32_t mine  = starts[lo + 1] - starts[lo]; // tiles of this group
    const int32_t other = p.swapped ? p.tiles_u : p.tiles_v;
    const int32_t own   = mine / other;
    int32_t u, v;
    scaled_tile_of(t - starts[lo], p.swapped ? other : own, p.swapped ? own : other, p.band, &u, &v);
    it.u0    = u * p.u_rows + (p.swapped ? 0 : row0[lo]);
    it.v0    = v * p.width + (p.swapped ? row0[lo] : 0);
    it.u_end = p.swapped ? p.ext_u : row1[lo];
    it.v_end = p.swapped ? row1[lo] : p.ext_v;
    return it;
}

// ---- host: which tile a problem gets ---------------------------------------------------------------
struct ScaledPlanInput
{
    int64_t M, N;
    int32_t num_kb;
    int32_t mode, groups;
    bool a_mn, b_mn;          // M- / N-contiguous operand
    int a_block, b_block;     // rows / columns per scale
    int sm_count;
    int cluster_cap[3];       // clusters of 2 / 4 / 8 CTAs resident at once
    int cols = 0, cg = 0, ksplit = 0; // pinned by the caller (0: free)
};
struct ScaledPlan
{
    ScaledTiles t;
    int cg;
    int num_tiles; // GROUP_ROWS: the largest number there can be
    int grid;
    double cycles;
};

// Cycles, fitted to timings of pinned tiles (N = K = 4096, 4 to 384 rows; 1.92 GHz): a K block costs its instructions and
// waits, not its bytes or products, and grows with the width.
//   per K block   256 x 128 / 192 / 256: 295 / 395 / 444 ns, with a scale per column 440 / - / 643 ns
//                 128 x 16 / 32 / 64 / 128 (single CTA, a scale per column): 282 / 305 / 406 / 506 ns, a tenth more with
//                 all SMs at work
//   per tile      its way out of the registers
//   K split       handing the parts over: 1.5 us at 16 columns to 5.1 us at 128 between 2 CTAs, a third more between 4;
//                 clusters beyond the first wave start only when a whole cluster has ended
inline double scaled_kb_cycles(int cg, int width, int vmode)
{
    if(cg == 2)
        return vmode == 0 ? 280.0 + 2.25 * width : 500.0 + 3.05 * width;
    return vmode == 0 ? 490.0 + 3.1 * width : 540.0 + 4.1 * width;
}
inline double scaled_tile_cycles(int cg, int width) { return (cg == 2 ? 10.0 : 8.0) * width; }
inline double scaled_split_cycles(int ksplit, int width)
{
    return ksplit == 1 ? 0.0 : (2300.0 + 64.0 * width) * (ksplit == 2 ? 1.0 : 1.3);
}

constexpr int kScaledWidths[2][4] = {{16, 32, 64, 128}, {128, 192, 224, 256}}; // columns of V per tile, by CTAs per tile

inline int scaled_vmode(int v_block) { return v_block == 128 ? 0 : 1; }

// Chooses tile, orientation and K split by estimated cycles; false when nothing fits (too many tiles, or a pinned
// configuration that the problem cannot use).
inline bool plan_scaled(const ScaledPlanInput& in, ScaledPlan* out)
{
    bool found = false;
    const bool rows = in.mode == SCALED_GROUP_ROWS;
    for(int cg = 1; cg <= 2; ++cg)
    {
        const int swap = cg == 1 ? 1 : 0;
        for(const int width : kScaledWidths[cg - 1])
            for(int ks = 1; ks <= (cg == 1 ? 8 : 1); ks *= 2)
            {
                if((in.cg && in.cg != cg) || (in.cols && in.cols != width) || (in.ksplit ? in.ksplit != ks : in.cols && ks != 1))
                    continue;
                const bool v_mn = swap ? in.a_mn : in.b_mn;
                if(cg == 1 && v_mn && width != 128) // an MN-major tile is 128 columns wide
                    continue;
                if(ks > 1 && (in.mode != SCALED_PLAIN || in.num_kb < 2 * ks))
                    continue;
                ScaledPlan p;
                p.cg          = cg;
                p.t.mode      = in.mode;
                p.t.swapped   = swap;
                p.t.u_rows    = 128 * cg;
                p.t.width     = width;
                const int64_t eu = swap ? in.N : in.M, ev = swap ? in.M : in.N;
                p.t.ext_u     = static_cast<int32_t>(eu);
                p.t.ext_v     = static_cast<int32_t>(ev);
                const int64_t tu = (eu + p.t.u_rows - 1) / p.t.u_rows, tv = (ev + width - 1) / width;
                p.t.tiles_u   = static_cast<int32_t>(tu);
                p.t.tiles_v   = static_cast<int32_t>(tv);
                p.t.num_kb    = in.num_kb;
                p.t.groups    = in.groups;
                p.t.ksplit    = ks;
                p.t.band      = 8;
                const int64_t most = in.mode == SCALED_PLAIN ? tu * tv : static_cast<int64_t>(in.groups) * tu * tv;
                if(most * ks > 0x7fffff00ll || tv * 8 > 0x7fffff00ll)
                    continue;
                // tiles there will be: with rows per group unknown, every group with rows has half a tile of waste
                double tiles = static_cast<double>(most), kb = in.num_kb;
                int64_t cap  = most;
                if(rows)
                {
                    const int64_t own = swap ? width : p.t.u_rows, other = swap ? tu : tv;
                    const double busy = in.M < in.groups ? static_cast<double>(in.M) : in.groups;
                    const double mean = in.M / busy;
                    const double per  = mean <= own / 2 ? 1.0 : mean / own + 0.5;
                    tiles             = busy * per * other;
                    cap               = (in.M / own + in.groups) * other; // offsets that do not decrease
                }
                else if(in.mode == SCALED_GROUP_K)
                    kb = static_cast<double>(in.num_kb) / in.groups;
                p.num_tiles = static_cast<int>(most);
                const int units = cg == 2 ? in.sm_count / 2 : ks == 1 ? in.sm_count : in.cluster_cap[ks == 2 ? 0 : ks == 4 ? 1 : 2];
                if(units < 1)
                    continue;
                const int vmode     = scaled_vmode(swap ? in.a_block : in.b_block);
                const double per    = scaled_kb_cycles(cg, width, vmode);
                const int64_t waves = (static_cast<int64_t>(tiles) + units - 1) / units;
                const int n_kb      = static_cast<int>((kb + ks - 1) / ks);
                p.cycles            = waves * (n_kb * per + scaled_tile_cycles(cg, width) + scaled_split_cycles(ks, width));
                const int64_t want  = ks > 1 ? most : (cap < units ? cap : units);
                p.grid              = static_cast<int>(want) * (cg == 2 ? 2 : ks);
                if(!found || p.cycles < out->cycles)
                {
                    *out  = p;
                    found = true;
                }
            }
    }
    return found;
}

} // namespace ckb
