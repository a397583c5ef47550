// Host side of the 8-bit products with block scales (ckb_scaled_gemm_*, ckb_scaled_grouped_gemm_*).
#include <cstdlib>
#include <cstring>
#include <mutex>

#include "ckb_host.h"
#include "ckb_scaled_launch.cuh"

namespace {

using namespace ckb;

constexpr int64_t kMaxExtent = 0x7ffff000ll; // TMA coordinates and tile starts are 32-bit

bool is_f8(int dtype) { return dtype == CKB_F8_E4M3 || dtype == CKB_F8_E5M2; }
bool is_wide(int dtype) { return dtype == CKB_BF16 || dtype == CKB_F16 || dtype == CKB_F32; }
int wide_bytes(int dtype) { return dtype == CKB_F32 ? 4 : 2; }

// One problem for both entry points.
struct ScaledProblem
{
    ckb_scaled_gemm_desc d;
    int mode, groups;
    const int32_t* offsets;
    int64_t b_group, b_scale_group, e_group;
};

int check_scaled(const ScaledProblem& q, bool need_pointers)
{
    const ckb_scaled_gemm_desc& d = q.d;
    if(!is_f8(d.a_dtype) || !is_f8(d.b_dtype))
        return host_fail(CKB_ERR_UNSUPPORTED, "A and B of an 8-bit product are CKB_F8_E4M3 or CKB_F8_E5M2");
    if(!is_wide(d.e_dtype))
        return host_fail(CKB_ERR_UNSUPPORTED, "E of an 8-bit product is CKB_BF16, CKB_F16 or CKB_F32");
    if((d.a_layout != CKB_ROW_MAJOR && d.a_layout != CKB_COL_MAJOR) || (d.b_layout != CKB_ROW_MAJOR && d.b_layout != CKB_COL_MAJOR))
        return host_fail(CKB_ERR_INVALID, "unknown layout");
    if((d.scale_block_m != 1 && d.scale_block_m != 128) || (d.scale_block_n != 1 && d.scale_block_n != 128))
        return host_fail(CKB_ERR_UNSUPPORTED, "a scale covers 1 or 128 rows of A and 1 or 128 columns of B");
    if(d.M < 1 || d.N < 1 || d.K < 1 || d.M > kMaxExtent || d.N > kMaxExtent || d.K > kMaxExtent)
        return host_fail(CKB_ERR_UNSUPPORTED, "M, N and K must be positive and below 2^31");
    const bool a_mn = d.a_layout == CKB_COL_MAJOR, b_mn = d.b_layout == CKB_ROW_MAJOR;
    if(d.lda < (a_mn ? d.M : d.K) || d.ldb < (b_mn ? d.N : d.K) || d.lde < d.N)
        return host_fail(CKB_ERR_INVALID, "a leading dimension is smaller than its row or column");
    if(d.lda % 16 != 0 || d.ldb % 16 != 0)
        return host_fail(CKB_ERR_UNSUPPORTED, "pitches of A and B must be multiples of 16 bytes");
    if(d.lda >= (1ll << 40) || d.ldb >= (1ll << 40))
        return host_fail(CKB_ERR_UNSUPPORTED, "pitches of A and B must be below 2^40 bytes");
    if(d.a_scale_stride_m < 0 || d.a_scale_stride_k < 0 || d.b_scale_stride_n < 0 || d.b_scale_stride_k < 0)
        return host_fail(CKB_ERR_INVALID, "scale strides must not be negative");
    if(q.mode != SCALED_PLAIN)
    {
        if(q.groups < 1 || q.groups > CKB_SCALED_MAX_GROUPS)
            return host_fail(CKB_ERR_LIMIT, "1 to %d groups, got %d", CKB_SCALED_MAX_GROUPS, q.groups);
        if(q.mode == SCALED_GROUP_ROWS)
        {
            if(a_mn || d.scale_block_m != 1)
                return host_fail(CKB_ERR_UNSUPPORTED, "groups of rows need a row-major A with a scale per row");
            if(q.b_group < 0 || q.b_group % 16 != 0 || q.b_group >= (1ll << 40) || q.b_scale_group < 0)
                return host_fail(CKB_ERR_INVALID, "b_group_stride must be a multiple of 16, no group stride negative");
        }
        // (a division, because the size of a matrix may pass 64 bits)
        else if(q.e_group < 0 || (q.groups > 1 && (q.e_group < d.N || (q.e_group - d.N) / d.lde < d.M - 1)))
            return host_fail(CKB_ERR_INVALID, "e_group_stride is smaller than a matrix of E");
    }
    const int cols = d.tile_config & 0xFFF, cg = (d.tile_config >> 12) & 0xF, ks = (d.tile_config >> 20) & 0xF;
    if(d.tile_config < 0 || (d.tile_config & ~0xF0FFFF) != 0 || cg > 2 || (d.tile_config != 0 && (cols == 0 || cg == 0)) ||
       !(ks == 0 || ks == 1 || ks == 2 || ks == 4 || ks == 8))
        return host_fail(CKB_ERR_INVALID, "tile_config 0x%x is not a CKB_SCALED_TILE value", d.tile_config);
    if(need_pointers)
    {
        if(!d.p_a || !d.p_b || !d.p_a_scale || !d.p_b_scale || !d.p_e || (q.mode != SCALED_PLAIN && !q.offsets))
            return host_fail(CKB_ERR_INVALID, "null tensor pointer");
        if((reinterpret_cast<uintptr_t>(d.p_a) | reinterpret_cast<uintptr_t>(d.p_b)) % 16 != 0)
            return host_fail(CKB_ERR_UNSUPPORTED, "A and B must start on 16-byte boundaries");
        if((reinterpret_cast<uintptr_t>(d.p_a_scale) | reinterpret_cast<uintptr_t>(d.p_b_scale) | reinterpret_cast<uintptr_t>(q.offsets)) % 4 != 0 ||
           reinterpret_cast<uintptr_t>(d.p_e) % wide_bytes(d.e_dtype) != 0)
            return host_fail(CKB_ERR_INVALID, "scales, offsets or E not aligned to their elements");
    }
    return CKB_OK;
}

// Test hook: CKB_TEST_SCALED_WAIT_EXTRA makes barriers of the products wait for one arrival more than will ever come, so that
// (with a short CKB_WAIT_LIMIT_MS) waits run out while copies and MMAs are on their way.  Bit 0: the scales' barriers, bit
// 1: those that say that a K block was multiplied; bit 2 / 3: only in even / odd CTAs (the first / second one of a pair).
uint32_t scaled_test_wait()
{
    const char* s = getenv("CKB_TEST_SCALED_WAIT_EXTRA");
    return s ? static_cast<uint32_t>(atoi(s)) & 15u : 0u;
}

// Clusters of 2 / 4 / 8 CTAs that the device (the part that CKB_SM_LIMIT leaves of it) holds at once, asked once per device:
// what the planner reckons with, and a K split over a cluster that does not fit (0) is not made.
int cluster_caps(const HostDevice& dev, int (&cap)[3])
{
    static std::mutex mutex;
    static int known[64][3];
    static bool asked[64];
    int ordinal = 0;
    if(cudaGetDevice(&ordinal) != cudaSuccess || ordinal < 0 || ordinal >= 64)
        return host_fail(CKB_ERR_CUDA, "no current device");
    std::lock_guard<std::mutex> lock(mutex);
    if(!asked[ordinal])
    {
        bool all = true;
        for(int i = 0; i < 3; ++i)
        {
            ScaledParams p;
            memset(&p, 0, sizeof(p));
            const int limit = dev.sm_count / (2 << i);
            int n           = 0;
            if(launch_scaled<0, 1>(128, p, (2 << i) * 64, nullptr, 2 << i, &n) != cudaSuccess)
            {
                cudaGetLastError(); // not an answer: as many as there are SMs for, and the next call asks again
                n   = limit;
                all = false;
            }
            known[ordinal][i] = n < limit ? n : limit;
        }
        asked[ordinal] = all;
    }
    for(int i = 0; i < 3; ++i)
        cap[i] = known[ordinal][i];
    return CKB_OK;
}

bool plan_problem(const ScaledProblem& q, int sm_count, const int (&cap)[3], ScaledPlan* plan)
{
    const ckb_scaled_gemm_desc& d = q.d;
    ScaledPlanInput in;
    in.M        = d.M;
    in.N        = d.N;
    in.num_kb   = static_cast<int32_t>((d.K + SCALED_BLOCK - 1) / SCALED_BLOCK);
    in.mode     = q.mode;
    in.groups   = q.mode == SCALED_PLAIN ? 1 : q.groups;
    in.a_mn     = d.a_layout == CKB_COL_MAJOR;
    in.b_mn     = d.b_layout == CKB_ROW_MAJOR;
    in.a_block  = d.scale_block_m;
    in.b_block  = d.scale_block_n;
    in.sm_count = sm_count;
    for(int i = 0; i < 3; ++i)
        in.cluster_cap[i] = cap[i];
    if(d.tile_config != 0)
    {
        in.cols   = d.tile_config & 0xFFF;
        in.cg     = (d.tile_config >> 12) & 0xF;
        in.ksplit = (d.tile_config >> 20) & 0xF;
        if(in.ksplit == 0)
            in.ksplit = 1;
    }
    return plan_scaled(in, plan);
}

int scaled_supported(const ScaledProblem& q)
{
    if(int rc = check_scaled(q, false))
        return rc;
    // a whole B200, or the part that CKB_SM_LIMIT leaves of it (the run asks the device, which this call does not need)
    ScaledPlan plan;
    const int sms = host_limited_sms(148);
    int cap[3]    = {64, 32, 16};
    for(int i = 0; i < 3; ++i)
        if(cap[i] > sms / (2 << i))
            cap[i] = sms / (2 << i);
    if(!plan_problem(q, sms, cap, &plan))
        return host_fail(CKB_ERR_UNSUPPORTED, "no tile fits: too many tiles, or a pinned tile that the problem cannot use");
    return CKB_OK;
}

int scaled_run(const ScaledProblem& q, void* stream_, int n_rep, float* avg_ms)
{
    if(int rc = check_scaled(q, true))
        return rc;
    const ckb_scaled_gemm_desc& d = q.d;
    HostDevice dev;
    if(int rc = host_device(&dev))
        return rc;
    const struct
    {
        const void* p;
        const char* name;
    } used[] = {{d.p_a, "A"}, {d.p_b, "B"}, {d.p_a_scale, "the scale of A"}, {d.p_b_scale, "the scale of B"}, {d.p_e, "E"}, {q.offsets, "offsets"}};
    for(const auto& u : used)
        if(int rc = host_check_pointer(u.p, u.name))
            return rc;
    int cap[3];
    if(int rc = cluster_caps(dev, cap))
        return rc;
    ScaledPlan plan;
    if(!plan_problem(q, dev.sm_count, cap, &plan))
        return host_fail(CKB_ERR_UNSUPPORTED, "no tile fits: too many tiles, or a pinned tile that the problem cannot use");

    const bool swapped = plan.t.swapped != 0;
    const bool rows    = q.mode == SCALED_GROUP_ROWS;
    const bool a_mn = d.a_layout == CKB_COL_MAJOR, b_mn = d.b_layout == CKB_ROW_MAJOR;
    ScaledParams p;
    memset(&p, 0, sizeof(p));
    p.tiles      = plan.t;
    p.num_tiles  = plan.num_tiles;
    p.num_units  = plan.grid / (plan.cg == 2 ? 2 : plan.t.ksplit);
    p.v_box_rows = plan.t.width / plan.cg;
    const int a_box = swapped ? p.v_box_rows : 128, b_box = swapped ? 128 : p.v_box_rows;
    CUtensorMap& tm_a = swapped ? p.tm_v : p.tm_u;
    CUtensorMap& tm_b = swapped ? p.tm_u : p.tm_v;
    // K-major: rows along M|N, box of `box` rows; MN-major: rows along K, box of the 128 rows of a K block
    int rc = host_encode_8bit(&tm_a, d.p_a, a_mn ? d.K : d.M, a_mn ? d.M : d.K, d.lda, a_mn ? SCALED_BLOCK : a_box, 0, 0, "A");
    if(rc)
        return rc;
    // a single group's stride is never used; the map wants a multiple of 16 all the same
    rc = host_encode_8bit(&tm_b, d.p_b, b_mn ? d.K : d.N, b_mn ? d.N : d.K, d.ldb, b_mn ? SCALED_BLOCK : b_box, rows ? q.groups : 0,
                          rows ? q.b_group : 0, "B");
    if(rc)
        return rc;
    const int64_t a_row = d.a_scale_stride_m, a_kb = d.a_scale_stride_k, b_row = d.b_scale_stride_n, b_kb = d.b_scale_stride_k;
    const int a_shift = d.scale_block_m == 128 ? 7 : 0, b_shift = d.scale_block_n == 128 ? 7 : 0;
    const int64_t b_grp = rows ? q.b_scale_group : 0;
    p.su       = swapped ? d.p_b_scale : d.p_a_scale;
    p.su_row   = swapped ? b_row : a_row;
    p.su_kb    = swapped ? b_kb : a_kb;
    p.su_group = swapped ? b_grp : 0;
    p.u_shift  = swapped ? b_shift : a_shift;
    p.sv       = swapped ? d.p_a_scale : d.p_b_scale;
    p.sv_row   = swapped ? a_row : b_row;
    p.sv_kb    = swapped ? a_kb : b_kb;
    p.sv_group = swapped ? 0 : b_grp;
    p.u_mn      = swapped ? b_mn : a_mn;
    p.v_mn      = swapped ? a_mn : b_mn;
    p.u_batched = rows && swapped;
    p.v_batched = rows && !swapped;
    p.e         = d.p_e;
    p.lde       = d.lde;
    p.e_group   = q.mode == SCALED_GROUP_K ? q.e_group : 0;
    p.e_dtype   = d.e_dtype;
    const int eb = wide_bytes(d.e_dtype);
    p.e_vec     = reinterpret_cast<uintptr_t>(d.p_e) % 16 == 0 && d.lde * eb % 16 == 0 && p.e_group * eb % 16 == 0;
    const uint32_t fa = d.a_dtype == CKB_F8_E5M2, fb = d.b_dtype == CKB_F8_E5M2;
    const uint32_t fu = swapped ? fb : fa, fv = swapped ? fa : fb;
    p.idesc = (1u << 4) | (fu << 7) | (fv << 10) | (static_cast<uint32_t>(p.u_mn) << 15) | (static_cast<uint32_t>(p.v_mn) << 16) |
              (static_cast<uint32_t>(plan.t.width) >> 3 << 17) | (static_cast<uint32_t>(plan.t.u_rows) >> 4 << 24);
    p.offsets       = q.offsets;
    p.wait_limit_ns = dev.wait_limit_ns;
    p.status        = dev.status;
    p.test_wait     = scaled_test_wait();
    const int vmode = scaled_vmode(swapped ? d.scale_block_m : d.scale_block_n);
    auto* fn        = plan.cg == 1 ? (vmode == 0 ? &launch_scaled<0, 1> : &launch_scaled<1, 1>)
                                   : (vmode == 0 ? &launch_scaled<0, 2> : &launch_scaled<1, 2>);
    host_note_plan("scaled%s tile=%dx%d cg=%d swapped=%d grid=%d ksplit=%d vmode=%d", rows ? " rows" : q.mode == SCALED_GROUP_K ? " kblocks" : "",
                   plan.t.u_rows, plan.t.width, plan.cg, plan.t.swapped, plan.grid, plan.t.ksplit, vmode);
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    return host_run_timed([&]() { return fn(plan.t.width, p, plan.grid, stream, 0, nullptr); }, 1, stream, n_rep, avg_ms);
}

ScaledProblem plain_problem(const ckb_scaled_gemm_desc* d)
{
    ScaledProblem q;
    memset(&q, 0, sizeof(q));
    q.d    = *d;
    q.mode = SCALED_PLAIN;
    return q;
}

int grouped_problem(const ckb_scaled_grouped_gemm_desc* g, ScaledProblem* q)
{
    if(!g)
        return host_fail(CKB_ERR_INVALID, "null descriptor");
    if(g->group_axis != CKB_GROUP_ROWS && g->group_axis != CKB_GROUP_K_BLOCKS)
        return host_fail(CKB_ERR_INVALID, "unknown group axis %d", g->group_axis);
    memset(q, 0, sizeof(*q));
    q->d             = g->gemm;
    q->mode          = g->group_axis == CKB_GROUP_ROWS ? SCALED_GROUP_ROWS : SCALED_GROUP_K;
    q->groups        = g->group_count;
    q->offsets       = g->p_offsets;
    q->b_group       = g->b_group_stride;
    q->b_scale_group = g->b_scale_group_stride;
    q->e_group       = g->e_group_stride;
    return CKB_OK;
}

} // namespace

extern "C" {

int ckb_scaled_gemm_supported(const ckb_scaled_gemm_desc* d)
{
    return d ? scaled_supported(plain_problem(d)) : host_fail(CKB_ERR_INVALID, "null descriptor");
}

int ckb_scaled_gemm_run(const ckb_scaled_gemm_desc* d, void* stream, int n_rep, float* avg_ms)
{
    return d ? scaled_run(plain_problem(d), stream, n_rep, avg_ms) : host_fail(CKB_ERR_INVALID, "null descriptor");
}

int ckb_scaled_grouped_gemm_supported(const ckb_scaled_grouped_gemm_desc* g)
{
    ScaledProblem q;
    const int rc = grouped_problem(g, &q);
    return rc ? rc : scaled_supported(q);
}

int ckb_scaled_grouped_gemm_run(const ckb_scaled_grouped_gemm_desc* g, void* stream, int n_rep, float* avg_ms)
{
    ScaledProblem q;
    const int rc = grouped_problem(g, &q);
    return rc ? rc : scaled_run(q, stream, n_rep, avg_ms);
}

} // extern "C"
