// Host side of the block quantizer and of layer norm (ckb_block_quantize_*, ckb_layernorm_*).
#include <atomic>
#include <cstring>
#include <numeric>

#include "ckb_host.h"
#include "ckb_rows.cuh"

namespace {

using namespace ckb;

constexpr int64_t kMaxRows = int64_t(1) << 40, kMaxCols = 0x7fff0000ll;

bool is_wide(int dtype) { return dtype == CKB_BF16 || dtype == CKB_F16 || dtype == CKB_F32; }
bool is_f8(int dtype) { return dtype == CKB_F8_E4M3 || dtype == CKB_F8_E5M2; }
int wide_bytes(int dtype) { return dtype == CKB_F32 ? 4 : 2; }
bool starts_on(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
float qmax_of(int dtype) { return dtype == CKB_F8_E5M2 ? 57344.f : 448.f; }
int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

template <typename P>
cudaError_t launch(void (*kern)(P), int64_t grid_x, int grid_y, int threads, cudaStream_t stream, const P& p, int smem = 0)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim            = dim3(static_cast<unsigned>(grid_x), grid_y, 1);
    cfg.blockDim           = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes   = smem;
    cfg.stream             = stream;
    cudaLaunchAttribute attr[1];
    int n = 0;
    host_add_pdl(attr, &n);
    cfg.attrs    = attr;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kern, p);
}

// The same for a kernel that takes more than 48 KB of shared memory at times: allowed once per device.
constexpr int kMaxSmem = 220 * 1024; // (the kernels have up to 6 KB besides)
template <auto KERN, typename P>
cudaError_t launch_big(int64_t grid_x, int threads, cudaStream_t stream, const P& p, int smem)
{
    static std::atomic<bool> done[64] = {};
    int dev         = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if(err != cudaSuccess)
        return err;
    if(dev < 0 || dev >= 64 || !done[dev])
    {
        err = cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
        if(err != cudaSuccess)
            return err;
        if(dev >= 0 && dev < 64)
            done[dev] = true;
    }
    return launch(KERN, grid_x, 1, threads, stream, p, smem);
}

// fn(T{}) with T = the type of a CKB_BF16 / CKB_F16 / CKB_F32 tensor
template <typename Fn>
auto with_type(int dtype, Fn fn)
{
    return dtype == CKB_BF16 ? fn(__nv_bfloat16{}) : dtype == CKB_F16 ? fn(__half{}) : fn(float{});
}
template <bool V>
struct Flag
{
    static constexpr bool value = V;
};

struct Used
{
    const void* p;
    const char* name;
};
template <int N>
int check_pointers(const Used (&used)[N])
{
    for(const Used& u : used)
        if(int rc = host_check_pointer(u.p, u.name))
            return rc;
    return CKB_OK;
}

// Whether two of the m x n blocks share a scale at strides sm and sn (none negative), which would be a race: the smallest step
// that leads from one scale to the same one is sn / gcd blocks down and sm / gcd back.
bool scales_collide(int64_t sm, int64_t sn, int64_t m, int64_t n)
{
    if(m <= 1 && n <= 1)
        return false;
    if(m <= 1 || n <= 1)
        return (m <= 1 ? sn : sm) == 0;
    const int64_t g = std::gcd(sm, sn);
    return g == 0 || (sn / g < m && sm / g < n);
}

// ---- block quantizer ------------------------------------------------------------------------------
int check_quantize(const ckb_block_quantize_desc* d, bool need_pointers)
{
    if(!d)
        return host_fail(CKB_ERR_INVALID, "null descriptor");
    if(!is_wide(d->x_dtype) || !is_f8(d->q_dtype))
        return host_fail(CKB_ERR_UNSUPPORTED, "the block quantizer reads CKB_BF16, CKB_F16 or CKB_F32 and writes CKB_F8_E4M3 or CKB_F8_E5M2");
    if(!((d->block_m == 1 && d->block_n == 128) || (d->block_m == 128 && (d->block_n == 1 || d->block_n == 128))))
        return host_fail(CKB_ERR_UNSUPPORTED, "blocks are 1 x 128, 128 x 1 or 128 x 128, got %d x %d", d->block_m, d->block_n);
    if((d->pow2_scale != 0 && d->pow2_scale != 1) || d->pad_ != 0)
        return host_fail(CKB_ERR_INVALID, "pow2_scale is 0 or 1, the padding field 0");
    if(d->M < 1 || d->N < 1 || d->N > kMaxCols || d->M > kMaxCols || d->ldx < d->N || d->ldq < d->N)
        return host_fail(CKB_ERR_INVALID, "extents must be positive and below 2^31, pitches at least N");
    if(d->scale_stride_m < 0 || d->scale_stride_n < 0)
        return host_fail(CKB_ERR_INVALID, "scale strides must not be negative");
    const int64_t blocks = div_up(d->M, d->block_m == 1 ? 1 : 128) * div_up(d->N, 128);
    if(blocks > 0x7fffffffll)
        return host_fail(CKB_ERR_UNSUPPORTED, "more than 2^31 blocks");
    if(scales_collide(d->scale_stride_m, d->scale_stride_n, div_up(d->M, d->block_m), div_up(d->N, d->block_n)))
        return host_fail(CKB_ERR_INVALID, "every block needs a scale of its own");
    if(need_pointers)
    {
        if(!d->p_x || !d->p_q || !d->p_scale)
            return host_fail(CKB_ERR_INVALID, "null tensor pointer");
        if(!starts_on(d->p_x, wide_bytes(d->x_dtype)) || !starts_on(d->p_scale, 4))
            return host_fail(CKB_ERR_INVALID, "a tensor is not aligned to its elements");
    }
    return CKB_OK;
}

// ---- layer norm -----------------------------------------------------------------------------------
int check_norm_types(int x_dtype, int w_dtype, int64_t M, int64_t N)
{
    if(!is_wide(x_dtype) || (w_dtype != x_dtype && w_dtype != CKB_F32))
        return host_fail(CKB_ERR_UNSUPPORTED, "layer norm works on CKB_BF16, CKB_F16 or CKB_F32 with weights of that type or CKB_F32");
    if(M < 1 || N < 1 || M > kMaxRows || N > kMaxCols)
        return host_fail(CKB_ERR_INVALID, "M and N must be positive, M below 2^40 and N below 2^31");
    return CKB_OK;
}

int check_fwd(const ckb_layernorm_fwd_desc* d, bool need_pointers)
{
    if(!d)
        return host_fail(CKB_ERR_INVALID, "null descriptor");
    if(int rc = check_norm_types(d->x_dtype, d->w_dtype, d->M, d->N))
        return rc;
    if(!(d->eps >= 0.f) || d->eps > 3.402823466e+38f)
        return host_fail(CKB_ERR_INVALID, "eps must be a number that is not negative");
    if(d->ldx < d->N || (d->p_y && d->ldy < d->N) || (d->p_q && d->ldq < d->N))
        return host_fail(CKB_ERR_INVALID, "a pitch is smaller than N");
    if(d->p_q)
    {
        if(!is_f8(d->q_dtype))
            return host_fail(CKB_ERR_UNSUPPORTED, "8-bit output is CKB_F8_E4M3 or CKB_F8_E5M2");
        if(!d->p_q_scale)
            return host_fail(CKB_ERR_INVALID, "8-bit output needs a tensor of scales");
        if(d->q_scale_stride_m < 0 || d->q_scale_stride_n < 0 || scales_collide(d->q_scale_stride_m, d->q_scale_stride_n, d->M, div_up(d->N, 128)))
            return host_fail(CKB_ERR_INVALID, "every block needs a scale of its own");
    }
    if(need_pointers)
    {
        if(!d->p_x || (!d->p_y && !d->p_q))
            return host_fail(CKB_ERR_INVALID, "layer norm needs an input and at least one output");
        const int xb = wide_bytes(d->x_dtype), wb = wide_bytes(d->w_dtype);
        if(!starts_on(d->p_x, xb) || !starts_on(d->p_y, xb) || !starts_on(d->p_gamma, wb) || !starts_on(d->p_beta, wb) ||
           !starts_on(d->p_q_scale, 4) || !starts_on(d->p_mean, 4) || !starts_on(d->p_rstd, 4))
            return host_fail(CKB_ERR_INVALID, "a tensor is not aligned to its elements");
    }
    return CKB_OK;
}

int check_bwd(const ckb_layernorm_bwd_desc* d, bool need_pointers)
{
    if(!d)
        return host_fail(CKB_ERR_INVALID, "null descriptor");
    if(int rc = check_norm_types(d->x_dtype, d->w_dtype, d->M, d->N))
        return rc;
    if(d->lddy < d->N || d->ldx < d->N || (d->p_dx && d->lddx < d->N))
        return host_fail(CKB_ERR_INVALID, "a pitch is smaller than N");
    if(need_pointers)
    {
        if(!d->p_dy || !d->p_x || !d->p_mean || !d->p_rstd || (!d->p_dx && !d->p_dgamma && !d->p_dbeta))
            return host_fail(CKB_ERR_INVALID, "the backward pass needs dy, x, mean, rstd and at least one output");
        const int xb = wide_bytes(d->x_dtype), wb = wide_bytes(d->w_dtype);
        if(!starts_on(d->p_dy, xb) || !starts_on(d->p_x, xb) || !starts_on(d->p_dx, xb) || !starts_on(d->p_gamma, wb) ||
           !starts_on(d->p_dgamma, wb) || !starts_on(d->p_dbeta, wb) || !starts_on(d->p_mean, 4) || !starts_on(d->p_rstd, 4))
            return host_fail(CKB_ERR_INVALID, "a tensor is not aligned to its elements");
    }
    return CKB_OK;
}

constexpr int kBwdRegisterCols = 8192; // longest row whose column sums fit the registers of a CTA

// Threads of a CTA for one row, each with V vectors of eight columns; `lean`: the kernel gets along with 80 registers at
// V = 1, so that 768 threads hold a row that would leave less than 16 warps of V = 2 on an SM.
struct BwdShape
{
    int V, threads;
};
BwdShape bwd_shape(int64_t N, bool lean)
{
    const int vecs = static_cast<int>(div_up(N, 8));
    const int V    = vecs <= 128 || (lean && vecs > 512 && vecs <= 768) ? 1 : 2;
    return {V, static_cast<int>(div_up(div_up(vecs, V), 32) * 32)};
}

// How many sets of rows sum columns on their own; depends on the sizes only, so that the workspace can be asked for
// before the device is known.
int bwd_parts(const ckb_layernorm_bwd_desc* d)
{
    int64_t want;
    if(d->N > kBwdRegisterCols)
        want = div_up(592, div_up(d->N, LONG_SLAB)); // 4 CTAs per SM in all
    else
    {
        // 16 warps per SM; more than 592 CTAs only where each has eight rows (what they sum is read once more)
        const int warps = bwd_shape(d->N, false).threads / 32; // (one CTA per SM where `lean` matters)
        want            = 148 * (warps < 16 ? 16 / warps : 1);
        if(want > 592)
            want = want < d->M / 8 ? want : d->M / 8 > 592 ? d->M / 8 : 592;
    }
    return static_cast<int>(want < d->M ? want : d->M);
}

template <typename T>
cudaError_t launch_bwd(LayernormBwdParams p, cudaStream_t stream)
{
    cudaError_t e   = cudaSuccess;
    const bool sums = p.dgamma || p.dbeta;
    if(p.N > kBwdRegisterCols)
    {
        if(p.dx)
        {
            e = p.vec ? launch(layernorm_bwd_long_kernel<T, true>, p.M < 296 ? p.M : 296, 1, 1024, stream, p)
                      : launch(layernorm_bwd_long_kernel<T, false>, p.M < 296 ? p.M : 296, 1, 1024, stream, p);
            if(e != cudaSuccess)
                return e;
        }
        if(!sums)
            return cudaSuccess;
        e = p.vec ? launch(layernorm_bwd_long_sums_kernel<T, true>, div_up(p.N, LONG_SLAB), p.parts, LONG_SLAB / 8, stream, p)
                  : launch(layernorm_bwd_long_sums_kernel<T, false>, div_up(p.N, LONG_SLAB), p.parts, LONG_SLAB / 8, stream, p);
    }
    else
    {
        if(!sums)
            p.partial = nullptr;
        // 16-bit rows on 16-byte boundaries as they lie, others shifted out of whole pieces; 32-bit rows column by column
        // (8192 x 4096: 96 us, shifted out of pieces 94; x 5120: 119 and 145; x 511: 107, x 512 in vectors 109)
        const bool lean    = sizeof(T) == 4 || p.vec;
        const BwdShape s   = bwd_shape(p.N, lean);
        const int threads  = s.threads;
        auto aligned       = [&](auto v, auto tail) {
            constexpr int V     = decltype(v)::value;
            constexpr bool TAIL = decltype(tail)::value;
            if constexpr(sizeof(T) == 4)
                return launch(layernorm_bwd_kernel<T, V, true, TAIL>, p.parts, 1, threads, stream, p);
            else
                return launch_big<&layernorm_bwd_kernel<T, V, false, TAIL>>(p.parts, threads, stream, p, RowRing<T, 2 * V>::bytes(threads));
        };
        auto either = [&](auto v) {
            const bool tail = sizeof(T) == 4 ? p.N < 8 * s.V * threads : p.N % 8 != 0;
            return tail ? aligned(v, std::true_type{}) : aligned(v, std::false_type{});
        };
        if(lean)
            e = s.V == 1 ? either(std::integral_constant<int, 1>{}) : either(std::integral_constant<int, 2>{});
        else if constexpr(sizeof(T) == 2)
            e = s.V == 1 ? launch_big<&layernorm_bwd_shifted_kernel<T, 1>>(p.parts, threads, stream, p, 2 * WarpRing<T, 256>::bytes(threads))
                         : launch_big<&layernorm_bwd_shifted_kernel<T, 2>>(p.parts, threads, stream, p, 2 * WarpRing<T, 512>::bytes(threads));
    }
    if(e != cudaSuccess || !sums)
        return e;
    return launch(layernorm_bwd_finish_kernel<T>, div_up(p.N, 32), 2, 1024, stream, p);
}

} // namespace

extern "C" {

int ckb_block_quantize_supported(const ckb_block_quantize_desc* d) { return check_quantize(d, false); }

int ckb_block_quantize_run(const ckb_block_quantize_desc* d, void* stream_, int n_rep, float* avg_ms)
{
    if(int rc = check_quantize(d, true))
        return rc;
    HostDevice dev;
    if(int rc = host_device(&dev))
        return rc;
    if(int rc = check_pointers({{d->p_x, "x"}, {d->p_q, "q"}, {d->p_scale, "scale"}}))
        return rc;
    const int xb = wide_bytes(d->x_dtype);
    QuantizeParams p;
    memset(&p, 0, sizeof(p));
    p.x = d->p_x, p.q = static_cast<uint8_t*>(d->p_q), p.scale = d->p_scale;
    p.ldx = d->ldx, p.ldq = d->ldq, p.ss_m = d->scale_stride_m, p.ss_n = d->scale_stride_n;
    p.M = static_cast<int32_t>(d->M), p.N = static_cast<int32_t>(d->N);
    p.blocks_n = static_cast<int32_t>(div_up(d->N, 128));
    if(p.blocks_n > 1)
    {
        // quotient by blocks_n of a 31-bit number as multiply-high and shift: p = 31 + ceil(log2), mul = ceil(2^p / n)
        uint32_t l = 0;
        while((1ull << l) < static_cast<uint64_t>(p.blocks_n))
            ++l;
        p.div_mul = static_cast<uint32_t>(((1ull << (31 + l)) + p.blocks_n - 1) / p.blocks_n);
        p.div_shr = l - 1;
    }
    p.total = static_cast<int32_t>(div_up(d->M, d->block_m == 1 ? 1 : 128) * p.blocks_n);
    p.pow2  = d->pow2_scale;
    const bool vec = starts_on(d->p_x, 16) && d->ldx * xb % 16 == 0 && starts_on(d->p_q, 8) && d->ldq % 8 == 0;
    p.qmax  = qmax_of(d->q_dtype);
    p.qmax_recip = 1.f / p.qmax;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    const bool rows = d->block_m == 1, square = d->block_n == 128;
    const int64_t want = rows ? div_up(p.total, 16 * QB) : p.total;
    const int64_t most = static_cast<int64_t>(dev.sm_count) * (rows ? 8 * 16 : 64);
    const int64_t grid = want < most ? want : most;
    host_note_plan("block_quantize %dx%d grid=%lld vec=%d", d->block_m, d->block_n, static_cast<long long>(grid), vec);
    auto once = [&]() {
        return with_type(d->x_dtype, [&](auto t) {
            using T   = decltype(t);
            auto both = [&](auto e5) {
                constexpr bool E5 = decltype(e5)::value;
                auto aligned      = [&](auto v) {
                    constexpr bool VEC = decltype(v)::value;
                    if(rows)
                        return launch(quantize_rows_kernel<T, E5, VEC>, grid, 1, 256, stream, p);
                    return square ? launch(quantize_tile_kernel<T, E5, true, VEC>, grid, 1, 256, stream, p)
                                  : launch(quantize_tile_kernel<T, E5, false, VEC>, grid, 1, 256, stream, p);
                };
                return vec ? aligned(Flag<true>{}) : aligned(Flag<false>{});
            };
            return d->q_dtype == CKB_F8_E5M2 ? both(Flag<true>{}) : both(Flag<false>{});
        });
    };
    return host_run_timed(once, 1, stream, n_rep, avg_ms);
}

int ckb_layernorm_fwd_supported(const ckb_layernorm_fwd_desc* d) { return check_fwd(d, false); }

int ckb_layernorm_fwd_run(const ckb_layernorm_fwd_desc* d, void* stream_, int n_rep, float* avg_ms)
{
    if(int rc = check_fwd(d, true))
        return rc;
    HostDevice dev;
    if(int rc = host_device(&dev))
        return rc;
    if(int rc = check_pointers({{d->p_x, "x"}, {d->p_gamma, "gamma"}, {d->p_beta, "beta"}, {d->p_y, "y"}, {d->p_q, "q"},
                                {d->p_q_scale, "the scale of q"}, {d->p_mean, "mean"}, {d->p_rstd, "rstd"}}))
        return rc;
    const int xb = wide_bytes(d->x_dtype);
    LayernormFwdParams p;
    memset(&p, 0, sizeof(p));
    p.x = d->p_x, p.gamma = d->p_gamma, p.beta = d->p_beta, p.y = d->p_y, p.q = static_cast<uint8_t*>(d->p_q);
    p.q_scale = d->p_q_scale, p.mean = d->p_mean, p.rstd = d->p_rstd;
    p.ldx = d->ldx, p.ldy = d->ldy, p.ldq = d->ldq, p.ss_m = d->q_scale_stride_m, p.ss_n = d->q_scale_stride_n;
    p.M = d->M, p.N = static_cast<int32_t>(d->N);
    p.w_f32 = d->w_dtype == CKB_F32;
    p.x_vec = starts_on(d->p_x, 16) && d->ldx * xb % 16 == 0;
    p.y_vec = starts_on(d->p_y, 16) && d->ldy * xb % 16 == 0;
    p.q_vec = starts_on(d->p_q, 16) && d->ldq % 16 == 0;
    p.w_vec = starts_on(d->p_gamma, 16) && starts_on(d->p_beta, 16);
    p.eps   = d->eps;
    p.qmax  = qmax_of(d->q_dtype);
    p.qmax_recip = 1.f / p.qmax;
    // A row of up to 1024 values per warp, of up to 8192 per part of a CTA, of up to 16384 per CTA in registers, longer
    // ones read again from L2.
    const int64_t units = div_up(d->N, 16);
    const bool warp = d->N <= 1024, lng = d->N > 16384, wide = d->N > 8192;
    // a CTA that gets one row has nothing to gain from weights in shared memory: twice the threads, everything direct
    // (7 rows of 4096: 3.4 us, 5.0 the other way)
    const bool few  = !warp && !wide && d->M <= dev.sm_count;
    const int U     = few || (warp && units <= 32) ? 1 : 2;
    p.tpr           = warp ? 32 : lng ? 1024 : static_cast<int>(div_up(div_up(units, U), 32) * 32);
    // parts of a CTA: 768 threads at most, rows and weights within shared memory, and no more than there are rows for
    const int ring = STAGE_DEPTH * (U * 512 * xb + 16) * (p.tpr / 32), weights = 2 * U * 16 * 4 * p.tpr;
    int parts      = warp ? 8 : 1;
    if(!warp && !wide && !few)
    {
        const int64_t rows = div_up(d->M, dev.sm_count);
        while(parts < 8 && (parts + 1) * p.tpr <= 768 && (parts + 1) * ring + weights <= kMaxSmem && parts < rows)
            ++parts;
    }
    const int threads  = parts * p.tpr;
    const int smem     = lng ? 0 : parts * ring + (warp || wide || few ? 0 : weights);
    p.w_offset         = parts * ring;
    const int64_t want = div_up(d->M, parts);
    const int64_t most = static_cast<int64_t>(dev.sm_count) * (lng ? 2 : warp ? 4 : 1);
    const int64_t grid = want < most ? want : most;
    host_note_plan("layernorm_fwd %s threads=%d vectors=%d grid=%lld vec=%d", warp ? "warp" : lng ? "long" : "cta", threads, 2 * U,
                   static_cast<long long>(grid), p.x_vec);
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    auto once = [&]() {
        return with_type(d->x_dtype, [&](auto t) {
            using T   = decltype(t);
            auto both = [&](auto e5) {
                constexpr bool E5 = decltype(e5)::value;
                if(lng)
                    return launch(layernorm_fwd_long_kernel<T, E5>, grid, 1, threads, stream, p);
                if(warp)
                    return U == 1 ? launch_big<&layernorm_fwd_kernel<T, E5, 1, ROW_WARP>>(grid, threads, stream, p, smem)
                                  : launch_big<&layernorm_fwd_kernel<T, E5, 2, ROW_WARP>>(grid, threads, stream, p, smem);
                if(few)
                    return launch_big<&layernorm_fwd_kernel<T, E5, 1, ROW_CTA>>(grid, threads, stream, p, smem);
                return wide ? launch_big<&layernorm_fwd_kernel<T, E5, 2, ROW_CTA>>(grid, threads, stream, p, smem)
                            : launch_big<&layernorm_fwd_kernel<T, E5, 2, ROW_GROUP>>(grid, threads, stream, p, smem);
            };
            return d->p_q && d->q_dtype == CKB_F8_E5M2 ? both(Flag<true>{}) : both(Flag<false>{});
        });
    };
    return host_run_timed(once, 1, stream, n_rep, avg_ms);
}

int ckb_layernorm_bwd_supported(const ckb_layernorm_bwd_desc* d) { return check_bwd(d, false); }

int ckb_layernorm_bwd_workspace_size(const ckb_layernorm_bwd_desc* d, size_t* bytes)
{
    if(int rc = check_bwd(d, false))
        return rc;
    if(!bytes)
        return host_fail(CKB_ERR_INVALID, "null output pointer");
    *bytes = d->p_dgamma || d->p_dbeta ? static_cast<size_t>(2) * bwd_parts(d) * d->N * sizeof(float) : 0;
    return CKB_OK;
}

int ckb_layernorm_bwd_run(const ckb_layernorm_bwd_desc* d, void* workspace, size_t workspace_bytes, void* stream_, int n_rep, float* avg_ms)
{
    if(int rc = check_bwd(d, true))
        return rc;
    size_t need = 0;
    if(int rc = ckb_layernorm_bwd_workspace_size(d, &need))
        return rc;
    if(need > 0 && (!workspace || workspace_bytes < need || !starts_on(workspace, 16)))
        return host_fail(CKB_ERR_WORKSPACE, "the backward pass needs %zu bytes of 16-byte aligned device workspace, got %zu", need,
                         workspace ? workspace_bytes : 0);
    HostDevice dev;
    if(int rc = host_device(&dev))
        return rc;
    if(int rc = check_pointers({{d->p_dy, "dy"}, {d->p_x, "x"}, {d->p_gamma, "gamma"}, {d->p_mean, "mean"}, {d->p_rstd, "rstd"},
                                {d->p_dx, "dx"}, {d->p_dgamma, "dgamma"}, {d->p_dbeta, "dbeta"}, {workspace, "the workspace"}}))
        return rc;
    const int xb = wide_bytes(d->x_dtype);
    LayernormBwdParams p;
    memset(&p, 0, sizeof(p));
    p.dy = d->p_dy, p.x = d->p_x, p.gamma = d->p_gamma, p.mean = d->p_mean, p.rstd = d->p_rstd;
    p.dx = d->p_dx, p.dgamma = d->p_dgamma, p.dbeta = d->p_dbeta;
    p.partial = static_cast<float*>(workspace);
    p.lddy = d->lddy, p.ldx = d->ldx, p.lddx = d->lddx;
    p.M = d->M, p.N = static_cast<int32_t>(d->N);
    p.parts = bwd_parts(d);
    p.w_f32 = d->w_dtype == CKB_F32;
    p.w_vec = starts_on(d->p_gamma, 16);
    p.vec   = starts_on(d->p_dy, 16) && starts_on(d->p_x, 16) && starts_on(d->p_dx, 16) && d->lddy * xb % 16 == 0 && d->ldx * xb % 16 == 0 &&
            (!d->p_dx || d->lddx * xb % 16 == 0);
    const bool lng  = d->N > kBwdRegisterCols, sums = d->p_dgamma || d->p_dbeta;
    const int count = lng ? (d->p_dx ? 1 : 0) + (sums ? 2 : 0) : 1 + (sums ? 1 : 0);
    host_note_plan("layernorm_bwd %s parts=%d vec=%d", lng ? "long" : "cta", p.parts, p.vec);
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    auto once = [&]() { return with_type(d->x_dtype, [&](auto t) { return launch_bwd<decltype(t)>(p, stream); }); };
    return host_run_timed(once, count, stream, n_rep, avg_ms);
}

} // extern "C"
