// Row and block kernels around the 8-bit products: block quantizer, layer norm forward and backward.
//
// All three are bound by memory: one read of the input, one write of the output, with the values between the two held
// in registers.  A thread works on vectors of 8 consecutive values (16 bytes of a 16-bit type); 16 neighbouring lanes
// hold the 128 values of a scale block, so its largest magnitude takes four shuffles.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "../../include/ckb200.h"
#include "ckb_ptx.cuh"

namespace ckb {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight consecutive values as they lie in memory.
template <typename T>
struct alignas(16) Vec8
{
    T v[8];
};

// `n` = values that exist (<= 0: none, the vector is zero); `vec`: p is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load8(Vec8<T>& r, const T* p, int n, bool vec)
{
    if(vec && n >= 8)
    {
        uint4* d       = reinterpret_cast<uint4*>(&r);
        const uint4* s = reinterpret_cast<const uint4*>(p);
#pragma unroll
        for(int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
            d[i] = __ldg(s + i);
    }
    else
    {
#pragma unroll
        for(int i = 0; i < 8; ++i)
            r.v[i] = i < n ? p[i] : from_f32<T>(0.f);
    }
}
template <typename T>
__device__ __forceinline__ void store8(const float (&f)[8], T* p, int n, bool vec)
{
    if(vec && n >= 8)
    {
        Vec8<T> r;
#pragma unroll
        for(int i = 0; i < 8; ++i)
            r.v[i] = from_f32<T>(f[i]);
        const uint4* s = reinterpret_cast<const uint4*>(&r);
#pragma unroll
        for(int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
            reinterpret_cast<uint4*>(p)[i] = s[i];
    }
    else
    {
#pragma unroll
        for(int i = 0; i < 8; ++i)
            if(i < n)
                p[i] = from_f32<T>(f[i]);
    }
}

// ---- 8-bit blocks ------------------------------------------------------------------------------
// Magnitudes are compared as bit patterns: NaN > infinity > numbers, so neither is lost in the maximum.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ float block_scale(uint32_t amax_bits, float qmax, bool pow2)
{
    if(amax_bits == 0)
        return 1.f;
    float s = __fdiv_rn(__uint_as_float(amax_bits), qmax);
    if(s < 1.17549435e-38f) // the smallest normal number: its reciprocal still exists (NaN passes)
        s = 1.17549435e-38f;
    if(pow2)
    {
        const uint32_t b = __float_as_uint(s);
        if((b & 0x7fffffu) != 0 && b < 0x7f800000u) // not a power of two, infinity and NaN stay
            s = __uint_as_float((b & 0x7f800000u) + 0x800000u);
    }
    return s;
}

// x / scale, correctly rounded, without a division per value: with r = 1 / scale rounded, q0 = x r,
// q = q0 + (x - q0 scale) r is the rounded quotient (P. Markstein, IBM J. Res. Dev. 34, 1990) as long as neither
// quotient nor remainder leaves the normal range.  Where a quotient matters to the 8-bit value (>= 2^-18) that holds for
// scales from 2^-80 to 2^120; other blocks divide.
struct BlockDivisor
{
    float scale, recip;
    bool fast;
    __device__ __forceinline__ explicit BlockDivisor(float s)
        : scale(s), recip(0.f), fast(s >= 8.27180613e-25f && s <= 1.32922800e+36f)
    {
        if(fast)
            recip = __frcp_rn(s);
    }
};
__device__ __forceinline__ uint64_t div_pair(uint64_t x, uint64_t nscale, uint64_t recip)
{
    const uint64_t q0 = mul_f32x2(x, recip);
    return fma_f32x2(fma_f32x2(q0, nscale, x), recip, q0);
}

template <bool E5M2>
__device__ __forceinline__ uint32_t to_f8x2(float lo, float hi)
{
    return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, E5M2 ? __NV_E5M2 : __NV_E4M3);
}

// Eight values over one scale -> eight bytes.
template <bool E5M2>
__device__ __forceinline__ uint2 quantize8(const float (&f)[8], const BlockDivisor& d)
{
    uint32_t w[4];
    if(d.fast)
    {
        const uint64_t ns = pack_f32x2(-d.scale, -d.scale), r = pack_f32x2(d.recip, d.recip);
#pragma unroll
        for(int i = 0; i < 4; ++i)
        {
            float lo, hi;
            unpack_f32x2(div_pair(pack_f32x2(f[2 * i], f[2 * i + 1]), ns, r), lo, hi);
            w[i] = to_f8x2<E5M2>(lo, hi);
        }
    }
    else
    {
#pragma unroll
        for(int i = 0; i < 4; ++i)
            w[i] = to_f8x2<E5M2>(__fdiv_rn(f[2 * i], d.scale), __fdiv_rn(f[2 * i + 1], d.scale));
    }
    return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
}

__device__ __forceinline__ void store_q8(uint2 w, uint8_t* p, int n, bool vec)
{
    if(vec && n >= 8)
        *reinterpret_cast<uint2*>(p) = w;
    else
    {
#pragma unroll
        for(int i = 0; i < 8; ++i)
            if(i < n)
                p[i] = static_cast<uint8_t>((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
    }
}

__device__ __forceinline__ uint32_t max16(uint32_t v) // over 16 neighbouring lanes
{
#pragma unroll
    for(int d = 8; d >= 1; d >>= 1)
        v = max(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}

struct QuantizeParams
{
    const void* x;
    uint8_t* q;
    float* scale;
    int64_t ldx, ldq, ss_m, ss_n;
    int32_t M, N;
    int32_t blocks_n; // blocks of 128 columns
    uint32_t div_mul, div_shr; // quotient by blocks_n (see FastDiv); mul = 0: blocks_n = 1
    int32_t total;    // blocks (1 x 128), or tiles of 128 x 128
    int32_t pow2;
    int32_t x_vec, q_vec;
    float qmax;
};
__device__ __forceinline__ int32_t block_row(const QuantizeParams& p, int32_t b)
{
    return p.div_mul == 0 ? b : static_cast<int32_t>(__umulhi(static_cast<uint32_t>(b), p.div_mul) >> p.div_shr);
}

// Blocks of 1 x 128: 16 lanes per block, QB blocks per thread in flight.
constexpr int QB = 4;
template <typename T, bool E5M2>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const __grid_constant__ QuantizeParams P)
{
    grid_dependency_wait();
    grid_launch_dependents();
    const T* x     = static_cast<const T*>(P.x);
    const int sub  = threadIdx.x & 15;
    const int unit = threadIdx.x >> 4; // 16 per CTA
    for(int64_t base = static_cast<int64_t>(blockIdx.x) * (16 * QB); base < P.total; base += static_cast<int64_t>(gridDim.x) * (16 * QB))
    {
        Vec8<T> raw[QB];
        int row[QB], c0[QB], n[QB];
#pragma unroll
        for(int j = 0; j < QB; ++j)
        {
            const int64_t b = base + j * 16 + unit;
            const bool on   = b < P.total;
            row[j]          = on ? block_row(P, static_cast<int32_t>(b)) : 0;
            c0[j]           = on ? (static_cast<int32_t>(b) - row[j] * P.blocks_n) * 128 + sub * 8 : 0;
            n[j]            = on ? P.N - c0[j] : -1000;
            load8(raw[j], x + row[j] * P.ldx + c0[j], n[j], P.x_vec != 0);
        }
#pragma unroll
        for(int j = 0; j < QB; ++j)
        {
            float f[8];
            uint32_t m = 0;
#pragma unroll
            for(int i = 0; i < 8; ++i)
            {
                f[i] = to_f32(raw[j].v[i]);
                m    = max(m, magnitude(f[i]));
            }
            const float s = block_scale(max16(m), P.qmax, P.pow2 != 0);
            if(n[j] <= -1000)
                continue; // (all 16 lanes of the block)
            const uint2 w = quantize8<E5M2>(f, BlockDivisor(s));
            store_q8(w, P.q + row[j] * P.ldq + c0[j], n[j], P.q_vec != 0);
            if(sub == 0)
                P.scale[row[j] * P.ss_m + (c0[j] >> 7) * P.ss_n] = s;
        }
    }
}

// Blocks of 128 x 128 (SQUARE) or 128 x 1: a CTA holds 128 rows x 128 columns in registers, 8 rows x 8 columns a
// thread.  Row r of the tile belongs to threads 16 (r mod 16) .. + 15.
template <typename T, bool E5M2, bool SQUARE>
__global__ void __launch_bounds__(256) quantize_tile_kernel(const __grid_constant__ QuantizeParams P)
{
    grid_dependency_wait();
    grid_launch_dependents();
    __shared__ uint32_t s_max[SQUARE ? 16 : 16 * 128];
    const T* x     = static_cast<const T*>(P.x);
    const int sub  = threadIdx.x & 15;
    const int unit = threadIdx.x >> 4;
    for(int b = blockIdx.x; b < P.total; b += gridDim.x)
    {
        const int br = block_row(P, b);
        const int bc = b - br * P.blocks_n;
        const int c0 = bc * 128 + sub * 8, n = P.N - c0;
        Vec8<T> raw[8];
#pragma unroll
        for(int i = 0; i < 8; ++i)
        {
            const int r = br * 128 + i * 16 + unit;
            load8(raw[i], x + r * P.ldx + c0, r < P.M ? n : 0, P.x_vec != 0);
        }
        float scale[8];
        if constexpr(SQUARE)
        {
            uint32_t m = 0;
#pragma unroll
            for(int i = 0; i < 8; ++i)
#pragma unroll
                for(int k = 0; k < 8; ++k)
                    m = max(m, magnitude(to_f32(raw[i].v[k])));
            m = max16(m);
            if(sub == 0)
                s_max[unit] = m;
            __syncthreads();
            m        = max16(s_max[sub]);
            scale[0] = block_scale(m, P.qmax, P.pow2 != 0);
            if(threadIdx.x == 0)
                P.scale[br * P.ss_m + bc * P.ss_n] = scale[0];
        }
        else
        {
#pragma unroll
            for(int k = 0; k < 8; ++k)
            {
                uint32_t m = 0;
#pragma unroll
                for(int i = 0; i < 8; ++i)
                    m = max(m, magnitude(to_f32(raw[i].v[k])));
                s_max[unit * 128 + k * 16 + sub] = m; // [unit][k][sub]: lanes write neighbouring words
            }
            __syncthreads();
#pragma unroll
            for(int k = 0; k < 8; ++k)
            {
                // every thread needs the scales of its own eight columns
                uint32_t m = 0;
#pragma unroll
                for(int u = 0; u < 16; ++u)
                    m = max(m, s_max[u * 128 + k * 16 + sub]);
                scale[k] = block_scale(m, P.qmax, P.pow2 != 0);
                if(unit == 0 && k < n)
                    P.scale[br * P.ss_m + (c0 + k) * P.ss_n] = scale[k];
            }
        }
#pragma unroll
        for(int i = 0; i < 8; ++i)
        {
            const int r = br * 128 + i * 16 + unit;
            if(r >= P.M)
                break;
            float f[8];
#pragma unroll
            for(int k = 0; k < 8; ++k)
                f[k] = to_f32(raw[i].v[k]);
            uint2 w;
            if constexpr(SQUARE)
                w = quantize8<E5M2>(f, BlockDivisor(scale[0]));
            else
            {
                uint32_t h[4];
#pragma unroll
                for(int k = 0; k < 8; k += 2)
                    h[k / 2] = to_f8x2<E5M2>(__fdiv_rn(f[k], scale[k]), __fdiv_rn(f[k + 1], scale[k + 1]));
                w = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
            }
            store_q8(w, P.q + r * P.ldq + c0, n, P.q_vec != 0);
        }
        __syncthreads(); // s_max is used again
    }
}

// ---- layer norm -----------------------------------------------------------------------------------
__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for(int d = 16; d >= 1; d >>= 1)
        v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

// Sums of two values over the threads of a row; `buf` holds 2 x 32 words per use, a __syncthreads lies between two
// uses of the same words.  WARP: the row belongs to one warp.
template <bool WARP>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* buf)
{
    a = warp_sum(a);
    b = warp_sum(b);
    if constexpr(!WARP)
    {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
        if(lane == 0)
        {
            buf[warp]      = a;
            buf[32 + warp] = b;
        }
        __syncthreads();
        a = warp_sum(lane < warps ? buf[lane] : 0.f);
        b = warp_sum(lane < warps ? buf[32 + lane] : 0.f);
    }
}

// From the mean square and the mean of the distances to the first mean.
__device__ __forceinline__ float rstd_of(float square, float shift, float eps)
{
    const float var = __fmaf_rn(-shift, shift, square);
    return __frsqrt_rn((var < 0.f ? 0.f : var) + eps); // (a NaN stays one)
}

struct LayernormFwdParams
{
    const void *x, *gamma, *beta;
    void* y;
    uint8_t* q;
    float *q_scale, *mean, *rstd;
    int64_t ldx, ldy, ldq, ss_m, ss_n;
    int64_t M;
    int32_t N;
    int32_t w_f32, x_vec, y_vec, q_vec, w_vec;
    float eps, qmax;
};

// Weights of columns c .. c + 7 (or every `step`-th from c) in 32 bits.
template <typename T>
__device__ __forceinline__ void load_weights8(float (&f)[8], const void* w, bool f32, int c, int N, bool vec, float none)
{
    if(!w)
    {
#pragma unroll
        for(int i = 0; i < 8; ++i)
            f[i] = none;
    }
    else if(f32)
    {
        Vec8<float> r;
        load8(r, static_cast<const float*>(w) + c, N - c, vec);
#pragma unroll
        for(int i = 0; i < 8; ++i)
            f[i] = r.v[i];
    }
    else
    {
        Vec8<T> r;
        load8(r, static_cast<const T*>(w) + c, N - c, vec);
#pragma unroll
        for(int i = 0; i < 8; ++i)
            f[i] = to_f32(r.v[i]);
    }
}

// y (and q) of 8 columns from their distances to the mean.
template <typename T, bool E5M2>
__device__ __forceinline__ void layernorm_out8(const LayernormFwdParams& P, int64_t row, int c, float (&d)[8], float rstd)
{
    const int n = P.N - c;
    float g[8], b[8];
    load_weights8<T>(g, P.gamma, P.w_f32 != 0, c, P.N, P.w_vec != 0, 1.f);
    load_weights8<T>(b, P.beta, P.w_f32 != 0, c, P.N, P.w_vec != 0, 0.f);
#pragma unroll
    for(int i = 0; i < 8; ++i)
        d[i] = __fmaf_rn(d[i] * rstd, g[i], b[i]);
    if(P.y)
        store8(d, static_cast<T*>(P.y) + row * P.ldy + c, n, P.y_vec != 0);
    if(P.q)
    {
        uint32_t m = 0;
#pragma unroll
        for(int i = 0; i < 8; ++i)
            m = max(m, i < n ? magnitude(d[i]) : 0u);
        const float s = block_scale(max16(m), P.qmax, false);
        const uint2 w = quantize8<E5M2>(d, BlockDivisor(s));
        store_q8(w, P.q + row * P.ldq + c, n, P.q_vec != 0);
        if((threadIdx.x & 15) == 0 && n > 0)
            P.q_scale[row * P.ss_m + (c >> 7) * P.ss_n] = s;
    }
}

// A row per warp (WARP, eight rows a CTA) or per CTA, V vectors of 8 values a thread: vector v of thread t holds columns
// 8 (v * threads + t) .. + 7.  The next row's values are on their way while this one is worked on.
// Mean and variance in two passes over the registers; the second pass also sums the distances themselves, which takes
// the rounding of the first mean out of both.
template <typename T, bool E5M2, int V, bool WARP>
__global__ void __launch_bounds__(WARP || V == 2 ? 256 : 512) layernorm_fwd_kernel(const __grid_constant__ LayernormFwdParams P)
{
    grid_dependency_wait();
    grid_launch_dependents();
    __shared__ float buf[4 * 64];
    const int tpr      = WARP ? 32 : static_cast<int>(blockDim.x);
    const int t        = WARP ? static_cast<int>(threadIdx.x) & 31 : static_cast<int>(threadIdx.x);
    const int64_t step = WARP ? static_cast<int64_t>(gridDim.x) * 8 : gridDim.x;
    int64_t row        = WARP ? static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5) : blockIdx.x;
    const T* x         = static_cast<const T*>(P.x);
    const float inv_n  = 1.f / static_cast<float>(P.N);
    Vec8<T> raw[V];
    auto fetch = [&](int64_t r) {
#pragma unroll
        for(int v = 0; v < V; ++v)
        {
            const int c = (v * tpr + t) * 8;
            load8(raw[v], x + r * P.ldx + c, r < P.M ? P.N - c : 0, P.x_vec != 0);
        }
    };
    fetch(row);
    int flip = 0;
    for(; row < P.M; row += step)
    {
        float d[V][8];
        float sum = 0.f, none = 0.f;
#pragma unroll
        for(int v = 0; v < V; ++v)
        {
            float part = 0.f;
#pragma unroll
            for(int i = 0; i < 8; ++i)
            {
                d[v][i] = to_f32(raw[v].v[i]);
                part += d[v][i];
            }
            sum += part;
        }
        fetch(row + step);
        row_sum2<WARP>(sum, none, buf + flip);
        float mean = sum * inv_n;
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for(int v = 0; v < V; ++v)
        {
            const int n = P.N - (v * tpr + t) * 8;
#pragma unroll
            for(int i = 0; i < 8; ++i)
            {
                d[v][i] = i < n ? d[v][i] - mean : 0.f;
                s1 += d[v][i];
                s2 = __fmaf_rn(d[v][i], d[v][i], s2);
            }
        }
        row_sum2<WARP>(s1, s2, buf + 64 + flip);
        const float shift = s1 * inv_n;
        const float rstd  = rstd_of(s2 * inv_n, shift, P.eps);
        mean += shift;
        if(t == 0)
        {
            if(P.mean)
                P.mean[row] = mean;
            if(P.rstd)
                P.rstd[row] = rstd;
        }
#pragma unroll
        for(int v = 0; v < V; ++v)
        {
            if(__all_sync(0xffffffffu, P.N - (v * tpr + t) * 8 <= 0))
                continue;
#pragma unroll
            for(int i = 0; i < 8; ++i)
                d[v][i] -= shift;
            layernorm_out8<T, E5M2>(P, row, (v * tpr + t) * 8, d[v], rstd);
        }
        flip ^= 128;
    }
}

// Rows that do not fit the registers of a CTA: the row is read three times (the second and third time from L2).
template <typename T, bool E5M2>
__global__ void __launch_bounds__(1024) layernorm_fwd_long_kernel(const __grid_constant__ LayernormFwdParams P)
{
    grid_dependency_wait();
    grid_launch_dependents();
    __shared__ float buf[4 * 64];
    const T* x    = static_cast<const T*>(P.x);
    const int t   = threadIdx.x;
    const float n = static_cast<float>(P.N);
    for(int64_t row = blockIdx.x; row < P.M; row += gridDim.x)
    {
        float sum = 0.f, none = 0.f;
        Vec8<T> r;
        for(int64_t c = t * 8; c < P.N; c += 8192)
        {
            load8(r, x + row * P.ldx + c, static_cast<int>(P.N - c), P.x_vec != 0);
            float part = 0.f;
#pragma unroll
            for(int i = 0; i < 8; ++i)
                part += to_f32(r.v[i]);
            sum += part;
        }
        row_sum2<false>(sum, none, buf);
        float mean = sum / n, s1 = 0.f, s2 = 0.f;
        for(int64_t c = t * 8; c < P.N; c += 8192)
        {
            load8(r, x + row * P.ldx + c, static_cast<int>(P.N - c), P.x_vec != 0);
            float p1 = 0.f, p2 = 0.f;
#pragma unroll
            for(int i = 0; i < 8; ++i)
            {
                const float d = c + i < P.N ? to_f32(r.v[i]) - mean : 0.f;
                p1 += d;
                p2 = __fmaf_rn(d, d, p2);
            }
            s1 += p1;
            s2 += p2;
        }
        row_sum2<false>(s1, s2, buf + 64);
        const float shift = s1 / n;
        const float rstd  = rstd_of(s2 / n, shift, P.eps);
        if(t == 0)
        {
            if(P.mean)
                P.mean[row] = mean + shift;
            if(P.rstd)
                P.rstd[row] = rstd;
        }
        for(int64_t c0 = 0; c0 < P.N; c0 += 8192)
        {
            const int64_t c = c0 + t * 8;
            if(__all_sync(0xffffffffu, c >= P.N))
                continue;
            // (a lane behind the row's end takes part in the shuffles with zeros)
            const int cc = c < P.N ? static_cast<int>(c) : P.N;
            load8(r, x + row * P.ldx + cc, P.N - cc, P.x_vec != 0);
            float d[8];
#pragma unroll
            for(int i = 0; i < 8; ++i)
                d[i] = c + i < P.N ? (to_f32(r.v[i]) - mean) - shift : 0.f;
            layernorm_out8<T, E5M2>(P, row, cc, d, rstd);
        }
        __syncthreads(); // buf is used again
    }
}

struct LayernormBwdParams
{
    const void *dy, *x, *gamma;
    const float *mean, *rstd;
    void *dx, *dgamma, *dbeta;
    float* partial; // [2][parts][N]: partial sums of dgamma, then of dbeta
    float* row_sums; // long rows: [2][M] means of w and of w xhat
    int64_t lddy, ldx, lddx;
    int64_t M;
    int32_t N, parts;
    int32_t w_f32, vec, w_vec;
};

// Where element i of vector v of a thread lies.  STRIDED: neighbouring lanes hold neighbouring columns, for rows that
// do not start on 16-byte boundaries.
template <bool STRIDED>
__device__ __forceinline__ int column_of(int v, int i, int t, int tpr)
{
    return STRIDED ? (v * 8 + i) * tpr + t : (v * tpr + t) * 8 + i;
}
template <typename T, bool STRIDED>
__device__ __forceinline__ void load_columns(Vec8<T>& r, const T* row, int v, int t, int tpr, int N, bool on)
{
    if constexpr(STRIDED)
    {
#pragma unroll
        for(int i = 0; i < 8; ++i)
        {
            const int c = column_of<true>(v, i, t, tpr);
            r.v[i]      = on && c < N ? row[c] : from_f32<T>(0.f);
        }
    }
    else
    {
        const int c = column_of<false>(v, 0, t, tpr);
        load8(r, row + c, on ? N - c : 0, true);
    }
}

// dx and the partial sums of dgamma and dbeta in one pass.  A CTA walks rows blockIdx.x, + gridDim.x, ...; a thread keeps
// the same V x 8 columns throughout, so the column sums stay in its registers until the CTA writes them once.
template <typename T, int V, bool STRIDED>
__global__ void __launch_bounds__(V == 1 ? 128 : 512) layernorm_bwd_kernel(const __grid_constant__ LayernormBwdParams P)
{
    grid_dependency_wait();
    grid_launch_dependents();
    __shared__ float buf[2 * 64];
    const int tpr = blockDim.x, t = threadIdx.x;
    const T* x  = static_cast<const T*>(P.x);
    const T* dy = static_cast<const T*>(P.dy);
    const float inv_n = 1.f / static_cast<float>(P.N);
    float g[V][8], dg[V][8], db[V][8];
#pragma unroll
    for(int v = 0; v < V; ++v)
    {
#pragma unroll
        for(int i = 0; i < 8; ++i)
        {
            const int c = column_of<STRIDED>(v, i, t, tpr);
            g[v][i]     = 0.f;
            if(c < P.N)
                g[v][i] = !P.gamma ? 1.f : P.w_f32 ? static_cast<const float*>(P.gamma)[c] : to_f32(static_cast<const T*>(P.gamma)[c]);
            dg[v][i] = db[v][i] = 0.f;
        }
    }
    Vec8<T> rx[V], ry[V];
    float mean = 0.f, rstd = 0.f;
    auto fetch = [&](int64_t r) {
        const bool on = r < P.M;
#pragma unroll
        for(int v = 0; v < V; ++v)
        {
            load_columns<T, STRIDED>(rx[v], x + r * P.ldx, v, t, tpr, P.N, on);
            load_columns<T, STRIDED>(ry[v], dy + r * P.lddy, v, t, tpr, P.N, on);
        }
        mean = on ? __ldg(P.mean + r) : 0.f;
        rstd = on ? __ldg(P.rstd + r) : 0.f;
    };
    int64_t row = blockIdx.x;
    fetch(row);
    int flip = 0;
    for(; row < P.M; row += gridDim.x)
    {
        float h[V][8], w[V][8];
        float s1 = 0.f, s2 = 0.f;
        const float rs = rstd;
#pragma unroll
        for(int v = 0; v < V; ++v)
#pragma unroll
            for(int i = 0; i < 8; ++i)
            {
                const bool in   = STRIDED ? column_of<true>(v, i, t, tpr) < P.N : true; // (elsewhere dy and gamma are zero)
                const float gy  = to_f32(ry[v].v[i]);
                h[v][i]         = in ? (to_f32(rx[v].v[i]) - mean) * rs : 0.f;
                dg[v][i]        = __fmaf_rn(gy, h[v][i], dg[v][i]);
                db[v][i] += gy;
                w[v][i] = gy * g[v][i];
                s1 += w[v][i];
                s2 = __fmaf_rn(w[v][i], h[v][i], s2);
            }
        const int64_t next = row + gridDim.x;
        fetch(next);
        row_sum2<false>(s1, s2, buf + flip);
        flip ^= 64;
        if(P.dx)
        {
            const float c1 = s1 * inv_n, c2 = s2 * inv_n;
            T* out = static_cast<T*>(P.dx) + row * P.lddx;
#pragma unroll
            for(int v = 0; v < V; ++v)
            {
                float o[8];
#pragma unroll
                for(int i = 0; i < 8; ++i)
                    o[i] = rs * (w[v][i] - c1 - h[v][i] * c2);
                if constexpr(STRIDED)
                {
#pragma unroll
                    for(int i = 0; i < 8; ++i)
                    {
                        const int c = column_of<true>(v, i, t, tpr);
                        if(c < P.N)
                            out[c] = from_f32<T>(o[i]);
                    }
                }
                else
                {
                    const int c = column_of<false>(v, 0, t, tpr);
                    store8(o, out + c, P.N - c, true);
                }
            }
        }
    }
    if(P.partial)
    {
        float* pg = P.partial + static_cast<int64_t>(blockIdx.x) * P.N;
        float* pb = pg + static_cast<int64_t>(P.parts) * P.N;
#pragma unroll
        for(int v = 0; v < V; ++v)
#pragma unroll
            for(int i = 0; i < 8; ++i)
            {
                const int c = column_of<STRIDED>(v, i, t, tpr);
                if(c < P.N)
                {
                    pg[c] = dg[v][i];
                    pb[c] = db[v][i];
                }
            }
    }
}

// Long rows, first half: means of w and w xhat of a row, then dx (the row is read twice, the second time from L2).
template <typename T>
__global__ void __launch_bounds__(1024) layernorm_bwd_long_kernel(const __grid_constant__ LayernormBwdParams P)
{
    grid_dependency_wait();
    grid_launch_dependents();
    __shared__ float buf[2 * 64];
    const float n = static_cast<float>(P.N);
    for(int64_t row = blockIdx.x; row < P.M; row += gridDim.x)
    {
        const T* x  = static_cast<const T*>(P.x) + row * P.ldx;
        const T* dy = static_cast<const T*>(P.dy) + row * P.lddy;
        const float mean = P.mean[row], rstd = P.rstd[row];
        auto weight = [&](int64_t c) {
            return !P.gamma ? 1.f : P.w_f32 ? static_cast<const float*>(P.gamma)[c] : to_f32(static_cast<const T*>(P.gamma)[c]);
        };
        float s1 = 0.f, s2 = 0.f;
        for(int64_t c = threadIdx.x; c < P.N; c += 1024)
        {
            const float w = to_f32(dy[c]) * weight(c);
            s1 += w;
            s2 = __fmaf_rn(w, (to_f32(x[c]) - mean) * rstd, s2);
        }
        row_sum2<false>(s1, s2, buf);
        const float c1 = s1 / n, c2 = s2 / n;
        T* out = static_cast<T*>(P.dx) + row * P.lddx;
        for(int64_t c = threadIdx.x; c < P.N; c += 1024)
            out[c] = from_f32<T>(rstd * (to_f32(dy[c]) * weight(c) - c1 - (to_f32(x[c]) - mean) * rstd * c2));
        __syncthreads();
    }
}
// Second half: column sums.  blockIdx.x = 1024 columns, blockIdx.y = one of P.parts sets of rows.
template <typename T>
__global__ void __launch_bounds__(1024) layernorm_bwd_long_sums_kernel(const __grid_constant__ LayernormBwdParams P)
{
    grid_dependency_wait();
    grid_launch_dependents();
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 1024 + threadIdx.x;
    if(c >= P.N)
        return;
    float dg = 0.f, db = 0.f;
    for(int64_t row = blockIdx.y; row < P.M; row += P.parts)
    {
        const float gy = to_f32(static_cast<const T*>(P.dy)[row * P.lddy + c]);
        dg = __fmaf_rn(gy, (to_f32(static_cast<const T*>(P.x)[row * P.ldx + c]) - __ldg(P.mean + row)) * __ldg(P.rstd + row), dg);
        db += gy;
    }
    P.partial[blockIdx.y * static_cast<int64_t>(P.N) + c]             = dg;
    P.partial[(P.parts + blockIdx.y) * static_cast<int64_t>(P.N) + c] = db;
}

// Sums the partial column sums in the order of the parts.  32 columns a CTA, eight threads a column.
template <typename T>
__global__ void __launch_bounds__(256) layernorm_bwd_finish_kernel(const __grid_constant__ LayernormBwdParams P)
{
    grid_dependency_wait();
    grid_launch_dependents();
    __shared__ float part[8][33];
    const int lane = threadIdx.x & 31, slot = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    void* out       = blockIdx.y == 0 ? P.dgamma : P.dbeta;
    const float* in = P.partial + static_cast<int64_t>(blockIdx.y) * P.parts * P.N;
    float sum       = 0.f;
    if(c < P.N && out)
    {
        int p = slot;
        for(; p + 24 < P.parts; p += 32) // four loads in flight
        {
            const float a = in[static_cast<int64_t>(p) * P.N + c], b = in[static_cast<int64_t>(p + 8) * P.N + c];
            const float d = in[static_cast<int64_t>(p + 16) * P.N + c], e = in[static_cast<int64_t>(p + 24) * P.N + c];
            sum += (a + b) + (d + e);
        }
        for(; p < P.parts; p += 8)
            sum += in[static_cast<int64_t>(p) * P.N + c];
    }
    part[slot][lane] = sum;
    __syncthreads();
    if(slot == 0 && c < P.N && out)
    {
#pragma unroll
        for(int s = 1; s < 8; ++s)
            sum += part[s][lane];
        if(P.w_f32)
            static_cast<float*>(out)[c] = sum;
        else
            static_cast<T*>(out)[c] = from_f32<T>(sum);
    }
}

} // namespace ckb
