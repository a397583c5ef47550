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
// Largest magnitude so far; a NaN stays (an infinity is larger than any number anyway), so that neither is lost.
__device__ __forceinline__ float max_abs(float m, float v)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(v)));
    return r;
}
__device__ __forceinline__ float max16(float v) // over 16 neighbouring lanes
{
#pragma unroll
    for(int d = 8; d >= 1; d >>= 1)
        v = max_abs(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}

// amax / qmax, correctly rounded (see below), at least the smallest normal number (its reciprocal still exists).
__device__ __forceinline__ float block_scale(float amax, float qmax, float qmax_recip, bool pow2)
{
    if(amax == 0.f)
        return 1.f;
    float s;
    if(amax >= 1e-28f && amax <= 3.402823466e+38f)
    {
        const float q0 = amax * qmax_recip;
        s              = __fmaf_rn(__fmaf_rn(-q0, qmax, amax), qmax_recip, q0);
    }
    else // tiny, infinite or NaN
    {
        s = __fdiv_rn(amax, qmax);
        if(s < 1.17549435e-38f)
            s = 1.17549435e-38f;
    }
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

// Eight values (four pairs) over one scale -> eight bytes.
template <bool E5M2>
__device__ __forceinline__ uint2 quantize8(const uint64_t (&f)[4], const BlockDivisor& d)
{
    uint32_t w[4];
    if(d.fast)
    {
        const uint64_t ns = pack_f32x2(-d.scale, -d.scale), r = pack_f32x2(d.recip, d.recip);
#pragma unroll
        for(int i = 0; i < 4; ++i)
        {
            float lo, hi;
            unpack_f32x2(div_pair(f[i], ns, r), lo, hi);
            w[i] = to_f8x2<E5M2>(lo, hi);
        }
    }
    else
    {
#pragma unroll
        for(int i = 0; i < 4; ++i)
        {
            float lo, hi;
            unpack_f32x2(f[i], lo, hi);
            w[i] = to_f8x2<E5M2>(__fdiv_rn(lo, d.scale), __fdiv_rn(hi, d.scale));
        }
    }
    return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
}

// The eight values of a vector as pairs, and their largest magnitude.
template <typename T>
__device__ __forceinline__ void to_pairs(const Vec8<T>& r, uint64_t (&f)[4])
{
#pragma unroll
    for(int i = 0; i < 4; ++i)
        f[i] = pack_f32x2(to_f32(r.v[2 * i]), to_f32(r.v[2 * i + 1]));
}
__device__ __forceinline__ float max_abs8(const Vec8<float>& r)
{
    float m = 0.f;
#pragma unroll
    for(int i = 0; i < 8; ++i)
        m = max_abs(m, r.v[i]);
    return m;
}
__device__ __forceinline__ float max_abs8(const Vec8<__half>& r)
{
    const __half2* h = reinterpret_cast<const __half2*>(&r);
    const __half2 m  = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
    return max_abs(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float max_abs8(const Vec8<__nv_bfloat16>& r)
{
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
    const __nv_bfloat162 m  = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
    return max_abs(__low2float(m), __high2float(m));
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
    float qmax, qmax_recip;
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
            const float s = block_scale(max16(max_abs8(raw[j])), P.qmax, P.qmax_recip, P.pow2 != 0);
            if(n[j] <= -1000)
                continue; // (all 16 lanes of the block)
            uint64_t f[4];
            to_pairs(raw[j], f);
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
    __shared__ float s_max[SQUARE ? 16 : 16 * 128];
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
        uint64_t nscale[4], recip[4]; // of this thread's columns (SQUARE: all the same)
        bool fast = true;
        float scale[8];
        if constexpr(SQUARE)
        {
            float m = 0.f;
#pragma unroll
            for(int i = 0; i < 8; ++i)
                m = max_abs(m, max_abs8(raw[i]));
            m = max16(m);
            if(sub == 0)
                s_max[unit] = m;
            __syncthreads();
            m        = max16(s_max[sub]);
            scale[0] = block_scale(m, P.qmax, P.qmax_recip, P.pow2 != 0);
            if(threadIdx.x == 0)
                P.scale[br * P.ss_m + bc * P.ss_n] = scale[0];
        }
        else
        {
#pragma unroll
            for(int k = 0; k < 8; ++k)
            {
                float m = 0.f;
#pragma unroll
                for(int i = 0; i < 8; ++i)
                    m = max_abs(m, to_f32(raw[i].v[k]));
                s_max[unit * 128 + k * 16 + sub] = m; // [unit][k][sub]: lanes write neighbouring words
            }
            __syncthreads();
            if(threadIdx.x < 128)
            {
                float m = 0.f;
#pragma unroll
                for(int u = 0; u < 16; ++u)
                    m = max_abs(m, s_max[u * 128 + threadIdx.x]);
                const float sc = block_scale(m, P.qmax, P.qmax_recip, P.pow2 != 0);
                s_max[threadIdx.x] = sc; // (only this thread reads or writes the column's words now)
                const int k = threadIdx.x >> 4, c = bc * 128 + (threadIdx.x & 15) * 8 + k;
                if(c < P.N)
                    P.scale[br * P.ss_m + c * P.ss_n] = sc;
            }
            __syncthreads();
#pragma unroll
            for(int k = 0; k < 8; ++k)
                scale[k] = s_max[k * 16 + sub];
#pragma unroll
            for(int k = 0; k < 4; ++k)
            {
                const BlockDivisor lo(scale[2 * k]), hi(scale[2 * k + 1]);
                nscale[k] = pack_f32x2(-lo.scale, -hi.scale);
                recip[k]  = pack_f32x2(lo.recip, hi.recip);
                fast      = fast && lo.fast && hi.fast;
            }
        }
#pragma unroll
        for(int i = 0; i < 8; ++i)
        {
            const int r = br * 128 + i * 16 + unit;
            if(r >= P.M)
                break;
            uint64_t f[4];
            to_pairs(raw[i], f);
            uint2 w;
            if constexpr(SQUARE)
                w = quantize8<E5M2>(f, BlockDivisor(scale[0]));
            else
            {
                uint32_t h[4];
#pragma unroll
                for(int k = 0; k < 4; ++k)
                {
                    float lo, hi;
                    if(fast)
                        unpack_f32x2(div_pair(f[k], nscale[k], recip[k]), lo, hi);
                    else
                    {
                        unpack_f32x2(f[k], lo, hi);
                        lo = __fdiv_rn(lo, scale[2 * k]);
                        hi = __fdiv_rn(hi, scale[2 * k + 1]);
                    }
                    h[k] = to_f8x2<E5M2>(lo, hi);
                }
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

// Rows on their way: asynchronous copies into shared memory, DEPTH rows ahead.  Every thread copies the vectors it works
// on itself and reads nobody else's, so only its own copies have to be waited for.  Vector v of thread t lies in pieces of
// 16 bytes, [row of the ring][vector][piece][thread].
constexpr int STAGE_DEPTH = 3;
template <typename T, int V>
struct RowRing
{
    static constexpr int PIECES = sizeof(T) / 2; // 16-byte pieces of a vector
    uint32_t base;                               // this thread's first piece
    int threads;
    static __host__ __device__ int bytes(int threads) { return STAGE_DEPTH * V * PIECES * threads * 16; }
    // `n` = values of the row from the vector's first one on
    __device__ __forceinline__ void copy(int slot, int v, const T* p, int n) const
    {
#pragma unroll
        for(int i = 0; i < PIECES; ++i)
        {
            constexpr int PER = 16 / static_cast<int>(sizeof(T));
            const int have    = n - i * PER < 0 ? 0 : n - i * PER > PER ? PER : n - i * PER;
            copy_async_16(base + (((slot * V + v) * PIECES + i) * threads) * 16, have > 0 ? p + i * PER : p, have * static_cast<int>(sizeof(T)));
        }
    }
    __device__ __forceinline__ void read(Vec8<T>& r, int slot, int v) const
    {
        uint32_t* d = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
        for(int i = 0; i < PIECES; ++i)
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(d[4 * i]), "=r"(d[4 * i + 1]), "=r"(d[4 * i + 2]), "=r"(d[4 * i + 3])
                         : "r"(base + (((slot * V + v) * PIECES + i) * threads) * 16)
                         : "memory");
    }
};

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
    float eps, qmax, qmax_recip;
};

// Weights of columns c .. c + 7 in 32 bits.
template <typename T>
__device__ __forceinline__ void load_weights8(uint64_t (&f)[4], const void* w, bool f32, int c, int N, bool vec, float none)
{
    if(!w)
    {
#pragma unroll
        for(int i = 0; i < 4; ++i)
            f[i] = pack_f32x2(none, none);
    }
    else if(f32)
    {
        Vec8<float> r;
        load8(r, static_cast<const float*>(w) + c, N - c, vec);
        to_pairs(r, f);
    }
    else
    {
        Vec8<T> r;
        load8(r, static_cast<const T*>(w) + c, N - c, vec);
        to_pairs(r, f);
    }
}

// y (and q) of 8 columns from their distances to the mean.
template <typename T, bool E5M2>
__device__ __forceinline__ void layernorm_out8(const LayernormFwdParams& P, int64_t row, int c, uint64_t (&d)[4], float rstd)
{
    const int n = P.N - c;
    uint64_t g[4], b[4];
    load_weights8<T>(g, P.gamma, P.w_f32 != 0, c, P.N, P.w_vec != 0, 1.f);
    load_weights8<T>(b, P.beta, P.w_f32 != 0, c, P.N, P.w_vec != 0, 0.f);
    const uint64_t r2 = pack_f32x2(rstd, rstd);
    float y[8];
#pragma unroll
    for(int i = 0; i < 4; ++i)
    {
        d[i] = fma_f32x2(mul_f32x2(d[i], r2), g[i], b[i]);
        unpack_f32x2(d[i], y[2 * i], y[2 * i + 1]);
    }
    if(P.y)
        store8(y, static_cast<T*>(P.y) + row * P.ldy + c, n, P.y_vec != 0);
    if(P.q)
    {
        float m = 0.f;
#pragma unroll
        for(int i = 0; i < 8; ++i)
            m = max_abs(m, n >= 8 || i < n ? y[i] : 0.f);
        const float s = block_scale(max16(m), P.qmax, P.qmax_recip, false);
        const uint2 w = quantize8<E5M2>(d, BlockDivisor(s));
        store_q8(w, P.q + row * P.ldq + c, n, P.q_vec != 0);
        if((threadIdx.x & 15) == 0 && n > 0)
            P.q_scale[row * P.ss_m + (c >> 7) * P.ss_n] = s;
    }
}

__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float sum_f32x2(uint64_t a)
{
    float lo, hi;
    unpack_f32x2(a, lo, hi);
    return lo + hi;
}
// Subtracts `mean` from the eight values, zero where there is no value (n of them exist).
__device__ __forceinline__ void distances(uint64_t (&d)[4], float mean, int n)
{
    const uint64_t m2 = pack_f32x2(-mean, -mean);
#pragma unroll
    for(int i = 0; i < 4; ++i)
        d[i] = add_f32x2(d[i], m2);
    if(n < 8)
    {
#pragma unroll
        for(int i = 0; i < 4; ++i)
        {
            float lo, hi;
            unpack_f32x2(d[i], lo, hi);
            d[i] = pack_f32x2(2 * i < n ? lo : 0.f, 2 * i + 1 < n ? hi : 0.f);
        }
    }
}

// A row per warp (WARP, eight rows a CTA) or per CTA, V vectors of 8 values a thread: vector v of thread t holds columns
// 8 (v * threads + t) .. + 7.  RING: rows come through shared memory, STAGE_DEPTH - 1 rows ahead (with one row ahead in
// registers three CTAs per SM have 30 KB on their way, half of what the memory needs: 8192 x 5120 took 90 us).
// Mean and variance in two passes over the registers; the second pass also sums the distances themselves, which takes
// the rounding of the first mean out of both.
template <typename T, bool E5M2, int V, bool WARP, bool RING>
__global__ void __launch_bounds__(WARP ? 256 : 512, WARP || V == 4 ? 1 : 2) layernorm_fwd_kernel(const __grid_constant__ LayernormFwdParams P)
{
    grid_dependency_wait();
    grid_launch_dependents();
    extern __shared__ __align__(16) uint8_t ring_smem[];
    __shared__ float buf[4 * 64];
    const int tpr      = WARP ? 32 : static_cast<int>(blockDim.x);
    const int t        = WARP ? static_cast<int>(threadIdx.x) & 31 : static_cast<int>(threadIdx.x);
    const int64_t step = WARP ? static_cast<int64_t>(gridDim.x) * 8 : gridDim.x;
    int64_t row        = WARP ? static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5) : blockIdx.x;
    const T* x         = static_cast<const T*>(P.x);
    const float inv_n  = 1.f / static_cast<float>(P.N);
    Vec8<T> raw[V];
    RowRing<T, V> ring{smem_u32(ring_smem) + t * 16, tpr};
    auto fetch = [&](int64_t r, int slot) {
#pragma unroll
        for(int v = 0; v < V; ++v)
        {
            const int c = (v * tpr + t) * 8, n = r < P.M ? P.N - c : 0;
            const T* p  = x + (n > 0 ? r * P.ldx + c : 0);
            if constexpr(RING)
                ring.copy(slot, v, p, n);
            else
                load8(raw[v], p, n, P.x_vec != 0);
        }
        if constexpr(RING)
            copy_async_commit();
    };
    int slot = 0;
    fetch(row, 0);
    if constexpr(RING)
#pragma unroll
        for(int i = 1; i < STAGE_DEPTH - 1; ++i)
            fetch(row + i * step, i);
    int flip = 0;
    for(; row < P.M; row += step)
    {
        if constexpr(RING)
        {
            fetch(row + (STAGE_DEPTH - 1) * step, slot == 0 ? STAGE_DEPTH - 1 : slot - 1);
            copy_async_wait<STAGE_DEPTH - 1>();
#pragma unroll
            for(int v = 0; v < V; ++v)
                ring.read(raw[v], slot, v);
            if(++slot == STAGE_DEPTH)
                slot = 0;
        }
        uint64_t d[V][4];
        float sum = 0.f, none = 0.f;
#pragma unroll
        for(int v = 0; v < V; ++v)
        {
            to_pairs(raw[v], d[v]);
            sum += sum_f32x2(add_f32x2(add_f32x2(d[v][0], d[v][1]), add_f32x2(d[v][2], d[v][3])));
        }
        if constexpr(!RING)
            fetch(row + step, 0);
        row_sum2<WARP>(sum, none, buf + flip);
        float mean = sum * inv_n;
        uint64_t s1v = 0, s2v = 0;
#pragma unroll
        for(int v = 0; v < V; ++v)
        {
            distances(d[v], mean, P.N - (v * tpr + t) * 8);
#pragma unroll
            for(int i = 0; i < 4; ++i)
            {
                s1v = add_f32x2(s1v, d[v][i]);
                s2v = fma_f32x2(d[v][i], d[v][i], s2v);
            }
        }
        float s1 = sum_f32x2(s1v), s2 = sum_f32x2(s2v);
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
            for(int i = 0; i < 4; ++i)
                d[v][i] = add_f32x2(d[v][i], pack_f32x2(-shift, -shift));
            layernorm_out8<T, E5M2>(P, row, (v * tpr + t) * 8, d[v], rstd);
        }
        flip ^= 128;
    }
    if constexpr(RING)
        copy_async_wait_all();
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
            uint64_t d[4];
            to_pairs(r, d);
            distances(d, mean, P.N - cc);
            distances(d, shift, P.N - cc);
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
template <typename T>
__device__ __forceinline__ void load_columns(Vec8<T>& r, const T* row, int v, int t, int tpr, int N, bool on)
{
#pragma unroll
    for(int i = 0; i < 8; ++i)
    {
        const int c = column_of<true>(v, i, t, tpr);
        r.v[i]      = on && c < N ? row[c] : from_f32<T>(0.f);
    }
}

// dx and the partial sums of dgamma and dbeta in one pass.  A CTA walks rows blockIdx.x, + gridDim.x, ...; a thread keeps
// the same V x 8 columns throughout, so the column sums stay in its registers until the CTA writes them once.  Rows that
// start on 16-byte boundaries come through shared memory (RowRing) and are read from there a second time for dx, which
// keeps xhat and w out of the registers while the row's sums are formed; STRIDED rows one ahead in registers.
template <typename T, int V, bool STRIDED>
__global__ void __launch_bounds__(V == 1 ? 128 : 512, V == 1 ? 4 : 1) layernorm_bwd_kernel(const __grid_constant__ LayernormBwdParams P)
{
    grid_dependency_wait();
    grid_launch_dependents();
    extern __shared__ __align__(16) uint8_t ring_smem[];
    __shared__ float buf[2 * 64];
    const int tpr = blockDim.x, t = threadIdx.x;
    const T* x  = static_cast<const T*>(P.x);
    const T* dy = static_cast<const T*>(P.dy);
    const float inv_n = 1.f / static_cast<float>(P.N);
    uint64_t g[V][4], dg[V][4], db[V][4];
#pragma unroll
    for(int v = 0; v < V; ++v)
    {
        float f[8];
#pragma unroll
        for(int i = 0; i < 8; ++i)
        {
            const int c = column_of<STRIDED>(v, i, t, tpr);
            f[i]        = 0.f;
            if(c < P.N)
                f[i] = !P.gamma ? 1.f : P.w_f32 ? static_cast<const float*>(P.gamma)[c] : to_f32(static_cast<const T*>(P.gamma)[c]);
        }
#pragma unroll
        for(int i = 0; i < 4; ++i)
        {
            g[v][i]  = pack_f32x2(f[2 * i], f[2 * i + 1]);
            dg[v][i] = db[v][i] = 0;
        }
    }
    Vec8<T> rx[V], ry[V];
    RowRing<T, 2 * V> ring{smem_u32(ring_smem) + t * 16, tpr}; // vectors of x, then of dy
    float mean = 0.f, rstd = 0.f;
    auto fetch = [&](int64_t r, int slot) {
        const bool on = r < P.M;
#pragma unroll
        for(int v = 0; v < V; ++v)
        {
            if constexpr(STRIDED)
            {
                load_columns<T>(rx[v], x + (on ? r * P.ldx : 0), v, t, tpr, P.N, on);
                load_columns<T>(ry[v], dy + (on ? r * P.lddy : 0), v, t, tpr, P.N, on);
            }
            else
            {
                const int c = (v * tpr + t) * 8, n = on ? P.N - c : 0;
                ring.copy(slot, v, x + (n > 0 ? r * P.ldx + c : 0), n);
                ring.copy(slot, V + v, dy + (n > 0 ? r * P.lddy + c : 0), n);
            }
        }
        if constexpr(!STRIDED)
            copy_async_commit();
    };
    auto statistics = [&](int64_t r) {
        mean = r < P.M ? __ldg(P.mean + r) : 0.f;
        rstd = r < P.M ? __ldg(P.rstd + r) : 0.f;
    };
    int64_t row = blockIdx.x;
    int slot    = 0;
    fetch(row, 0);
    if constexpr(!STRIDED)
#pragma unroll
        for(int i = 1; i < STAGE_DEPTH - 1; ++i)
            fetch(row + i * static_cast<int64_t>(gridDim.x), i);
    statistics(row);
    int flip = 0;
    for(; row < P.M; row += gridDim.x)
    {
        if constexpr(!STRIDED)
        {
            fetch(row + (STAGE_DEPTH - 1) * static_cast<int64_t>(gridDim.x), slot == 0 ? STAGE_DEPTH - 1 : slot - 1);
            copy_async_wait<STAGE_DEPTH - 1>();
        }
        const uint64_t m2 = pack_f32x2(-mean, -mean), r2 = pack_f32x2(rstd, rstd);
        const float rs = rstd;
        uint64_t h[V][4], w[V][4];
        // xhat and w of vector v
        auto values = [&](int v, uint64_t (&hv)[4], uint64_t (&gy)[4], uint64_t (&wv)[4]) {
            if constexpr(!STRIDED)
            {
                ring.read(rx[v], slot, v);
                ring.read(ry[v], slot, V + v);
            }
            to_pairs(rx[v], hv);
            to_pairs(ry[v], gy);
#pragma unroll
            for(int i = 0; i < 4; ++i)
            {
                hv[i] = mul_f32x2(add_f32x2(hv[i], m2), r2);
                wv[i] = mul_f32x2(gy[i], g[v][i]);
            }
        };
        uint64_t s1v = 0, s2v = 0;
#pragma unroll
        for(int v = 0; v < V; ++v)
        {
            uint64_t gy[4];
            values(v, h[v], gy, w[v]);
            // (behind the row's end dy and gamma are zero, and so is all that xhat is multiplied with)
#pragma unroll
            for(int i = 0; i < 4; ++i)
            {
                dg[v][i] = fma_f32x2(gy[i], h[v][i], dg[v][i]);
                db[v][i] = add_f32x2(db[v][i], gy[i]);
                s1v      = add_f32x2(s1v, w[v][i]);
                s2v      = fma_f32x2(w[v][i], h[v][i], s2v);
            }
        }
        float s1 = sum_f32x2(s1v), s2 = sum_f32x2(s2v);
        const int64_t next = row + gridDim.x;
        if constexpr(STRIDED)
            fetch(next, 0);
        statistics(next);
        row_sum2<false>(s1, s2, buf + flip);
        flip ^= 64;
        if(P.dx)
        {
            const float c1 = s1 * inv_n, c2 = s2 * inv_n;
            const uint64_t c1v = pack_f32x2(-c1, -c1), c2v = pack_f32x2(-c2, -c2), rsv = pack_f32x2(rs, rs);
            T* out = static_cast<T*>(P.dx) + row * P.lddx;
#pragma unroll
            for(int v = 0; v < V; ++v)
            {
                if constexpr(!STRIDED)
                {
                    uint64_t gy[4];
                    values(v, h[v], gy, w[v]);
                }
                float o[8];
#pragma unroll
                for(int i = 0; i < 4; ++i)
                    unpack_f32x2(mul_f32x2(rsv, fma_f32x2(h[v][i], c2v, add_f32x2(w[v][i], c1v))), o[2 * i], o[2 * i + 1]);
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
        if(++slot == STAGE_DEPTH)
            slot = 0;
    }
    if constexpr(!STRIDED)
        copy_async_wait_all();
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
                float a[2], b[2];
                unpack_f32x2(dg[v][i / 2], a[0], a[1]);
                unpack_f32x2(db[v][i / 2], b[0], b[1]);
                if(c < P.N)
                {
                    pg[c] = a[i & 1];
                    pb[c] = b[i & 1];
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
