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

// Eight consecutive values as they lie in memory, in words.
template <typename T>
struct Vec8
{
    static constexpr int WORDS = 2 * sizeof(T);
    uint32_t w[WORDS];
};
__device__ __forceinline__ uint32_t bits_of(float v) { return __float_as_uint(v); }
__device__ __forceinline__ uint32_t bits_of(__half v) { return __half_as_ushort(v); }
__device__ __forceinline__ uint32_t bits_of(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }

// What a partial or unaligned vector needs is in functions of its own: inlined, the compiler turns it into predicated
// instructions that every vector issues (a quarter to a half of all instructions of these kernels).
// `n` = values that exist (<= 0: none, the vector is zero).
template <typename T>
__device__ __noinline__ Vec8<T> load8_slow(const T* p, int n)
{
    Vec8<T> r;
    uint32_t e[8];
#pragma unroll
    for(int i = 0; i < 8; ++i)
        e[i] = i < n ? bits_of(p[i]) : 0u;
#pragma unroll
    for(int i = 0; i < Vec8<T>::WORDS; ++i)
        r.w[i] = sizeof(T) == 4 ? e[i & 7] : e[(2 * i) & 7] | e[(2 * i + 1) & 7] << 16;
    return r;
}
template <typename T>
__device__ __forceinline__ void load8(Vec8<T>& r, const T* p, int n, bool vec)
{
    if(vec && n >= 8) // p is 16-byte aligned
    {
        const uint4* s = reinterpret_cast<const uint4*>(p);
#pragma unroll
        for(int i = 0; i < Vec8<T>::WORDS / 4; ++i)
        {
            const uint4 q = __ldg(s + i);
            r.w[4 * i] = q.x, r.w[4 * i + 1] = q.y, r.w[4 * i + 2] = q.z, r.w[4 * i + 3] = q.w;
        }
    }
    else
        r = load8_slow(p, n);
}

// Eight values that start anywhere, in two steps, so that a thread has the loads of several vectors in flight before it
// shifts the first one: the 16-byte pieces that hold them (VEC: p is 16-byte aligned, and they are the vector), then the
// values.  A piece may reach up to 15 bytes beyond the tensor, never beyond the 16-byte granule of its first or last
// value, so it stays inside the allocation.
template <typename T, bool VEC>
struct Raw8
{
    static constexpr int WORDS = Vec8<T>::WORDS + (VEC ? 0 : 4);
    uint32_t w[WORDS];
};
template <typename T, bool VEC>
__device__ __forceinline__ void fetch8(Raw8<T, VEC>& r, const T* p, int n)
{
    if constexpr(VEC)
    {
        Vec8<T> v;
        load8(v, p, n, true);
#pragma unroll
        for(int i = 0; i < Vec8<T>::WORDS; ++i)
            r.w[i] = v.w[i];
    }
    else
    {
        const uintptr_t at = reinterpret_cast<uintptr_t>(p);
        const int off      = static_cast<int>(at & 15);
        const uint4* s     = reinterpret_cast<const uint4*>(at - off);
        const int end      = n <= 0 ? 0 : off + (n < 8 ? n : 8) * static_cast<int>(sizeof(T));
#pragma unroll
        for(int i = 0; i < Raw8<T, VEC>::WORDS / 4; ++i)
        {
            uint4 q = make_uint4(0u, 0u, 0u, 0u);
            if(i * 16 < end)
                q = __ldg(s + i);
            r.w[4 * i] = q.x, r.w[4 * i + 1] = q.y, r.w[4 * i + 2] = q.z, r.w[4 * i + 3] = q.w;
        }
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void settle8(Vec8<T>& v, const Raw8<T, VEC>& r, const T* p, int n)
{
    constexpr int W = Vec8<T>::WORDS;
    if constexpr(VEC)
    {
#pragma unroll
        for(int i = 0; i < W; ++i)
            v.w[i] = r.w[i];
    }
    else
    {
        const int off = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15);
        uint32_t a[W + 2], b[W + 1];
#pragma unroll
        for(int i = 0; i < W + 2; ++i)
            a[i] = off & 8 ? r.w[i + 2] : r.w[i];
#pragma unroll
        for(int i = 0; i < W + 1; ++i)
            b[i] = off & 4 ? a[i + 1] : a[i];
#pragma unroll
        for(int i = 0; i < W; ++i)
            v.w[i] = sizeof(T) == 4 ? b[i] : __funnelshift_r(b[i], b[i + 1], (off & 3) * 8);
        if(n < 8) // values behind the row's end are zeros
        {
#pragma unroll
            for(int i = 0; i < W; ++i)
            {
                const int first = sizeof(T) == 4 ? i : 2 * i; // value in the low half of the word
                if(first >= n)
                    v.w[i] = 0u;
                else if(sizeof(T) == 2 && first + 1 >= n)
                    v.w[i] &= 0xffffu;
            }
        }
    }
}

// Two values, rounded, in one word (f32: as they are).
__device__ __forceinline__ uint32_t round_pair(const __half*, float lo, float hi)
{
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t round_pair(const __nv_bfloat16*, float lo, float hi)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __noinline__ void store8_slow(float4 lo, float4 hi, T* p, int n)
{
    const float f[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for(int i = 0; i < 8; ++i)
        if(i < n)
            p[i] = from_f32<T>(f[i]);
}
template <typename T>
__device__ __forceinline__ void store8(const float (&f)[8], T* p, int n, bool vec)
{
    if(vec && n >= 8)
    {
        if constexpr(sizeof(T) == 4)
        {
            reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
        }
        else
            *reinterpret_cast<uint4*>(p) = make_uint4(round_pair(p, f[0], f[1]), round_pair(p, f[2], f[3]), round_pair(p, f[4], f[5]),
                                                      round_pair(p, f[6], f[7]));
    }
    else if(n > 0)
        store8_slow(make_float4(f[0], f[1], f[2], f[3]), make_float4(f[4], f[5], f[6], f[7]), p, n);
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

__device__ __noinline__ float block_scale_slow(float amax, float qmax)
{
    const float s = __fdiv_rn(amax, qmax);
    return s < 1.17549435e-38f ? 1.17549435e-38f : s; // (a NaN stays)
}
// amax / qmax, correctly rounded (see below), at least the smallest normal number (its reciprocal still exists).
__device__ __forceinline__ float block_scale(float amax, float qmax, float qmax_recip, bool pow2)
{
    if(amax == 0.f)
        return 1.f;
    const float q0 = amax * qmax_recip;
    float s        = __fmaf_rn(__fmaf_rn(-q0, qmax, amax), qmax_recip, q0);
    if(!(amax >= 1e-28f && amax <= 3.402823466e+38f)) // tiny, infinite or NaN
        s = block_scale_slow(amax, qmax);
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
// The last step would add the remainder +0 of a zero to it, and -0 would come out as +0.  So the quotient by -scale is
// formed, whose last step adds (+0)(-r) = -0 and leaves a zero as it is; the sign bits are turned in the 8-bit values.
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
constexpr uint32_t F8_SIGNS = 0x80808080u;
// -(x / scale); minus_recip: -1 / scale
__device__ __forceinline__ uint64_t minus_quotient(uint64_t x, uint64_t scale, uint64_t minus_recip)
{
    const uint64_t q0 = mul_f32x2(x, minus_recip);
    return fma_f32x2(fma_f32x2(q0, scale, x), minus_recip, q0);
}

template <bool E5M2>
__device__ __forceinline__ uint32_t to_f8x2(float lo, float hi)
{
    return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, E5M2 ? __NV_E5M2 : __NV_E4M3);
}

// Eight values (four pairs) over one scale -> eight bytes.
template <bool E5M2>
__device__ __noinline__ uint2 quantize8_slow(ulonglong2 a, ulonglong2 b, float scale)
{
    const uint64_t f[4] = {a.x, a.y, b.x, b.y};
    uint32_t w[4];
#pragma unroll
    for(int i = 0; i < 4; ++i)
    {
        float lo, hi;
        unpack_f32x2(f[i], lo, hi);
        w[i] = to_f8x2<E5M2>(__fdiv_rn(lo, scale), __fdiv_rn(hi, scale));
    }
    return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
}
template <bool E5M2>
__device__ __forceinline__ uint2 quantize8(const uint64_t (&f)[4], const BlockDivisor& d)
{
    if(!d.fast)
        return quantize8_slow<E5M2>(make_ulonglong2(f[0], f[1]), make_ulonglong2(f[2], f[3]), d.scale);
    uint32_t w[4];
    const uint64_t s2 = pack_f32x2(d.scale, d.scale), mr = pack_f32x2(-d.recip, -d.recip);
#pragma unroll
    for(int i = 0; i < 4; ++i)
    {
        float lo, hi;
        unpack_f32x2(minus_quotient(f[i], s2, mr), lo, hi);
        w[i] = to_f8x2<E5M2>(lo, hi);
    }
    return make_uint2((w[0] | w[1] << 16) ^ F8_SIGNS, (w[2] | w[3] << 16) ^ F8_SIGNS);
}

// The eight values of a vector as pairs, and their largest magnitude.
__device__ __forceinline__ void to_pairs(const Vec8<float>& r, uint64_t (&f)[4])
{
#pragma unroll
    for(int i = 0; i < 4; ++i)
        f[i] = pack_f32x2(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
}
__device__ __forceinline__ void to_pairs(const Vec8<__half>& r, uint64_t (&f)[4])
{
#pragma unroll
    for(int i = 0; i < 4; ++i)
    {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
        f[i]           = pack_f32x2(v.x, v.y);
    }
}
__device__ __forceinline__ void to_pairs(const Vec8<__nv_bfloat16>& r, uint64_t (&f)[4])
{
#pragma unroll
    for(int i = 0; i < 4; ++i) // a bf16 is the upper half of the 32-bit number
        f[i] = pack_f32x2(__uint_as_float(r.w[i] << 16), __uint_as_float(r.w[i] & 0xffff0000u));
}
__device__ __forceinline__ float value_of(const Vec8<float>& r, int k) { return __uint_as_float(r.w[k]); }
__device__ __forceinline__ float value_of(const Vec8<__half>& r, int k)
{
    return __half2float(__ushort_as_half(static_cast<unsigned short>(r.w[k / 2] >> (16 * (k & 1)))));
}
__device__ __forceinline__ float value_of(const Vec8<__nv_bfloat16>& r, int k)
{
    return __uint_as_float(k & 1 ? r.w[k / 2] & 0xffff0000u : r.w[k / 2] << 16);
}
__device__ __forceinline__ float max_abs8(const Vec8<float>& r)
{
    float m = 0.f;
#pragma unroll
    for(int i = 0; i < 8; ++i)
        m = max_abs(m, __uint_as_float(r.w[i]));
    return m;
}
__device__ __forceinline__ float max_abs8(const Vec8<__half>& r)
{
    const __half2* h = reinterpret_cast<const __half2*>(r.w);
    const __half2 m  = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
    return max_abs(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float max_abs8(const Vec8<__nv_bfloat16>& r)
{
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(r.w);
    const __nv_bfloat162 m  = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
    return max_abs(__low2float(m), __high2float(m));
}

__device__ __noinline__ void store_q8_slow(uint2 w, uint8_t* p, int n)
{
#pragma unroll
    for(int i = 0; i < 8; ++i)
        if(i < n)
            p[i] = static_cast<uint8_t>((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
}
__device__ __forceinline__ void store_q8(uint2 w, uint8_t* p, int n, bool vec)
{
    if(vec && n >= 8)
        *reinterpret_cast<uint2*>(p) = w;
    else if(n > 0)
        store_q8_slow(w, p, n);
}

// 128 bytes of a block's row, eight from each of 16 lanes, to any address: each lane writes the aligned 8 bytes in which its
// own ones begin, with the end of its neighbour's; the pieces of less than 8 bytes at both ends are 4, 2 and 1 bytes.
__device__ __forceinline__ void store_q128(uint2 w, uint8_t* p, int sub)
{
    const uint32_t group = 0xffffu << (threadIdx.x & 16);
    const int off        = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 7);
    const uint2 before   = make_uint2(__shfl_up_sync(group, w.x, 1, 16), __shfl_up_sync(group, w.y, 1, 16));
    uint8_t* word        = p - off;
    const uint64_t own = static_cast<uint64_t>(w.y) << 32 | w.x, prev = static_cast<uint64_t>(before.y) << 32 | before.x;
    if(sub != 0 || off == 0) // bytes 8 - off .. 15 - off of (prev, own)
        *reinterpret_cast<uint64_t*>(word) = off == 0 ? own : own << (8 * off) | prev >> (64 - 8 * off);
    if(off != 0 && (sub == 0 || sub == 15))
    {
        // sub 0: bytes off .. 7 of its word; sub 15: bytes 0 .. off - 1 of the one behind its own
        const int count    = sub == 0 ? 8 - off : off;
        uint8_t* dst       = sub == 0 ? p : word + 8;
        const uint64_t src = sub == 0 ? own : own >> (64 - 8 * off);
        // pieces that end on a boundary come small ones first, pieces that start on one large ones first
        const int at4 = sub == 0 ? count & 3 : 0, at2 = sub == 0 ? count & 1 : count & 4, at1 = sub == 0 ? 0 : count & 6;
        if(count & 4)
            *reinterpret_cast<uint32_t*>(dst + at4) = static_cast<uint32_t>(src >> (8 * at4));
        if(count & 2)
            *reinterpret_cast<uint16_t*>(dst + at2) = static_cast<uint16_t>(src >> (8 * at2));
        if(count & 1)
            dst[at1] = static_cast<uint8_t>(src >> (8 * at1));
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
    float qmax, qmax_recip;
};
__device__ __forceinline__ int32_t block_row(const QuantizeParams& p, int32_t b)
{
    return p.div_mul == 0 ? b : static_cast<int32_t>(__umulhi(static_cast<uint32_t>(b), p.div_mul) >> p.div_shr);
}

// Block quantizer: one read of x, one write of q.  VEC: rows of x start on 16-byte and rows of q on 8-byte boundaries;
// other rows come in whole pieces (fetch8).
//
// Blocks of 1 x 128: 16 lanes per block, QB blocks per thread in flight.  8192 x 4096 bf16: 27.5 us (3.7 TB/s), bound by its
// instructions: 20 per value, 71 % of the issue slots at 45 % of the warps; f32 33.9 us (5.0 TB/s); 8192 x 4097 bf16: 42.5 us,
// 47.3 with a load per value, 54 with the bytes of q shifted between lanes (store_q128), which costs more here than stores byte
// by byte.
constexpr int QB = 4;
template <typename T, bool E5M2, bool VEC>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const __grid_constant__ QuantizeParams P)
{
    grid_dependency_wait();
    grid_launch_dependents();
    const T* x     = static_cast<const T*>(P.x);
    const int sub  = threadIdx.x & 15;
    const int unit = threadIdx.x >> 4; // 16 per CTA
    for(int64_t base = static_cast<int64_t>(blockIdx.x) * (16 * QB); base < P.total; base += static_cast<int64_t>(gridDim.x) * (16 * QB))
    {
        Raw8<T, VEC> fetched[QB];
        int row[QB], c0[QB], n[QB];
#pragma unroll
        for(int j = 0; j < QB; ++j)
        {
            const int64_t b = base + j * 16 + unit;
            const bool on   = b < P.total;
            row[j]          = on ? block_row(P, static_cast<int32_t>(b)) : 0;
            c0[j]           = on ? (static_cast<int32_t>(b) - row[j] * P.blocks_n) * 128 + sub * 8 : 0;
            n[j]            = on ? P.N - c0[j] : -1000;
            fetch8(fetched[j], x + row[j] * P.ldx + c0[j], n[j]);
        }
#pragma unroll
        for(int j = 0; j < QB; ++j)
        {
            Vec8<T> raw;
            settle8(raw, fetched[j], x + row[j] * P.ldx + c0[j], n[j]);
            const float s = block_scale(max16(max_abs8(raw)), P.qmax, P.qmax_recip, P.pow2 != 0);
            if(n[j] <= -1000)
                continue; // (all 16 lanes of the block)
            uint64_t f[4];
            to_pairs(raw, f);
            const uint2 w = quantize8<E5M2>(f, BlockDivisor(s));
            store_q8(w, P.q + row[j] * P.ldq + c0[j], n[j], VEC);
            if(sub == 0)
                P.scale[row[j] * P.ss_m + (c0[j] >> 7) * P.ss_n] = s;
        }
    }
}

// Blocks of 128 x 128 (SQUARE) or 128 x 1: a CTA holds 128 rows x 128 columns in registers, 8 rows x 8 columns a
// thread.  8192 x 4096 bf16: 22.0 us (128 x 128, 4.6 TB/s) and 33.0 (128 x 1: a scale per value to divide by, 117 registers
// and with them 16 warps per SM, 42 % of the issue slots), f32 32.5 and 36.9; 8192 x 4097 bf16: 52 and 59 us, 77 and 98 with a
// load per value and byte stores, 55 and 73 with byte stores alone.
// Row r of the tile belongs to threads 16 (r mod 16) .. + 15.
template <typename T, bool E5M2, bool SQUARE, bool VEC>
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
        Raw8<T, VEC> fetched[8];
        Vec8<T> raw[8];
#pragma unroll
        for(int i = 0; i < 8; ++i)
        {
            const int r = br * 128 + i * 16 + unit;
            fetch8(fetched[i], x + r * P.ldx + c0, r < P.M ? n : 0);
        }
#pragma unroll
        for(int i = 0; i < 8; ++i)
        {
            const int r = br * 128 + i * 16 + unit;
            settle8(raw[i], fetched[i], x + r * P.ldx + c0, r < P.M ? n : 0);
        }
        uint64_t scales[4], minus_recip[4]; // of this thread's columns (SQUARE: all the same)
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
                    m = max_abs(m, value_of(raw[i], k));
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
                scales[k]      = pack_f32x2(lo.scale, hi.scale);
                minus_recip[k] = pack_f32x2(-lo.recip, -hi.recip);
                fast           = fast && lo.fast && hi.fast;
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
                        unpack_f32x2(minus_quotient(f[k], scales[k], minus_recip[k]), lo, hi);
                    else
                    {
                        unpack_f32x2(f[k], lo, hi);
                        lo = __fdiv_rn(lo, scale[2 * k]);
                        hi = __fdiv_rn(hi, scale[2 * k + 1]);
                    }
                    h[k] = to_f8x2<E5M2>(lo, hi);
                }
                const uint32_t turn = fast ? F8_SIGNS : 0u;
                w = make_uint2((h[0] | h[1] << 16) ^ turn, (h[2] | h[3] << 16) ^ turn);
            }
            if(VEC || (c0 | 127) >= P.N)
                store_q8(w, P.q + r * P.ldq + c0, n, VEC);
            else
                store_q128(w, P.q + r * P.ldq + c0, sub);
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

// Threads that share a row: a warp, a whole CTA or (GROUPS) one of several equal parts of a CTA.
enum { ROW_WARP, ROW_CTA, ROW_GROUP };
template <int KIND>
__device__ __forceinline__ void row_barrier(int group, int threads)
{
    if constexpr(KIND == ROW_CTA)
        __syncthreads();
    else if constexpr(KIND == ROW_GROUP)
        asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(threads) : "memory");
}

// Sum of one value over the threads of a row (up to 16 warps; LONG: up to 32); `buf` holds 32 words per use, a barrier
// lies between two uses of the same words.
template <int KIND, bool LONG = false>
__device__ __forceinline__ float row_sum(float a, float* buf, int group, int threads)
{
    a = warp_sum(a);
    if constexpr(KIND != ROW_WARP)
    {
        const int warp = (threadIdx.x - group * threads) >> 5, lane = threadIdx.x & 31, warps = threads >> 5;
        if(lane == 0)
            buf[warp] = a;
        row_barrier<KIND>(group, threads);
        constexpr int W = LONG ? 32 : 16;
        const int i     = lane & (W - 1);
        a               = i < warps ? buf[i] : 0.f;
#pragma unroll
        for(int d = W / 2; d >= 1; d >>= 1)
            a += __shfl_xor_sync(0xffffffffu, a, d);
    }
    return a;
}
// Of two values at once (64 words): the lower half of a warp sums the first, the upper half the second.
template <int KIND, bool LONG = false>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* buf, int group, int threads)
{
    const int lane  = threadIdx.x & 31;
    const bool high = lane >= 16;
    float v         = (high ? b : a) + __shfl_xor_sync(0xffffffffu, high ? a : b, 16);
#pragma unroll
    for(int d = 8; d >= 1; d >>= 1)
        v += __shfl_xor_sync(0xffffffffu, v, d);
    if constexpr(KIND != ROW_WARP)
    {
        const int warp = (threadIdx.x - group * threads) >> 5, warps = threads >> 5, i = lane & 15;
        if(i == 0)
            buf[(high ? 32 : 0) + warp] = v;
        row_barrier<KIND>(group, threads);
        const float* mine = buf + (high ? 32 : 0);
        v                 = i < warps ? mine[i] : 0.f;
        if constexpr(LONG)
            v += i + 16 < warps ? mine[i + 16] : 0.f;
#pragma unroll
        for(int d = 8; d >= 1; d >>= 1)
            v += __shfl_xor_sync(0xffffffffu, v, d);
    }
    const float other = __shfl_xor_sync(0xffffffffu, v, 16);
    a                 = high ? other : v;
    b                 = high ? v : other;
}

// From the mean square and the mean of the distances to the first mean.
__device__ __forceinline__ float rstd_of(float square, float shift, float eps)
{
    const float var = __fmaf_rn(-shift, shift, square);
    return __frsqrt_rn((var < 0.f ? 0.f : var) + eps); // (a NaN stays one)
}

// Words of shared memory from byte `off` (0 .. 15) behind a 16-byte boundary on.
template <int NW>
__device__ __forceinline__ void lds_words(uint32_t (&out)[NW], uint32_t addr, int off)
{
    uint32_t w[NW + 4];
    auto load = [&](int i) {
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[4 * i]), "=r"(w[4 * i + 1]), "=r"(w[4 * i + 2]), "=r"(w[4 * i + 3])
                     : "r"(addr + i * 16)
                     : "memory");
    };
#pragma unroll
    for(int i = 0; i < NW / 4; ++i)
        load(i);
    if(off == 0)
    {
#pragma unroll
        for(int i = 0; i < NW; ++i)
            out[i] = w[i];
        return;
    }
    load(NW / 4);
    if(off & 8)
    {
#pragma unroll
        for(int i = 0; i < NW + 2; ++i)
            w[i] = w[i + 2];
    }
    if(off & 4)
    {
#pragma unroll
        for(int i = 0; i < NW + 1; ++i)
            w[i] = w[i + 1];
    }
#pragma unroll
    for(int i = 0; i < NW; ++i)
        out[i] = __funnelshift_r(w[i], w[i + 1], (off & 3) * 8);
}
__device__ __forceinline__ void sts_words(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Rows on their way: asynchronous copies into shared memory, STAGE_DEPTH - 1 rows ahead.  A warp has ELEMS neighbouring
// values of the row and a ring of its own; only its lanes have to meet.  Rows may start anywhere: the 16-byte pieces that
// hold them are copied whole and in order (a sector is fetched once, whatever vectors the lanes work on), and a lane
// shifts its vectors out of them.  (The piece that holds a tensor's first values may begin up to 15 bytes before the
// tensor, inside the same allocation: those start on 256-byte boundaries.)
constexpr int STAGE_DEPTH = 3;
template <typename T, int ELEMS>
struct WarpRing
{
    static constexpr int BYTES = ELEMS * sizeof(T);
    static constexpr int SLOT  = BYTES + 16;
    uint32_t base; // of the warp
    static __host__ __device__ int bytes(int threads) { return STAGE_DEPTH * SLOT * (threads / 32); }
    __device__ __forceinline__ WarpRing(const void* smem, int which = 0, int of = 1)
        : base(smem_u32(smem) + ((threadIdx.x >> 5) * of + which) * (STAGE_DEPTH * SLOT))
    {
    }
    // `n` = values of the row from p, the warp's first one, on
    __device__ __forceinline__ void copy(int slot, const T* p, int n) const
    {
        const uintptr_t at = reinterpret_cast<uintptr_t>(p);
        const int off      = static_cast<int>(at & 15);
        const char* src    = reinterpret_cast<const char*>(at - off) + (threadIdx.x & 31) * 16;
        const uint32_t dst = base + slot * SLOT + (threadIdx.x & 31) * 16;
        const int all      = n < ELEMS ? n : ELEMS;                                                              // values
        const int left     = off + all * static_cast<int>(sizeof(T)) - (static_cast<int>(threadIdx.x) & 31) * 16; // bytes from this lane's piece on
        if(off == 0 && all == ELEMS)
        {
#pragma unroll
            for(int i = 0; i < BYTES / 512; ++i)
                copy_async_16(dst + i * 512, src + i * 512, 16);
        }
        else if(all > 0)
        {
#pragma unroll
            for(int i = 0; i <= BYTES / 512; ++i)
            {
                const int have = left - i * 512;
                if(i < BYTES / 512 || (threadIdx.x & 31) == 0) // (one piece more than the values fill)
                    copy_async_16(dst + i * 512, have > 0 ? src + i * 512 : src, have < 0 ? 0 : have > 16 ? 16 : have);
            }
        }
    }
    // words of the `count` values from value `first` of the span on (first * sizeof(T) a multiple of 16)
    template <int NW>
    __device__ __forceinline__ void read(uint32_t (&w)[NW], int slot, int first, int off) const
    {
        lds_words(w, base + slot * SLOT + first * static_cast<int>(sizeof(T)), off);
    }
};

// A warp's values leave through a piece of its shared memory, 16 bytes per lane and instruction, in order.  `stage` holds
// BYTES of output from its start on; dst: where its first byte goes (any alignment); n: how many bytes exist.
template <int BYTES, int ELEM>
__device__ __forceinline__ void store_span(uint32_t stage, uint8_t* dst, int n)
{
    const int lane = threadIdx.x & 31;
    const int off  = static_cast<int>(reinterpret_cast<uintptr_t>(dst) & 15);
    __syncwarp();
    if(off == 0 && n >= BYTES)
    {
#pragma unroll
        for(int i = 0; i < (BYTES + 511) / 512; ++i)
        {
            if(BYTES % 512 != 0 && i * 512 + lane * 16 >= BYTES)
                break;
            uint32_t w[4];
            lds_words(w, stage + i * 512 + lane * 16, 0);
            *reinterpret_cast<uint4*>(dst + i * 512 + lane * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    else
    {
        n              = n > BYTES ? BYTES : n < 0 ? 0 : n;
        const int head = off == 0 ? 0 : n < 16 - off ? n : 16 - off; // bytes before dst's first boundary
        const int tail = head + ((n - head) & ~15);                  // where the last whole piece ends
        for(int from = head + lane * 16; from < tail; from += 512)
        {
            uint32_t w[4];
            lds_words(w, stage + (from & ~15), from & 15);
            *reinterpret_cast<uint4*>(dst + from) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        // both ends at once, an element per lane (one lane after the other they took longer than the rest)
        const int b = (lane & 15) * ELEM + (lane & 16 ? tail : 0);
        if(b < (lane & 16 ? n : head))
        {
            uint32_t v;
            if constexpr(ELEM == 4)
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(stage + b) : "memory");
            else if constexpr(ELEM == 2)
                asm volatile("{.reg .b16 t; ld.shared.b16 t, [%1]; cvt.u32.u16 %0, t;}" : "=r"(v) : "r"(stage + b) : "memory");
            else
                asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(stage + b) : "memory");
            if constexpr(ELEM == 4)
                *reinterpret_cast<uint32_t*>(dst + b) = v;
            else if constexpr(ELEM == 2)
                *reinterpret_cast<uint16_t*>(dst + b) = static_cast<uint16_t>(v);
            else
                dst[b] = static_cast<uint8_t>(v);
        }
    }
    __syncwarp();
}
// Eight values, rounded to T, into the stage.
template <typename T>
__device__ __forceinline__ void stage8(uint32_t addr, const float (&f)[8])
{
    const T* t = nullptr;
    if constexpr(sizeof(T) == 4)
    {
        sts_words(addr, __float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
        sts_words(addr + 16, __float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7]));
    }
    else
        sts_words(addr, round_pair(t, f[0], f[1]), round_pair(t, f[2], f[3]), round_pair(t, f[4], f[5]), round_pair(t, f[6], f[7]));
}

// The same for rows that start on 16-byte boundaries and vectors that lie in order: every thread copies the vectors it
// works on itself and reads nobody else's, so only its own copies have to be waited for.  A warp's part of the ring is
// [row][vector][16-byte piece][lane]: with that, and with a warp's columns side by side in the matrix, all addresses of a
// row are one register plus constants (laid out over the whole CTA the address arithmetic was 200 of 640 instructions per
// row and thread).
template <typename T, int V>
struct RowRing
{
    static constexpr int PIECES = sizeof(T) / 2; // 16-byte pieces of a vector
    static constexpr int PER    = 16 / sizeof(T);
    static constexpr int SLOT   = V * PIECES * 512; // bytes of a row and warp
    uint32_t base;                                  // this lane's first piece
    static __host__ __device__ int bytes(int threads) { return STAGE_DEPTH * V * PIECES * threads * 16; }
    __device__ __forceinline__ RowRing(const void* smem)
        : base(smem_u32(smem) + (threadIdx.x >> 5) * (STAGE_DEPTH * SLOT) + (threadIdx.x & 31) * 16)
    {
    }
    // `n` = values of the row from the vector's first one on (<= 0: none, p is not read)
    __device__ __forceinline__ void copy(int slot, int v, const T* p, int n) const
    {
        const uint32_t dst = base + slot * SLOT + v * (PIECES * 512);
        if(n >= 8)
        {
#pragma unroll
            for(int i = 0; i < PIECES; ++i)
                copy_async_16(dst + i * 512, p + i * PER, 16);
        }
        else
            copy_slow(dst, p, n);
    }
    static __device__ __noinline__ void copy_slow(uint32_t dst, const T* p, int n)
    {
#pragma unroll
        for(int i = 0; i < PIECES; ++i)
        {
            const int have = (n - i * PER) * static_cast<int>(sizeof(T)); // bytes
            copy_async_16(dst + i * 512, have > 0 ? p + i * PER : p, have < 0 ? 0 : have > 16 ? 16 : have);
        }
    }
    __device__ __forceinline__ void read(Vec8<T>& r, int slot, int v) const
    {
        const uint32_t src = base + slot * SLOT + v * (PIECES * 512);
#pragma unroll
        for(int i = 0; i < PIECES; ++i)
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(r.w[4 * i]), "=r"(r.w[4 * i + 1]), "=r"(r.w[4 * i + 2]), "=r"(r.w[4 * i + 3])
                         : "r"(src + i * 512)
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
    int32_t tpr;      // threads of a row (ROW_GROUP, ROW_CTA)
    int32_t w_offset; // ROW_GROUP: where gamma and beta lie in shared memory
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
struct Pairs4
{
    uint64_t p[4];
};
// The first n values of eight, zero for the others.
__device__ __noinline__ Pairs4 first_of(Pairs4 d, int n)
{
#pragma unroll
    for(int i = 0; i < 4; ++i)
    {
        float lo, hi;
        unpack_f32x2(d.p[i], lo, hi);
        d.p[i] = pack_f32x2(2 * i < n ? lo : 0.f, 2 * i + 1 < n ? hi : 0.f);
    }
    return d;
}
__device__ __forceinline__ void keep_first(uint64_t (&d)[4], int n)
{
    const Pairs4 r = first_of(Pairs4{{d[0], d[1], d[2], d[3]}}, n);
#pragma unroll
    for(int i = 0; i < 4; ++i)
        d[i] = r.p[i];
}
// Subtracts `mean` from the eight values, zero where there is no value (n of them exist).
__device__ __forceinline__ void distances(uint64_t (&d)[4], float mean, int n)
{
    const uint64_t m2 = pack_f32x2(-mean, -mean);
#pragma unroll
    for(int i = 0; i < 4; ++i)
        d[i] = add_f32x2(d[i], m2);
    if(n < 8)
        keep_first(d, n);
}

// y of 16 columns, `have` of which (at most) exist: y = (d - shift) * rstd * gamma + beta, d = distances to the first mean
// (zero where there is no value).  weights(h, g, b): gamma and beta of columns 8 h .. + 7.
template <typename Weights>
__device__ __forceinline__ void layernorm_y16(uint64_t (&d)[2][4], int have, float shift, float rstd, Weights weights)
{
    const uint64_t r2 = pack_f32x2(rstd, rstd), s2 = pack_f32x2(-shift, -shift);
#pragma unroll
    for(int h = 0; h < 2; ++h)
    {
        uint64_t g[4], b[4];
        weights(h, g, b);
#pragma unroll
        for(int i = 0; i < 4; ++i)
            d[h][i] = fma_f32x2(mul_f32x2(add_f32x2(d[h][i], s2), r2), g[i], b[i]);
        if(have - h * 8 < 8)
            keep_first(d[h], have - h * 8); // (what does not exist must not count in a block's largest value)
    }
}
// Eight neighbouring lanes hold a block of 128 columns: its scale, and this lane's sixteen values over it.
template <bool E5M2>
__device__ __forceinline__ float layernorm_q16(const uint64_t (&d)[2][4], float qmax, float qmax_recip, uint4& q)
{
    float m = 0.f;
#pragma unroll
    for(int h = 0; h < 2; ++h)
#pragma unroll
        for(int i = 0; i < 4; ++i)
        {
            float lo, hi;
            unpack_f32x2(d[h][i], lo, hi);
            m = max_abs(max_abs(m, lo), hi);
        }
#pragma unroll
    for(int k = 4; k >= 1; k >>= 1)
        m = max_abs(m, __shfl_xor_sync(0xffffffffu, m, k));
    const float s = block_scale(m, qmax, qmax_recip, false);
    const BlockDivisor div(s);
    const uint2 w0 = quantize8<E5M2>(d[0], div), w1 = quantize8<E5M2>(d[1], div);
    q = make_uint4(w0.x, w0.y, w1.x, w1.y);
    return s;
}

// U units of 16 values a thread: unit u of a lane of the row's warp w holds columns 512 (w U + u) + 16 lane .. + 15, so a
// scale block belongs to eight lanes.
//   ROW_WARP   a row per warp, eight rows a CTA
//   ROW_GROUP  one CTA per SM works on as many rows side by side as fit; gamma and beta wait in shared memory in 32 bits
//              (read for every row from L2 they were 2.6 times the bytes of the rows, and their latency most of the time)
//   ROW_CTA    longer rows, or a row per CTA: the weights from L2
// Rows come and go through shared memory in 16-byte pieces, in order (WarpRing, store_span).
// 8192 x 4096 bf16: 43 us (3.1 TB/s), x 4097 61; f32 83 us (3.2 TB/s), x 4097 130; 8192 x 5120 bf16 to 8 bits: 53 us.  Neither
// DRAM (21 to 31 %) nor the issue slots (25 to 60 %) are full: norm and quantizer take 26 instructions per value, 30 us at full
// issue.  Each part of a CTA takes its row through one chain - two sums with a barrier each, the weights, the way out through
// shared memory - and 12 to 24 warps are all that overlap.
// Mean and variance in two passes over the registers; the second pass also sums the distances themselves, which takes
// the rounding of the first mean out of both.
template <typename T, bool E5M2, int U, int KIND>
__global__ void __launch_bounds__(KIND == ROW_WARP ? 256 : KIND == ROW_GROUP ? 768 : 512, KIND == ROW_WARP ? 2 : 1)
    layernorm_fwd_kernel(const __grid_constant__ LayernormFwdParams P)
{
    grid_dependency_wait();
    grid_launch_dependents();
    extern __shared__ __align__(16) uint8_t ring_smem[];
    __shared__ float sums[KIND == ROW_WARP ? 1 : KIND == ROW_GROUP ? 8 * 192 : 192];
    const int tpr       = KIND == ROW_WARP ? 32 : P.tpr;
    const int groups    = KIND == ROW_WARP ? 8 : static_cast<int>(blockDim.x) / tpr;
    const int group     = static_cast<int>(threadIdx.x) / tpr;
    const int t         = static_cast<int>(threadIdx.x) - group * tpr;
    const int lane      = t & 31;
    const int64_t step  = static_cast<int64_t>(gridDim.x) * groups;
    int64_t row         = static_cast<int64_t>(blockIdx.x) * groups + group;
    const T* x          = static_cast<const T*>(P.x);
    const float inv_n   = 1.f / static_cast<float>(P.N);
    float* buf          = sums + (KIND == ROW_GROUP ? group * 192 : 0); // two rows in turn, 96 words each
    using Ring          = WarpRing<T, U * 512>;
    const Ring ring(ring_smem);
    const int warp_col  = (t >> 5) * (U * 512);           // the warp's first column
    const int warp_have = P.N - warp_col;                 // values of the row from there on
    const int have      = warp_have - lane * 16;          // and from this lane's first one on
    const T* ahead      = x + row * P.ldx + (warp_have > 0 ? warp_col : 0); // of the row that is fetched next
    const T* now        = ahead;
    const int64_t row_step = step * P.ldx;
    int64_t ahead_row      = row;
    auto fetch = [&](int slot) {
        if(ahead_row < P.M)
            ring.copy(slot, ahead, warp_have);
        copy_async_commit();
        ahead += row_step;
        ahead_row += step;
    };
    int slot = 0;
#pragma unroll
    for(int i = 0; i < STAGE_DEPTH - 1; ++i)
        fetch(i);
    // ROW_GROUP: [warp of the row][gamma, beta][unit][half][four values][lane]
    constexpr int W_WARP = 2 * U * 2 * 2 * 32; // 16-byte pieces of a warp
    float4* w_smem       = reinterpret_cast<float4*>(ring_smem + (KIND == ROW_GROUP ? P.w_offset : 0));
    if constexpr(KIND == ROW_GROUP)
    {
        for(int i = threadIdx.x; i < 2 * U * 2 * tpr; i += blockDim.x)
        {
            const int ln = i & 31, vec = (i >> 5) % (2 * U * 2), w = (i >> 5) / (2 * U * 2);
            const int which = vec / (U * 2), uh = vec % (U * 2);
            const int c     = w * (U * 512) + (uh >> 1) * 512 + ln * 16 + (uh & 1) * 8;
            uint64_t f[4];
            load_weights8<T>(f, which ? P.beta : P.gamma, P.w_f32 != 0, c < P.N ? c : 0, c < P.N ? P.N : 0, P.w_vec != 0, which ? 0.f : 1.f);
#pragma unroll
            for(int k = 0; k < 2; ++k)
            {
                float4 v;
                unpack_f32x2(f[2 * k], v.x, v.y);
                unpack_f32x2(f[2 * k + 1], v.z, v.w);
                w_smem[w * W_WARP + (vec * 2 + k) * 32 + ln] = v;
            }
        }
        __syncthreads();
    }
    const float4* w_mine = w_smem + (t >> 5) * W_WARP + lane;
    T* y_row             = static_cast<T*>(P.y) + (P.y ? row * P.ldy + warp_col : 0);
    uint8_t* q_row       = P.q + (P.q ? row * P.ldq + warp_col : 0);
    float* s_row         = P.q_scale + (P.q ? row * P.ss_m + ((warp_col + lane * 16) >> 7) * P.ss_n : 0);
    int flip             = 0;
    for(; row < P.M; row += step)
    {
        __syncwarp(); // the slot that is filled now was the last row's way out
        fetch(slot == 0 ? STAGE_DEPTH - 1 : slot - 1);
        copy_async_wait<STAGE_DEPTH - 1>();
        __syncwarp();
        const int off = static_cast<int>(reinterpret_cast<uintptr_t>(now) & 15);
        uint64_t d[U][2][4];
        uint64_t sv = 0;
#pragma unroll
        for(int u = 0; u < U; ++u)
        {
            uint32_t w[4 * sizeof(T)];
            ring.read(w, slot, u * 512 + lane * 16, off);
#pragma unroll
            for(int h = 0; h < 2; ++h)
            {
                Vec8<T> r;
#pragma unroll
                for(int i = 0; i < Vec8<T>::WORDS; ++i)
                    r.w[i] = w[h * Vec8<T>::WORDS + i];
                to_pairs(r, d[u][h]);
                if(have - u * 512 - h * 8 < 8)
                    keep_first(d[u][h], have - u * 512 - h * 8); // (what lies behind the row's end was never copied)
                sv = add_f32x2(sv, add_f32x2(add_f32x2(d[u][h][0], d[u][h][1]), add_f32x2(d[u][h][2], d[u][h][3])));
            }
        }
        float mean   = row_sum<KIND>(sum_f32x2(sv), buf + flip, group, tpr) * inv_n;
        uint64_t s1v = 0, s2v = 0;
#pragma unroll
        for(int u = 0; u < U; ++u)
#pragma unroll
            for(int h = 0; h < 2; ++h)
            {
                distances(d[u][h], mean, have - u * 512 - h * 8);
#pragma unroll
                for(int i = 0; i < 4; ++i)
                {
                    s1v = add_f32x2(s1v, d[u][h][i]);
                    s2v = fma_f32x2(d[u][h][i], d[u][h][i], s2v);
                }
            }
        float s1 = sum_f32x2(s1v), s2 = sum_f32x2(s2v);
        row_sum2<KIND>(s1, s2, buf + 32 + flip, group, tpr);
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
        if(warp_have > 0)
        {
            const uint32_t stage = ring.base + slot * Ring::SLOT; // (the row is in registers)
#pragma unroll
            for(int u = 0; u < U; ++u)
            {
                layernorm_y16(d[u], have - u * 512, shift, rstd, [&](int h, uint64_t (&g)[4], uint64_t (&b)[4]) {
                    if constexpr(KIND == ROW_GROUP)
                    {
#pragma unroll
                        for(int k = 0; k < 2; ++k)
                        {
                            const ulonglong2 gv = *reinterpret_cast<const ulonglong2*>(w_mine + ((u * 2 + h) * 2 + k) * 32);
                            const ulonglong2 bv = *reinterpret_cast<const ulonglong2*>(w_mine + ((U * 2 + u * 2 + h) * 2 + k) * 32);
                            g[2 * k] = gv.x, g[2 * k + 1] = gv.y, b[2 * k] = bv.x, b[2 * k + 1] = bv.y;
                        }
                    }
                    else
                    {
                        const int c = warp_col + u * 512 + lane * 16 + h * 8;
                        load_weights8<T>(g, P.gamma, P.w_f32 != 0, c, P.N, P.w_vec != 0, 1.f);
                        load_weights8<T>(b, P.beta, P.w_f32 != 0, c, P.N, P.w_vec != 0, 0.f);
                    }
                });
            }
            __syncwarp(); // every lane has read its part of the row
            if(P.y)
            {
#pragma unroll
                for(int u = 0; u < U; ++u)
#pragma unroll
                    for(int h = 0; h < 2; ++h)
                    {
                        float y[8];
#pragma unroll
                        for(int i = 0; i < 4; ++i)
                            unpack_f32x2(d[u][h][i], y[2 * i], y[2 * i + 1]);
                        stage8<T>(stage + (u * 512 + lane * 16 + h * 8) * static_cast<int>(sizeof(T)), y);
                    }
                store_span<Ring::BYTES, sizeof(T)>(stage, reinterpret_cast<uint8_t*>(y_row), warp_have < U * 512 ? warp_have * static_cast<int>(sizeof(T)) : Ring::BYTES);
            }
            if(P.q)
            {
#pragma unroll
                for(int u = 0; u < U; ++u)
                {
                    uint4 q;
                    const float s = layernorm_q16<E5M2>(d[u], P.qmax, P.qmax_recip, q);
                    if((lane & 7) == 0 && have - u * 512 > 0)
                        s_row[u * 4 * P.ss_n] = s;
                    if(P.q_vec && have - u * 512 >= 16) // (16 bytes a lane, in order already)
                        *reinterpret_cast<uint4*>(q_row + u * 512 + lane * 16) = q;
                    else if(!P.q_vec)
                        sts_words(stage + u * 512 + lane * 16, q.x, q.y, q.z, q.w);
                    else if(have - u * 512 > 0)
                    {
                        store_q8(make_uint2(q.x, q.y), q_row + u * 512 + lane * 16, have - u * 512, false);
                        store_q8(make_uint2(q.z, q.w), q_row + u * 512 + lane * 16 + 8, have - u * 512 - 8, false);
                    }
                }
                if(!P.q_vec)
                    store_span<U * 512, 1>(stage, q_row, warp_have < U * 512 ? warp_have : U * 512);
            }
        }
        now += row_step;
        y_row += step * P.ldy;
        q_row += step * P.ldq;
        s_row += step * P.ss_m;
        if(++slot == STAGE_DEPTH)
            slot = 0;
        flip ^= 96;
    }
    copy_async_wait_all();
}

// Rows that do not fit the registers of a CTA: the row is read three times (the second and third time from L2).
// 1024 x 32768 bf16: 82 us.  Rows off 16-byte boundaries are loaded and stored value by value: x 32767 280 us.
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
        float sum = 0.f;
        Vec8<T> r;
        uint64_t d[2][4];
        for(int64_t c = t * 8; c < P.N; c += 8192)
        {
            load8(r, x + row * P.ldx + c, static_cast<int>(P.N - c), P.x_vec != 0);
            to_pairs(r, d[0]);
            sum += sum_f32x2(add_f32x2(add_f32x2(d[0][0], d[0][1]), add_f32x2(d[0][2], d[0][3])));
        }
        const float mean = row_sum<ROW_CTA, true>(sum, buf, 0, 1024) / n;
        float s1 = 0.f, s2 = 0.f;
        for(int64_t c = t * 8; c < P.N; c += 8192)
        {
            load8(r, x + row * P.ldx + c, static_cast<int>(P.N - c), P.x_vec != 0);
            to_pairs(r, d[0]);
            distances(d[0], mean, static_cast<int>(P.N - c));
            uint64_t p1 = 0, p2 = 0;
#pragma unroll
            for(int i = 0; i < 4; ++i)
            {
                p1 = add_f32x2(p1, d[0][i]);
                p2 = fma_f32x2(d[0][i], d[0][i], p2);
            }
            s1 += sum_f32x2(p1);
            s2 += sum_f32x2(p2);
        }
        row_sum2<ROW_CTA, true>(s1, s2, buf + 64, 0, 1024);
        const float shift = s1 / n;
        const float rstd  = rstd_of(s2 / n, shift, P.eps);
        if(t == 0)
        {
            if(P.mean)
                P.mean[row] = mean + shift;
            if(P.rstd)
                P.rstd[row] = rstd;
        }
        for(int64_t c0 = 0; c0 < P.N; c0 += 16384)
        {
            const int64_t c = c0 + t * 16;
            if(__all_sync(0xffffffffu, c >= P.N))
                continue;
            // (a lane behind the row's end takes part in the shuffles with zeros)
            const int cc = c < P.N ? static_cast<int>(c) : P.N;
#pragma unroll
            for(int h = 0; h < 2; ++h)
            {
                const int m = P.N - cc - h * 8;
                load8(r, x + row * P.ldx + (m > 0 ? cc + h * 8 : 0), m, P.x_vec != 0);
                to_pairs(r, d[h]);
                distances(d[h], mean, m);
            }
            layernorm_y16(d, P.N - cc, shift, rstd, [&](int h, uint64_t (&g)[4], uint64_t (&b)[4]) {
                load_weights8<T>(g, P.gamma, P.w_f32 != 0, cc + h * 8, P.N, P.w_vec != 0, 1.f);
                load_weights8<T>(b, P.beta, P.w_f32 != 0, cc + h * 8, P.N, P.w_vec != 0, 0.f);
            });
            if(P.y)
#pragma unroll
                for(int h = 0; h < 2; ++h)
                {
                    float y[8];
#pragma unroll
                    for(int i = 0; i < 4; ++i)
                        unpack_f32x2(d[h][i], y[2 * i], y[2 * i + 1]);
                    store8(y, static_cast<T*>(P.y) + row * P.ldy + cc + h * 8, P.N - cc - h * 8, P.y_vec != 0);
                }
            if(P.q)
            {
                uint4 q;
                const float s = layernorm_q16<E5M2>(d, P.qmax, P.qmax_recip, q);
                if((t & 7) == 0 && cc < P.N)
                    P.q_scale[row * P.ss_m + (cc >> 7) * P.ss_n] = s;
                store_q8(make_uint2(q.x, q.y), P.q + row * P.ldq + cc, P.N - cc, P.q_vec != 0);
                store_q8(make_uint2(q.z, q.w), P.q + row * P.ldq + cc + 8, P.N - cc - 8, P.q_vec != 0);
            }
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
    int64_t lddy, ldx, lddx;
    int64_t M;
    int32_t N, parts;
    int32_t w_f32, w_vec;
    int32_t vec; // rows of dy, x and dx start on 16-byte boundaries
};

// Where element i of vector v of a thread lies.  STRIDED: neighbouring lanes hold neighbouring columns, for rows that
// do not start on 16-byte boundaries.
template <int V, bool STRIDED>
__device__ __forceinline__ int column_of(int v, int i, int t, int tpr)
{
    return STRIDED ? (v * 8 + i) * tpr + t : ((t >> 5) * V + v) * 256 + (t & 31) * 8 + i;
}
// Columns behind the row's end hold zero, or (REPEAT) its first value.
template <bool REPEAT, typename T>
__device__ __forceinline__ void load_columns(Vec8<T>& r, const T* row, int v, int t, int tpr, int N, bool on)
{
    uint32_t e[8];
#pragma unroll
    for(int i = 0; i < 8; ++i)
    {
        const int c = column_of<1, true>(v, i, t, tpr);
        e[i]        = on && (REPEAT || c < N) ? bits_of(row[c < N ? c : 0]) : 0u;
    }
#pragma unroll
    for(int i = 0; i < Vec8<T>::WORDS; ++i)
        r.w[i] = sizeof(T) == 4 ? e[i & 7] : e[(2 * i) & 7] | e[(2 * i + 1) & 7] << 16;
}

// Behind the row's end dy and gamma are zero, and so is w.  What xhat is there counts nothing as long as it is a number, and
// -mean * rstd, the xhat of a zero, is none in a row of values next to 1e36 and little else.  So x is one of the row's own
// values there, or xhat is cut off.
//
// dx and the partial sums of dgamma and dbeta in one pass.  A CTA walks rows blockIdx.x, + gridDim.x, ...; a thread keeps
// the same V x 8 columns throughout, so the column sums stay in its registers until the CTA writes them once.  Rows that
// start on 16-byte boundaries come through shared memory (RowRing), STRIDED ones one ahead in registers.
// bf16: 8192 x 4096 50 us (4.0 TB/s, 61 % of a copy's rate), x 5120 67 us; f32, STRIDED: 8192 x 4096 97 us (4.2 TB/s),
// 65536 x 511 107 us.  Few warps, each with a row's chain of loads, sums, a barrier and stores: latency, not bytes.
// TAIL (see above): STRIDED, the threads have more columns than the row, x repeats its first value behind its end (8192 x 4097
// f32 107 us, 103 without); else, the row ends inside a vector, whose xhat is cut off (in every kernel 2 to 7 % of the time).
// Without TAIL a thread's vector lies in the row, or is copied from its start.
template <typename T, int V, bool STRIDED, bool TAIL>
__global__ void __launch_bounds__(V == 1 ? 768 : 512, 1) layernorm_bwd_kernel(const __grid_constant__ LayernormBwdParams P)
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
            const int c = column_of<V, STRIDED>(v, i, t, tpr);
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
    const RowRing<T, 2 * V> ring(ring_smem); // vectors of x, then of dy
    float mean = 0.f, rstd = 0.f;
    const int col0 = STRIDED ? 0 : column_of<V, false>(0, 0, t, tpr);
    const int have = P.N - col0; // values of the row from this thread's first column on
    const T* x_ahead  = x + blockIdx.x * P.ldx; // of the row that is fetched next
    const T* dy_ahead = dy + blockIdx.x * P.lddy + (have > 0 ? col0 : 0);
    const int64_t x_step = gridDim.x * P.ldx, dy_step = gridDim.x * P.lddy;
    int64_t ahead_row = blockIdx.x;
    auto fetch = [&](int slot) {
        const bool on = ahead_row < P.M;
#pragma unroll
        for(int v = 0; v < V; ++v)
        {
            if constexpr(STRIDED)
            {
                load_columns<TAIL>(rx[v], x_ahead, v, t, tpr, P.N, on);
                load_columns<false>(ry[v], dy_ahead, v, t, tpr, P.N, on);
            }
            else if(on)
            {
                if constexpr(TAIL)
                    ring.copy(slot, v, x_ahead + (have > 0 ? col0 : 0) + v * 256, have - v * 256);
                else
                    ring.copy(slot, v, x_ahead + (have > v * 256 ? col0 + v * 256 : 0), 8);
                ring.copy(slot, V + v, dy_ahead + v * 256, have - v * 256);
            }
        }
        x_ahead += x_step;
        dy_ahead += dy_step;
        if constexpr(!STRIDED)
            copy_async_commit();
        ahead_row += gridDim.x;
    };
    const float *mean_at = P.mean + blockIdx.x, *rstd_at = P.rstd + blockIdx.x;
    T* out               = P.dx ? static_cast<T*>(P.dx) + blockIdx.x * P.lddx + col0 : nullptr;
    const int64_t dx_step = gridDim.x * P.lddx;
    auto statistics = [&](bool on) {
        mean = on ? __ldg(mean_at) : 0.f;
        rstd = on ? __ldg(rstd_at) : 0.f;
        mean_at += gridDim.x;
        rstd_at += gridDim.x;
    };
    int64_t row = blockIdx.x;
    int slot    = 0;
    fetch(0);
    if constexpr(!STRIDED)
#pragma unroll
        for(int i = 1; i < STAGE_DEPTH - 1; ++i)
            fetch(i);
    statistics(row < P.M);
    int flip = 0;
    for(; row < P.M; row += gridDim.x)
    {
        if constexpr(!STRIDED)
        {
            fetch(slot == 0 ? STAGE_DEPTH - 1 : slot - 1);
            copy_async_wait<STAGE_DEPTH - 1>();
        }
        const uint64_t m2 = pack_f32x2(-mean, -mean), r2 = pack_f32x2(rstd, rstd);
        const float rs = rstd;
        uint64_t h[V][4], w[V][4];
        uint64_t s1v = 0, s2v = 0;
#pragma unroll
        for(int v = 0; v < V; ++v)
        {
            if constexpr(!STRIDED)
            {
                ring.read(rx[v], slot, v);
                ring.read(ry[v], slot, V + v);
            }
            uint64_t gy[4];
            to_pairs(rx[v], h[v]);
            to_pairs(ry[v], gy);
#pragma unroll
            for(int i = 0; i < 4; ++i)
            {
                h[v][i] = mul_f32x2(add_f32x2(h[v][i], m2), r2);
                w[v][i] = mul_f32x2(gy[i], g[v][i]);
            }
            if(!STRIDED && TAIL && have - v * 256 < 8)
                keep_first(h[v], have - v * 256);
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
        if constexpr(STRIDED)
            fetch(0);
        statistics(row + gridDim.x < P.M);
        row_sum2<ROW_CTA, V == 1>(s1, s2, buf + flip, 0, tpr); // (one vector a thread: more than 16 warps)
        flip ^= 64;
        if(P.dx)
        {
            const float c1 = s1 * inv_n, c2 = s2 * inv_n;
            const uint64_t c1v = pack_f32x2(-c1, -c1), c2v = pack_f32x2(-c2, -c2), rsv = pack_f32x2(rs, rs);
#pragma unroll
            for(int v = 0; v < V; ++v)
            {
                float o[8];
#pragma unroll
                for(int i = 0; i < 4; ++i)
                    unpack_f32x2(mul_f32x2(rsv, fma_f32x2(h[v][i], c2v, add_f32x2(w[v][i], c1v))), o[2 * i], o[2 * i + 1]);
                if constexpr(STRIDED)
                {
#pragma unroll
                    for(int i = 0; i < 8; ++i)
                    {
                        const int c = column_of<1, true>(v, i, t, tpr);
                        if(c < P.N)
                            out[c] = from_f32<T>(o[i]);
                    }
                }
                else
                {
                    store8(o, out + v * 256, have - v * 256, true);
                }
            }
        }
        if(P.dx)
            out += dx_step;
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
                const int c = column_of<V, STRIDED>(v, i, t, tpr);
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

// The same for 16-bit rows that start anywhere: they come and go through shared memory in whole 16-byte pieces, as in the
// forward pass (8192 x 4097 bf16: 111 us, STRIDED 249; with rows on 16-byte boundaries the kernel above takes 50 us for 4096
// columns and this one 65).  Bound by its instructions: shifting and the row's ends next to 16 values a lane.
// Vector v of a lane of warp w: columns 256 (w V + v) + 8 lane .. + 7.
template <typename T, int V>
__global__ void __launch_bounds__(V == 1 ? 128 : 512, V == 1 ? 4 : 1) layernorm_bwd_shifted_kernel(const __grid_constant__ LayernormBwdParams P)
{
    grid_dependency_wait();
    grid_launch_dependents();
    extern __shared__ __align__(16) uint8_t ring_smem[];
    __shared__ float buf[2 * 64];
    const int tpr = blockDim.x, t = threadIdx.x, lane = t & 31;
    const float inv_n = 1.f / static_cast<float>(P.N);
    const int warp_col = (t >> 5) * (V * 256), warp_have = P.N - warp_col, have = warp_have - lane * 8;
    uint64_t g[V][4], dg[V][4], db[V][4];
#pragma unroll
    for(int v = 0; v < V; ++v)
    {
        const int c = warp_col + v * 256 + lane * 8;
        load_weights8<T>(g[v], P.gamma, P.w_f32 != 0, c < P.N ? c : 0, c < P.N ? P.N : 0, P.w_vec != 0, 1.f);
        if(have - v * 256 < 8)
            keep_first(g[v], have - v * 256);
#pragma unroll
        for(int i = 0; i < 4; ++i)
            dg[v][i] = db[v][i] = 0;
    }
    using Ring = WarpRing<T, V * 256>;
    const Ring x_ring(ring_smem, 0, 2), dy_ring(ring_smem, 1, 2);
    const T* x_ahead  = static_cast<const T*>(P.x) + blockIdx.x * P.ldx + (warp_have > 0 ? warp_col : 0); // of the row that is fetched next
    const T* dy_ahead = static_cast<const T*>(P.dy) + blockIdx.x * P.lddy + (warp_have > 0 ? warp_col : 0);
    const T *x_now = x_ahead, *dy_now = dy_ahead;
    const int64_t x_step = gridDim.x * P.ldx, dy_step = gridDim.x * P.lddy;
    int64_t ahead_row = blockIdx.x;
    auto fetch = [&](int slot) {
        if(ahead_row < P.M)
        {
            x_ring.copy(slot, x_ahead, warp_have);
            dy_ring.copy(slot, dy_ahead, warp_have);
        }
        copy_async_commit();
        x_ahead += x_step;
        dy_ahead += dy_step;
        ahead_row += gridDim.x;
    };
    const float *mean_at = P.mean + blockIdx.x, *rstd_at = P.rstd + blockIdx.x;
    T* out                = static_cast<T*>(P.dx) + (P.dx ? blockIdx.x * P.lddx + warp_col : 0);
    const int64_t dx_step = gridDim.x * P.lddx;
    float mean = 0.f, rstd = 0.f;
    auto statistics = [&](bool on) {
        mean = on ? __ldg(mean_at) : 0.f;
        rstd = on ? __ldg(rstd_at) : 0.f;
        mean_at += gridDim.x;
        rstd_at += gridDim.x;
    };
    int64_t row = blockIdx.x;
    int slot    = 0;
#pragma unroll
    for(int i = 0; i < STAGE_DEPTH - 1; ++i)
        fetch(i);
    statistics(row < P.M);
    int flip = 0;
    for(; row < P.M; row += gridDim.x)
    {
        __syncwarp(); // the slot that is filled now was the last row's way out
        fetch(slot == 0 ? STAGE_DEPTH - 1 : slot - 1);
        copy_async_wait<STAGE_DEPTH - 1>();
        __syncwarp();
        const int x_off = static_cast<int>(reinterpret_cast<uintptr_t>(x_now) & 15), dy_off = static_cast<int>(reinterpret_cast<uintptr_t>(dy_now) & 15);
        const uint64_t m2 = pack_f32x2(-mean, -mean), r2 = pack_f32x2(rstd, rstd);
        const float rs = rstd;
        uint64_t h[V][4], w[V][4];
        uint64_t s1v = 0, s2v = 0;
#pragma unroll
        for(int v = 0; v < V; ++v)
        {
            Vec8<T> rx, ry;
            x_ring.read(rx.w, slot, v * 256 + lane * 8, x_off);
            dy_ring.read(ry.w, slot, v * 256 + lane * 8, dy_off);
            uint64_t gy[4];
            to_pairs(rx, h[v]);
            to_pairs(ry, gy);
#pragma unroll
            for(int i = 0; i < 4; ++i)
                h[v][i] = mul_f32x2(add_f32x2(h[v][i], m2), r2);
            if(have - v * 256 < 8)
            {
                keep_first(h[v], have - v * 256); // (what lies behind the row's end was never copied)
                keep_first(gy, have - v * 256);
            }
#pragma unroll
            for(int i = 0; i < 4; ++i)
            {
                w[v][i]  = mul_f32x2(gy[i], g[v][i]);
                dg[v][i] = fma_f32x2(gy[i], h[v][i], dg[v][i]);
                db[v][i] = add_f32x2(db[v][i], gy[i]);
                s1v      = add_f32x2(s1v, w[v][i]);
                s2v      = fma_f32x2(w[v][i], h[v][i], s2v);
            }
        }
        float s1 = sum_f32x2(s1v), s2 = sum_f32x2(s2v);
        statistics(row + gridDim.x < P.M);
        row_sum2<ROW_CTA>(s1, s2, buf + flip, 0, tpr);
        flip ^= 64;
        if(P.dx && warp_have > 0)
        {
            const float c1 = s1 * inv_n, c2 = s2 * inv_n;
            const uint64_t c1v = pack_f32x2(-c1, -c1), c2v = pack_f32x2(-c2, -c2), rsv = pack_f32x2(rs, rs);
            const uint32_t stage = x_ring.base + slot * Ring::SLOT; // (the row is in registers, and all lanes have met since)
#pragma unroll
            for(int v = 0; v < V; ++v)
            {
                float o[8];
#pragma unroll
                for(int i = 0; i < 4; ++i)
                    unpack_f32x2(mul_f32x2(rsv, fma_f32x2(h[v][i], c2v, add_f32x2(w[v][i], c1v))), o[2 * i], o[2 * i + 1]);
                stage8<T>(stage + (v * 256 + lane * 8) * static_cast<int>(sizeof(T)), o);
            }
            store_span<Ring::BYTES, sizeof(T)>(stage, reinterpret_cast<uint8_t*>(out), warp_have < V * 256 ? warp_have * static_cast<int>(sizeof(T)) : Ring::BYTES);
        }
        out += dx_step;
        x_now += x_step;
        dy_now += dy_step;
        if(++slot == STAGE_DEPTH)
            slot = 0;
    }
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
                const int c = warp_col + v * 256 + lane * 8 + i;
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

// Long rows (the column sums of a thread no longer fit its registers), first half: means of w and w xhat of a row, then dx
// (the row is read twice, the second time from L2; both halves at 2048 x 16384 bf16: 105 us, 219 with a value per thread and
// load; x 16383: 192).
template <typename T, bool VEC>
__global__ void __launch_bounds__(1024) layernorm_bwd_long_kernel(const __grid_constant__ LayernormBwdParams P)
{
    grid_dependency_wait();
    grid_launch_dependents();
    __shared__ float buf[2 * 64];
    const float n = static_cast<float>(P.N);
    for(int64_t row = blockIdx.x; row < P.M; row += gridDim.x)
    {
        const T* x      = static_cast<const T*>(P.x) + row * P.ldx;
        const T* dy     = static_cast<const T*>(P.dy) + row * P.lddy;
        const float rstd = P.rstd[row];
        const uint64_t rs = pack_f32x2(rstd, rstd), minus_mean = pack_f32x2(-P.mean[row], -P.mean[row]);
        // w and xhat of eight columns (w = 0 behind the row's end)
        auto eight = [&](int64_t c, uint64_t (&w)[4], uint64_t (&h)[4]) {
            const int have = static_cast<int>(P.N - c);
            Raw8<T, VEC> ra, rb;
            Vec8<T> a, b;
            uint64_t g[4];
            fetch8(ra, dy + c, have);
            fetch8(rb, x + c, have);
            settle8(a, ra, dy + c, have);
            settle8(b, rb, x + c, have);
            load_weights8<T>(g, P.gamma, P.w_f32 != 0, static_cast<int>(c), P.N, P.w_vec != 0, 1.f);
            to_pairs(a, w);
            to_pairs(b, h);
#pragma unroll
            for(int i = 0; i < 4; ++i)
            {
                w[i] = mul_f32x2(w[i], g[i]);
                h[i] = mul_f32x2(add_f32x2(h[i], minus_mean), rs);
            }
            if(have < 8)
                keep_first(h, have);
        };
        uint64_t p1 = 0, p2 = 0, w[4], h[4];
        for(int64_t c = threadIdx.x * 8; c < P.N; c += 8192)
        {
            eight(c, w, h);
#pragma unroll
            for(int i = 0; i < 4; ++i)
            {
                p1 = add_f32x2(p1, w[i]);
                p2 = fma_f32x2(w[i], h[i], p2);
            }
        }
        float s1 = sum_f32x2(p1), s2 = sum_f32x2(p2);
        row_sum2<ROW_CTA, true>(s1, s2, buf, 0, 1024);
        const float c1 = -s1 / n, c2 = -s2 / n;
        const uint64_t c1v = pack_f32x2(c1, c1), c2v = pack_f32x2(c2, c2);
        T* out = static_cast<T*>(P.dx) + row * P.lddx;
        for(int64_t c = threadIdx.x * 8; c < P.N; c += 8192)
        {
            eight(c, w, h);
            float o[8];
#pragma unroll
            for(int i = 0; i < 4; ++i)
                unpack_f32x2(mul_f32x2(rs, fma_f32x2(h[i], c2v, add_f32x2(w[i], c1v))), o[2 * i], o[2 * i + 1]);
            store8(o, out + c, static_cast<int>(P.N - c), P.vec != 0);
        }
        __syncthreads();
    }
}
// Second half: column sums.  blockIdx.x = LONG_SLAB columns, eight a thread, blockIdx.y = one of P.parts sets of rows, two
// rows in flight.
constexpr int LONG_SLAB = 2048;
template <typename T, bool VEC>
__global__ void __launch_bounds__(LONG_SLAB / 8) layernorm_bwd_long_sums_kernel(const __grid_constant__ LayernormBwdParams P)
{
    grid_dependency_wait();
    grid_launch_dependents();
    const int64_t c = static_cast<int64_t>(blockIdx.x) * LONG_SLAB + threadIdx.x * 8;
    if(c >= P.N)
        return;
    const int have = static_cast<int>(P.N - c);
    const T* x     = static_cast<const T*>(P.x) + c;
    const T* dy    = static_cast<const T*>(P.dy) + c;
    uint64_t dg[4] = {}, db[4] = {};
    for(int64_t row = blockIdx.y; row < P.M; row += 2 * P.parts)
    {
        Raw8<T, VEC> a[2], b[2];
        float mean[2], rstd[2];
#pragma unroll
        for(int k = 0; k < 2; ++k)
        {
            const int64_t r = row + k * P.parts;
            const bool on   = r < P.M;
            mean[k]         = on ? __ldg(P.mean + r) : 0.f;
            rstd[k]         = on ? __ldg(P.rstd + r) : 0.f;
            fetch8(a[k], dy + r * P.lddy, on ? have : 0);
            fetch8(b[k], x + r * P.ldx, on ? have : 0);
        }
#pragma unroll
        for(int k = 0; k < 2; ++k)
        {
            const int64_t r = row + k * P.parts;
            Vec8<T> v;
            uint64_t g[4], h[4];
            settle8(v, a[k], dy + r * P.lddy, r < P.M ? have : 0);
            to_pairs(v, g);
            settle8(v, b[k], x + r * P.ldx, r < P.M ? have : 0);
            to_pairs(v, h);
            const uint64_t rs = pack_f32x2(rstd[k], rstd[k]), minus_mean = pack_f32x2(-mean[k], -mean[k]);
#pragma unroll
            for(int i = 0; i < 4; ++i)
            {
                dg[i] = fma_f32x2(g[i], mul_f32x2(add_f32x2(h[i], minus_mean), rs), dg[i]);
                db[i] = add_f32x2(db[i], g[i]);
            }
        }
    }
    float* pg = P.partial + blockIdx.y * static_cast<int64_t>(P.N) + c;
    float* pb = pg + static_cast<int64_t>(P.parts) * P.N;
#pragma unroll
    for(int i = 0; i < 8; ++i)
    {
        float a[2], b[2];
        unpack_f32x2(dg[i / 2], a[0], a[1]);
        unpack_f32x2(db[i / 2], b[0], b[1]);
        if(i < have)
        {
            pg[i] = a[i & 1];
            pb[i] = b[i & 1];
        }
    }
}

// Sums the partial column sums, always in the same order: 32 columns a CTA, 32 threads a column (thread s takes parts
// s, s + 32, ..., eight loads in flight; with eight threads a column this took longer than a third of a small backward
// pass, all of it latency).
template <typename T>
__global__ void __launch_bounds__(1024) layernorm_bwd_finish_kernel(const __grid_constant__ LayernormBwdParams P)
{
    grid_dependency_wait();
    grid_launch_dependents();
    __shared__ float part[32][33];
    const int lane = threadIdx.x & 31, slot = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    void* out       = blockIdx.y == 0 ? P.dgamma : P.dbeta;
    if(!out)
        return;
    const float* in = P.partial + static_cast<int64_t>(blockIdx.y) * P.parts * P.N + c;
    float sum       = 0.f;
    if(c < P.N)
    {
        for(int p = slot; p < P.parts; p += 256)
        {
            float v[8];
#pragma unroll
            for(int i = 0; i < 8; ++i)
                v[i] = p + i * 32 < P.parts ? in[static_cast<int64_t>(p + i * 32) * P.N] : 0.f;
            sum += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        }
    }
    part[slot][lane] = sum;
    __syncthreads();
    // warp s sums column s: its lanes hold the 32 partial sums
    const float total  = warp_sum(part[lane][slot]);
    const int64_t mine = static_cast<int64_t>(blockIdx.x) * 32 + slot;
    if(lane == 0 && mine < P.N)
    {
        if(P.w_f32)
            static_cast<float*>(out)[mine] = total;
        else
            static_cast<T*>(out)[mine] = from_f32<T>(total);
    }
}

} // namespace ckb
