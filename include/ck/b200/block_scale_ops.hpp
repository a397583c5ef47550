// Device operations around 8-bit products with block scales and layer norm, in the manner of device_ops.hpp: typed class
// templates with MakeArgument / MakeInvoker / IsSupportedArgument and their polymorphic forms, realised through the C ABI of
// ckb200.h (which states the formulas, layouts and limits).  A layer's chain is
//   DeviceLayernormFwd (writes 8-bit rows and their scales) or DeviceBlockQuantize -> DeviceGemmABScale
// and its gradients DeviceGemmABScale on B row-major (input) and on both operands along the tokens (weights), then
// DeviceLayernormBwd; DeviceGroupedGemmABScale does the same for experts whose row counts only the device knows.
#pragma once
#include <cmath>
#include <cstdint>
#include <cstring>

#include "ck/b200/device_ops.hpp"

namespace ck {

// 8-bit floats as they are stored; type_convert rounds to nearest even and limits what is larger to the largest value.
struct f8_t // 4 exponent bits, 3 of mantissa, largest value 448, one NaN pattern per sign, no infinity
{
    uint8_t data;
};
struct bf8_t // 5 exponent bits, 2 of mantissa, largest value 57344, infinities and NaN as in binary16
{
    uint8_t data;
};

namespace b200 {
// One decoder and encoder for both: `mant` bits of mantissa, exponent bias `bias`.
inline float f8_decode(uint8_t v, int mant, int bias, bool has_inf)
{
    const int ebits = 7 - mant, e = (v & 0x7f) >> mant, m = v & ((1 << mant) - 1), top = (1 << ebits) - 1;
    float x;
    if(has_inf && e == top)
        x = m ? NAN : INFINITY;
    else if(!has_inf && (v & 0x7f) == 0x7f)
        x = NAN;
    else
        x = std::ldexp(static_cast<float>(e ? m + (1 << mant) : m), (e ? e : 1) - bias - mant);
    return v & 0x80 ? -x : x;
}
inline uint8_t f8_encode(float x, int mant, int bias, float largest, uint8_t nan)
{
    uint32_t bits;
    std::memcpy(&bits, &x, 4);
    const uint8_t sign = static_cast<uint8_t>(bits >> 24 & 0x80);
    if(std::isnan(x))
        return sign | nan;
    const float a = std::fabs(x) < largest ? std::fabs(x) : largest;
    if(a == 0.f)
        return sign;
    int e = 0;
    std::frexp(a, &e);                                 // a = f * 2^e, f in [0.5, 1)
    e            = e - 1 < 1 - bias ? 1 - bias : e - 1; // exponent of the binade, the smallest one for subnormals
    const long q = std::lrint(std::ldexp(static_cast<double>(a), mant - e)); // nearest even (default rounding mode)
    // q counts units of the binade; reaching 2^(mant+1) carries into the next binade by itself
    return sign | static_cast<uint8_t>(((e + bias - 1) << mant) + q);
}
} // namespace b200

template <>
inline float type_convert<float, f8_t>(f8_t v)
{
    return b200::f8_decode(v.data, 3, 7, false);
}
template <>
inline f8_t type_convert<f8_t, float>(float x)
{
    return f8_t{b200::f8_encode(x, 3, 7, 448.f, 0x7f)};
}
template <>
inline float type_convert<float, bf8_t>(bf8_t v)
{
    return b200::f8_decode(v.data, 2, 15, true);
}
template <>
inline bf8_t type_convert<bf8_t, float>(float x)
{
    return bf8_t{b200::f8_encode(x, 2, 15, 57344.f, 0x7f)};
}

namespace b200 {

// CKB_* value of a type of these operations
template <typename T>
struct row_dtype;
template <>
struct row_dtype<half_t>
{
    static constexpr int32_t value     = CKB_F16;
    static constexpr const char* name = "F16";
};
template <>
struct row_dtype<bhalf_t>
{
    static constexpr int32_t value     = CKB_BF16;
    static constexpr const char* name = "BF16";
};
template <>
struct row_dtype<float>
{
    static constexpr int32_t value     = CKB_F32;
    static constexpr const char* name = "F32";
};
template <>
struct row_dtype<f8_t>
{
    static constexpr int32_t value     = CKB_F8_E4M3;
    static constexpr const char* name = "F8";
};
template <>
struct row_dtype<bf8_t>
{
    static constexpr int32_t value     = CKB_F8_E5M2;
    static constexpr const char* name = "BF8";
};

// Argument and invoker of an operation that is one descriptor of the C ABI.  Ops: `supported` and `run`.
template <typename Ops>
struct DescArgument : dev::BaseArgument
{
    typename Ops::Desc desc{};
};

template <typename Ops>
struct DescInvoker : dev::BaseInvoker
{
    float Run(const DescArgument<Ops>& arg, const StreamConfig& stream_config = StreamConfig{})
    {
        if(Ops::supported(&arg.desc) != CKB_OK)
            throw_invalid_setting();
        float ms = 0.f;
        check_runtime(Ops::run(arg, stream_config.stream_id_, stream_config.time_kernel_ ? kTimedRepeats : 0, &ms));
        return ms;
    }
    float Run(const dev::BaseArgument* p_arg, const StreamConfig& stream_config = StreamConfig{}) override
    {
        return Run(argument_cast<DescArgument<Ops>>(p_arg), stream_config);
    }
};

template <typename D, int (*Supported)(const D*), int (*Launch)(const D*, void*, int, float*)>
struct DescOps
{
    using Desc = D;
    static int supported(const Desc* d) { return Supported(d); }
    static int run(const DescArgument<DescOps>& a, void* stream, int n_rep, float* ms) { return Launch(&a.desc, stream, n_rep, ms); }
};
using ScaledGemmOps        = DescOps<ckb_scaled_gemm_desc, ckb_scaled_gemm_supported, ckb_scaled_gemm_run>;
using ScaledGroupedGemmOps = DescOps<ckb_scaled_grouped_gemm_desc, ckb_scaled_grouped_gemm_supported, ckb_scaled_grouped_gemm_run>;
using BlockQuantizeOps     = DescOps<ckb_block_quantize_desc, ckb_block_quantize_supported, ckb_block_quantize_run>;
using LayernormFwdOps      = DescOps<ckb_layernorm_fwd_desc, ckb_layernorm_fwd_supported, ckb_layernorm_fwd_run>;
struct LayernormBwdOps
{
    using Desc = ckb_layernorm_bwd_desc;
    static int supported(const Desc* d) { return ckb_layernorm_bwd_supported(d); }
    static int run(const DescArgument<LayernormBwdOps>& a, void* stream, int n_rep, float* ms)
    {
        size_t bytes = 0; // SetWorkSpacePointer's contract: memory of GetWorkSpaceSize() bytes
        if(a.p_workspace_)
            check_runtime(ckb_layernorm_bwd_workspace_size(&a.desc, &bytes));
        return ckb_layernorm_bwd_run(&a.desc, a.p_workspace_, bytes, stream, n_rep, ms);
    }
};

template <typename Ops>
struct DescOperator : dev::BaseOperator
{
    using Argument = DescArgument<Ops>;
    using Invoker  = DescInvoker<Ops>;
    static auto MakeInvoker() { return Invoker{}; }
    std::unique_ptr<dev::BaseInvoker> MakeInvokerPointer() { return std::make_unique<Invoker>(); }
    static bool IsSupportedArgument(const Argument& arg) { return Ops::supported(&arg.desc) == CKB_OK; }
    bool IsSupportedArgument(const dev::BaseArgument* p_arg) override
    {
        return IsSupportedArgument(argument_cast<Argument>(p_arg));
    }
};

} // namespace b200

namespace tensor_operation {
namespace device {

using BlockScaleStrides = std::array<long long, 2>; // elements from one block of rows (columns) to the next, from one K block to the next

// E[m, n] = sum over blocks of 128 k of AScale * BScale * sum A[m, k] * B[k, n]; a scale covers ScaleBlockM rows of A and
// ScaleBlockN columns of B (1 or 128).
template <typename ALayout, typename BLayout, typename ADataType, typename BDataType, typename EDataType, index_t ScaleBlockM,
          index_t ScaleBlockN>
struct DeviceGemmABScale : public b200::DescOperator<b200::ScaledGemmOps>
{
    static Argument MakeArgument(const void* p_a, const void* p_b, const float* p_a_scale, const float* p_b_scale, void* p_e,
                                 long long M, long long N, long long K, long long StrideA, long long StrideB, long long StrideE,
                                 BlockScaleStrides AScaleStrides, BlockScaleStrides BScaleStrides, int32_t tile_config = 0)
    {
        Argument arg;
        Fill(arg.desc, p_a, p_b, p_a_scale, p_b_scale, p_e, M, N, K, StrideA, StrideB, StrideE, AScaleStrides, BScaleStrides);
        arg.desc.tile_config = tile_config;
        return arg;
    }
    std::unique_ptr<BaseArgument> MakeArgumentPointer(const void* p_a, const void* p_b, const float* p_a_scale,
                                                      const float* p_b_scale, void* p_e, long long M, long long N, long long K,
                                                      long long StrideA, long long StrideB, long long StrideE,
                                                      BlockScaleStrides AScaleStrides, BlockScaleStrides BScaleStrides)
    {
        return std::make_unique<Argument>(MakeArgument(p_a, p_b, p_a_scale, p_b_scale, p_e, M, N, K, StrideA, StrideB, StrideE,
                                                       AScaleStrides, BScaleStrides, this->tile_config_));
    }
    std::string GetTypeString() const override { return "DeviceGemmABScale" + Types(); }
    std::string GetBackendString() const override
    {
        if(this->tile_config_ == 0)
            return "B200 tcgen05 + TMA, tile shape chosen by the library";
        const int cols = this->tile_config_ & 0xFFF, cg = (this->tile_config_ >> 12) & 0xF, ks = (this->tile_config_ >> 20) & 0xF;
        return "B200 tcgen05 + TMA, " + (cg == 2 ? "256 x " + std::to_string(cols) + " tile per CTA pair" : std::to_string(cols) + " x 128 tile") +
               (ks > 1 ? ", K split over " + std::to_string(ks) + " CTAs" : "");
    }

    static void Fill(ckb_scaled_gemm_desc& d, const void* p_a, const void* p_b, const float* p_a_scale, const float* p_b_scale,
                     void* p_e, long long M, long long N, long long K, long long StrideA, long long StrideB, long long StrideE,
                     BlockScaleStrides AScaleStrides, BlockScaleStrides BScaleStrides)
    {
        d.a_dtype          = b200::row_dtype<ADataType>::value;
        d.b_dtype          = b200::row_dtype<BDataType>::value;
        d.e_dtype          = b200::row_dtype<EDataType>::value;
        d.a_layout         = b200::layout_of<ALayout>::value;
        d.b_layout         = b200::layout_of<BLayout>::value;
        d.scale_block_m    = ScaleBlockM;
        d.scale_block_n    = ScaleBlockN;
        d.M                = M;
        d.N                = N;
        d.K                = K;
        d.lda              = StrideA;
        d.ldb              = StrideB;
        d.lde              = StrideE;
        d.a_scale_stride_m = AScaleStrides[0];
        d.a_scale_stride_k = AScaleStrides[1];
        d.b_scale_stride_n = BScaleStrides[0];
        d.b_scale_stride_k = BScaleStrides[1];
        d.p_a              = p_a;
        d.p_b              = p_b;
        d.p_a_scale        = p_a_scale;
        d.p_b_scale        = p_b_scale;
        d.p_e              = p_e;
    }
    static std::string Types()
    {
        std::ostringstream s;
        s << "<" << b200::row_dtype<ADataType>::name << ", " << b200::row_dtype<BDataType>::name << ", "
          << b200::row_dtype<EDataType>::name << ", " << ScaleBlockM << "x128, 128x" << ScaleBlockN << ">";
        return s.str();
    }
};

// The same over groups whose extents a device array of group_count + 1 int32 holds.  GroupAxis CKB_GROUP_ROWS: group g owns
// rows offsets[g] .. offsets[g + 1] of A and E and its own B; CKB_GROUP_K_BLOCKS: the K blocks offsets[g] .. offsets[g + 1]
// and its own E.
template <int GroupAxis, typename ALayout, typename BLayout, typename ADataType, typename BDataType, typename EDataType,
          index_t ScaleBlockM, index_t ScaleBlockN>
struct DeviceGroupedGemmABScale : public b200::DescOperator<b200::ScaledGroupedGemmOps>
{
    using Gemm = DeviceGemmABScale<ALayout, BLayout, ADataType, BDataType, EDataType, ScaleBlockM, ScaleBlockN>;
    static Argument MakeArgument(const void* p_a, const void* p_b, const float* p_a_scale, const float* p_b_scale, void* p_e,
                                 const int32_t* p_offsets, int group_count, long long M, long long N, long long K,
                                 long long StrideA, long long StrideB, long long StrideE, BlockScaleStrides AScaleStrides,
                                 BlockScaleStrides BScaleStrides, long long GroupStrideB, long long GroupStrideBScale,
                                 long long GroupStrideE, int32_t tile_config = 0)
    {
        Argument arg;
        Gemm::Fill(arg.desc.gemm, p_a, p_b, p_a_scale, p_b_scale, p_e, M, N, K, StrideA, StrideB, StrideE, AScaleStrides,
                   BScaleStrides);
        arg.desc.gemm.tile_config     = tile_config;
        arg.desc.group_axis           = GroupAxis;
        arg.desc.group_count          = group_count;
        arg.desc.p_offsets            = p_offsets;
        arg.desc.b_group_stride       = GroupStrideB;
        arg.desc.b_scale_group_stride = GroupStrideBScale;
        arg.desc.e_group_stride       = GroupStrideE;
        return arg;
    }
    std::unique_ptr<BaseArgument>
    MakeArgumentPointer(const void* p_a, const void* p_b, const float* p_a_scale, const float* p_b_scale, void* p_e,
                        const int32_t* p_offsets, int group_count, long long M, long long N, long long K, long long StrideA,
                        long long StrideB, long long StrideE, BlockScaleStrides AScaleStrides, BlockScaleStrides BScaleStrides,
                        long long GroupStrideB, long long GroupStrideBScale, long long GroupStrideE)
    {
        return std::make_unique<Argument>(MakeArgument(p_a, p_b, p_a_scale, p_b_scale, p_e, p_offsets, group_count, M, N, K, StrideA,
                                                       StrideB, StrideE, AScaleStrides, BScaleStrides, GroupStrideB,
                                                       GroupStrideBScale, GroupStrideE, this->tile_config_));
    }
    std::string GetTypeString() const override
    {
        return std::string("DeviceGroupedGemmABScale") + (GroupAxis == CKB_GROUP_ROWS ? "_Rows" : "_KBlocks") + Gemm::Types();
    }
};

// X (M x N) -> 8-bit values and a scale per BlockM x BlockN (1 x 128, 128 x 1 or 128 x 128)
template <typename XDataType, typename QDataType, index_t BlockM, index_t BlockN>
struct DeviceBlockQuantize : public b200::DescOperator<b200::BlockQuantizeOps>
{
    static Argument MakeArgument(const void* p_x, void* p_q, float* p_scale, long long M, long long N, long long StrideX,
                                 long long StrideQ, BlockScaleStrides ScaleStrides, bool pow2_scale = false)
    {
        Argument arg;
        auto& d          = arg.desc;
        d.x_dtype        = b200::row_dtype<XDataType>::value;
        d.q_dtype        = b200::row_dtype<QDataType>::value;
        d.block_m        = BlockM;
        d.block_n        = BlockN;
        d.pow2_scale     = pow2_scale;
        d.M              = M;
        d.N              = N;
        d.ldx            = StrideX;
        d.ldq            = StrideQ;
        d.scale_stride_m = ScaleStrides[0];
        d.scale_stride_n = ScaleStrides[1];
        d.p_x            = p_x;
        d.p_q            = p_q;
        d.p_scale        = p_scale;
        return arg;
    }
    std::unique_ptr<BaseArgument> MakeArgumentPointer(const void* p_x, void* p_q, float* p_scale, long long M, long long N,
                                                      long long StrideX, long long StrideQ, BlockScaleStrides ScaleStrides,
                                                      bool pow2_scale = false)
    {
        return std::make_unique<Argument>(MakeArgument(p_x, p_q, p_scale, M, N, StrideX, StrideQ, ScaleStrides, pow2_scale));
    }
    std::string GetTypeString() const override
    {
        std::ostringstream s;
        s << "DeviceBlockQuantize<" << b200::row_dtype<XDataType>::name << ", " << b200::row_dtype<QDataType>::name << ", "
          << BlockM << "x" << BlockN << ">";
        return s.str();
    }
    std::string GetBackendString() const override { return "B200, one pass"; }
};

// y = (x - mean) * rstd * gamma + beta per row, as XDataType (p_y) and (or) 8-bit blocks of 1 x 128 (p_q, p_q_scale)
template <typename XDataType, typename WDataType, typename QDataType = f8_t>
struct DeviceLayernormFwd : public b200::DescOperator<b200::LayernormFwdOps>
{
    static Argument MakeArgument(const void* p_x, const void* p_gamma, const void* p_beta, void* p_y, float* p_mean, float* p_rstd,
                                 long long M, long long N, long long StrideX, long long StrideY, float eps, void* p_q = nullptr,
                                 float* p_q_scale = nullptr, long long StrideQ = 0, BlockScaleStrides QScaleStrides = {0, 0})
    {
        Argument arg;
        auto& d            = arg.desc;
        d.x_dtype          = b200::row_dtype<XDataType>::value;
        d.w_dtype          = b200::row_dtype<WDataType>::value;
        d.q_dtype          = b200::row_dtype<QDataType>::value;
        d.eps              = eps;
        d.M                = M;
        d.N                = N;
        d.ldx              = StrideX;
        d.ldy              = StrideY;
        d.ldq              = StrideQ;
        d.q_scale_stride_m = QScaleStrides[0];
        d.q_scale_stride_n = QScaleStrides[1];
        d.p_x              = p_x;
        d.p_gamma          = p_gamma;
        d.p_beta           = p_beta;
        d.p_y              = p_y;
        d.p_q              = p_q;
        d.p_q_scale        = p_q_scale;
        d.p_mean           = p_mean;
        d.p_rstd           = p_rstd;
        return arg;
    }
    std::unique_ptr<BaseArgument> MakeArgumentPointer(const void* p_x, const void* p_gamma, const void* p_beta, void* p_y,
                                                      float* p_mean, float* p_rstd, long long M, long long N, long long StrideX,
                                                      long long StrideY, float eps, void* p_q = nullptr, float* p_q_scale = nullptr,
                                                      long long StrideQ = 0, BlockScaleStrides QScaleStrides = {0, 0})
    {
        return std::make_unique<Argument>(MakeArgument(p_x, p_gamma, p_beta, p_y, p_mean, p_rstd, M, N, StrideX, StrideY, eps, p_q,
                                                       p_q_scale, StrideQ, QScaleStrides));
    }
    std::string GetTypeString() const override
    {
        std::ostringstream s;
        s << "DeviceLayernormFwd<" << b200::row_dtype<XDataType>::name << ", " << b200::row_dtype<WDataType>::name << ">";
        return s.str();
    }
    std::string GetBackendString() const override { return "B200, one read of x"; }
};

// dx, dgamma, dbeta from dy, x and the forward's mean and rstd; needs a device workspace of GetWorkSpaceSize() bytes
template <typename XDataType, typename WDataType>
struct DeviceLayernormBwd : public b200::DescOperator<b200::LayernormBwdOps>
{
    static Argument MakeArgument(const void* p_dy, const void* p_x, const void* p_gamma, const float* p_mean, const float* p_rstd,
                                 void* p_dx, void* p_dgamma, void* p_dbeta, long long M, long long N, long long StrideDY,
                                 long long StrideX, long long StrideDX)
    {
        Argument arg;
        auto& d    = arg.desc;
        d.x_dtype  = b200::row_dtype<XDataType>::value;
        d.w_dtype  = b200::row_dtype<WDataType>::value;
        d.M        = M;
        d.N        = N;
        d.lddy     = StrideDY;
        d.ldx      = StrideX;
        d.lddx     = StrideDX;
        d.p_dy     = p_dy;
        d.p_x      = p_x;
        d.p_gamma  = p_gamma;
        d.p_mean   = p_mean;
        d.p_rstd   = p_rstd;
        d.p_dx     = p_dx;
        d.p_dgamma = p_dgamma;
        d.p_dbeta  = p_dbeta;
        return arg;
    }
    std::unique_ptr<BaseArgument> MakeArgumentPointer(const void* p_dy, const void* p_x, const void* p_gamma, const float* p_mean,
                                                      const float* p_rstd, void* p_dx, void* p_dgamma, void* p_dbeta, long long M,
                                                      long long N, long long StrideDY, long long StrideX, long long StrideDX)
    {
        return std::make_unique<Argument>(MakeArgument(p_dy, p_x, p_gamma, p_mean, p_rstd, p_dx, p_dgamma, p_dbeta, M, N, StrideDY,
                                                       StrideX, StrideDX));
    }
    size_t GetWorkSpaceSize(const BaseArgument* p_arg) const override
    {
        size_t bytes = 0;
        b200::check_runtime(ckb_layernorm_bwd_workspace_size(&b200::argument_cast<Argument>(p_arg).desc, &bytes));
        return bytes;
    }
    std::string GetTypeString() const override
    {
        std::ostringstream s;
        s << "DeviceLayernormBwd<" << b200::row_dtype<XDataType>::name << ", " << b200::row_dtype<WDataType>::name << ">";
        return s.str();
    }
    std::string GetBackendString() const override { return "B200, column sums in a fixed order"; }
};

} // namespace device
} // namespace tensor_operation
} // namespace ck
