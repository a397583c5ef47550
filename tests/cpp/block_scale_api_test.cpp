// Host-only checks of ck/b200/block_scale_ops.hpp (no GPU call is made): 8-bit types, what IsSupportedArgument answers, what
// an invoker throws, workspace sizes, type strings, and the CPU reference operators on values worked out by hand.
#include <cmath>
#include <cstdio>
#include <iostream>

#include "ck/ck.hpp"
#include "ck/library/reference_tensor_operation/cpu/reference_block_quantize.hpp"
#include "ck/library/reference_tensor_operation/cpu/reference_gemm_ab_scale.hpp"
#include "ck/library/reference_tensor_operation/cpu/reference_layernorm.hpp"
#include "ck/tensor_operation/gpu/device/device_block_quantize.hpp"
#include "ck/tensor_operation/gpu/device/device_gemm_ab_scale.hpp"
#include "ck/tensor_operation/gpu/device/device_grouped_gemm_ab_scale.hpp"
#include "ck/tensor_operation/gpu/device/device_layernorm_bwd.hpp"
#include "ck/tensor_operation/gpu/device/device_layernorm_fwd.hpp"

static int g_failed = 0;
#define EXPECT(cond)                                                          \
    do                                                                        \
    {                                                                         \
        if(!(cond))                                                           \
        {                                                                     \
            std::printf("FAILED %s:%d  %s\n", __FILE__, __LINE__, #cond);     \
            ++g_failed;                                                       \
        }                                                                     \
    } while(0)

using Row = ck::tensor_layout::gemm::RowMajor;
using Col = ck::tensor_layout::gemm::ColumnMajor;
namespace dev = ck::tensor_operation::device;
namespace ref = ck::tensor_operation::host;

template <typename T>
static void test_8bit(int mant, int bias, float largest)
{
    using ck::type_convert;
    float last = -1.f;
    for(int v = 0; v < 128; ++v) // every finite value comes back, in order
    {
        const float x = type_convert<float>(T{static_cast<uint8_t>(v)});
        if(!std::isfinite(x))
            continue;
        EXPECT(x > last);
        last = x;
        EXPECT((type_convert<T, float>(x).data == v));
        EXPECT((type_convert<T, float>(-x).data == (v | 0x80)));
        EXPECT(type_convert<float>(T{static_cast<uint8_t>(v | 0x80)}) == -x);
        if(x < largest)
        {
            // between two neighbours: the nearer one, the even one in the middle
            const float up = type_convert<float>(T{static_cast<uint8_t>(v + 1)}), mid = (x + up) / 2;
            EXPECT((type_convert<T, float>(mid).data == (v & 1 ? v + 1 : v)));
            EXPECT((type_convert<T, float>(std::nextafter(mid, 0.f)).data == v));
            EXPECT((type_convert<T, float>(std::nextafter(mid, largest)).data == v + 1));
        }
    }
    EXPECT(last == largest);
    EXPECT(type_convert<float>(type_convert<T, float>(1e30f)) == largest);
    EXPECT(std::isnan(type_convert<float>(type_convert<T, float>(NAN))));
    EXPECT(type_convert<float>(T{1}) == std::ldexp(1.f, 1 - bias - mant));
}

template <typename Op>
static bool throws(Op& op, const dev::BaseArgument* arg)
{
    try
    {
        op.MakeInvokerPointer()->Run(arg);
    }
    catch(const std::runtime_error&)
    {
        return true;
    }
    return false;
}

static void test_products()
{
    dev::DeviceGemmABScale<Row, Col, ck::f8_t, ck::bf8_t, ck::bhalf_t, 1, 128> op;
    EXPECT(op.GetTypeString() == "DeviceGemmABScale<F8, BF8, BF16, 1x128, 128x128>");
    auto make = [&](long long M, long long N, long long K, long long lda) {
        return op.MakeArgument(nullptr, nullptr, nullptr, nullptr, nullptr, M, N, K, lda, (K + 15) / 16 * 16, N, {1, M}, {1, 1});
    };
    EXPECT(op.IsSupportedArgument(make(5, 7, 100, 112)));
    EXPECT(!op.IsSupportedArgument(make(5, 7, 100, 100))); // pitch of 100 bytes
    EXPECT(!op.IsSupportedArgument(make(5, 7, 100, 96)));  // shorter than a row
    EXPECT(!op.IsSupportedArgument(make(0, 7, 128, 128)));
    op.SetTileConfig(CKB_SCALED_TILE(64, 1, 4)); // four slices of two K blocks at least
    EXPECT(!op.IsSupportedArgument(op.MakeArgumentPointer(nullptr, nullptr, nullptr, nullptr, nullptr, 5, 7, 512, 512, 512, 7, {1, 5}, {1, 1}).get()));
    auto ok = op.MakeArgumentPointer(nullptr, nullptr, nullptr, nullptr, nullptr, 5, 7, 1024, 1024, 1024, 7, {1, 5}, {1, 1});
    EXPECT(op.IsSupportedArgument(ok.get()));
    EXPECT(throws(op, ok.get())); // null pointers
    EXPECT(op.GetBackendString() == "B200 tcgen05 + TMA, 64 x 128 tile, K split over 4 CTAs");

    dev::DeviceGroupedGemmABScale<CKB_GROUP_ROWS, Row, Row, ck::f8_t, ck::f8_t, float, 1, 128> rows;
    auto g = [&](int groups, long long stride_b) {
        return rows.MakeArgument(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, groups, 64, 32, 128, 128, 32, 32, {1, 64}, {1, 1}, stride_b, 1, 0);
    };
    EXPECT(rows.IsSupportedArgument(g(4, 128 * 32)));
    EXPECT(!rows.IsSupportedArgument(g(0, 128 * 32)));
    EXPECT(!rows.IsSupportedArgument(g(CKB_SCALED_MAX_GROUPS + 1, 128 * 32)));
    EXPECT(!rows.IsSupportedArgument(g(4, 128 * 32 + 8)));
    dev::DeviceGroupedGemmABScale<CKB_GROUP_ROWS, Col, Row, ck::f8_t, ck::f8_t, float, 1, 128> columns; // rows of a column-major A
    EXPECT(!columns.IsSupportedArgument(columns.MakeArgument(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 4, 64, 32, 128, 64, 32, 32,
                                                             {1, 64}, {1, 1}, 4096, 1, 0)));
    EXPECT(rows.GetTypeString() == "DeviceGroupedGemmABScale_Rows<F8, F8, F32, 1x128, 128x128>");
}

static void test_rows()
{
    dev::DeviceBlockQuantize<ck::bhalf_t, ck::f8_t, 1, 128> quant;
    EXPECT(quant.IsSupportedArgument(quant.MakeArgument(nullptr, nullptr, nullptr, 3, 130, 130, 131, {2, 1})));
    EXPECT(!quant.IsSupportedArgument(quant.MakeArgument(nullptr, nullptr, nullptr, 3, 130, 129, 131, {2, 1})));
    dev::DeviceBlockQuantize<ck::bhalf_t, ck::f8_t, 64, 64> other_block;
    EXPECT(!other_block.IsSupportedArgument(other_block.MakeArgument(nullptr, nullptr, nullptr, 3, 130, 130, 131, {2, 1})));
    dev::DeviceLayernormFwd<ck::half_t, float> fwd;
    int dummy = 0;
    EXPECT(fwd.IsSupportedArgument(fwd.MakeArgument(nullptr, nullptr, nullptr, &dummy, nullptr, nullptr, 3, 130, 130, 130, 1e-5f)));
    // pointers are the run's business, as for every operation: no output is refused there
    EXPECT(throws(fwd, fwd.MakeArgumentPointer(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 3, 130, 130, 130, 1e-5f).get()));
    EXPECT(!fwd.IsSupportedArgument(fwd.MakeArgument(nullptr, nullptr, nullptr, &dummy, nullptr, nullptr, 3, 130, 130, 130, -1.f)));
    dev::DeviceLayernormBwd<ck::half_t, ck::half_t> bwd;
    auto arg = bwd.MakeArgumentPointer(nullptr, nullptr, nullptr, nullptr, nullptr, &dummy, &dummy, nullptr, 300, 130, 130, 130, 130);
    EXPECT(bwd.IsSupportedArgument(arg.get()));
    EXPECT(bwd.GetWorkSpaceSize(arg.get()) > 0);
    EXPECT(throws(bwd, arg.get()));
    EXPECT(bwd.GetTypeString() == "DeviceLayernormBwd<F16, F16>");
    // an argument of another operation
    dev::DeviceLayernormFwd<ck::half_t, ck::half_t> wrong;
    EXPECT(throws(wrong, arg.get()));
}

static void test_references()
{
    // one row of two values, K = 2 in one block: (1 * 2) * 0.5 * 4 + (3 * -1) * 0.5 * 4
    Tensor<ck::f8_t> a(std::vector<std::size_t>{1, 2}), b(std::vector<std::size_t>{2, 1});
    Tensor<float> as(std::vector<std::size_t>{1, 1}), bs(as.mDesc);
    Tensor<double> e(std::vector<std::size_t>{1, 1}), size(e.mDesc);
    const float av[] = {1, 3}, bv[] = {2, -1};
    for(int k = 0; k < 2; ++k)
        a(0, k) = ck::type_convert<ck::f8_t, float>(av[k]), b(k, 0) = ck::type_convert<ck::f8_t, float>(bv[k]);
    as(0, 0) = 0.5f, bs(0, 0) = 4.f;
    ref::ReferenceGemmABScale<ck::f8_t, ck::f8_t>::Run(a, b, as, bs, 1, 128, e, size);
    EXPECT(e(0, 0) == -2 && size(0, 0) == 10);

    Tensor<float> x(std::vector<std::size_t>{1, 3}), s(std::vector<std::size_t>{1, 1});
    Tensor<ck::f8_t> q(std::vector<std::size_t>{1, 3});
    x(0, 0) = 896.f, x(0, 1) = -2.f, x(0, 2) = 0.f;
    ref::ReferenceBlockQuantize<float, ck::f8_t>::Run(x, q, s, 1, 128);
    EXPECT(s(0, 0) == 2.f && q(0, 0).data == 0x7e && ck::type_convert<float>(q(0, 1)) == -1.f && q(0, 2).data == 0);

    // a row (-1, 1) with variance 1: eps 0 gives xhat = x
    Tensor<float> row(std::vector<std::size_t>{1, 2}), gamma(std::vector<std::size_t>{2}), beta(gamma.mDesc), mean(std::vector<std::size_t>{1}), rstd(mean.mDesc);
    row(0, 0) = -1, row(0, 1) = 1, gamma(0) = 2, gamma(1) = 3, beta(0) = 0.5f, beta(1) = 0;
    Tensor<double> y(std::vector<std::size_t>{1, 2}), m(std::vector<std::size_t>{1}), r(m.mDesc);
    ref::ReferenceLayernormFwd<float, float>::Run(row, gamma, beta, 0.f, y, m, r);
    EXPECT(y(0, 0) == -1.5 && y(0, 1) == 3 && m(0) == 0 && r(0) == 1);
    // dy (1, 1): w = (2, 3), mean of w = 2.5, mean of w * xhat = 0.5 -> dx = w - 2.5 - xhat / 2 = 0
    Tensor<float> dy(std::vector<std::size_t>{1, 2});
    dy(0, 0) = dy(0, 1) = 1;
    mean(0) = 0, rstd(0) = 1;
    Tensor<double> dx(std::vector<std::size_t>{1, 2}), dg(std::vector<std::size_t>{2}), db(dg.mDesc);
    ref::ReferenceLayernormBwd<float, float>::Run(dy, row, gamma, mean, rstd, dx, dg, db);
    EXPECT(dx(0, 0) == 0 && dx(0, 1) == 0 && dg(0) == -1 && dg(1) == 1 && db(0) == 1 && db(1) == 1);
}

int main()
{
    test_8bit<ck::f8_t>(3, 7, 448.f);
    test_8bit<ck::bf8_t>(2, 15, 57344.f);
    test_products();
    test_rows();
    test_references();
    if(g_failed)
    {
        std::printf("%d checks failed\n", g_failed);
        return 1;
    }
    std::printf("all block scale API checks passed\n");
    return 0;
}
