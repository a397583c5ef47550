// ck_profiler sub-commands of the 8-bit products with block scales, their quantizer and layer norm:
//
//   ck_profiler gemm_ab_scale         <E 1 fp16|2 bf16|3 fp32> <form> <verify> <init> <log> <time> M N K
//   ck_profiler grouped_gemm_ab_scale <E 1 fp16|2 bf16|3 fp32> <form> <verify> <init> <log> <time> Ms N K
//       form 1: A[m, k] * B[n, k], scales 1 x 128 and 128 x 128 (forward)
//            0: A[m, k] * B[k, n], scales 1 x 128 and 128 x 128 (gradient of the input)
//            2: A[k, m] * B[k, n], scales of 128 x 1 on both    (gradient of the weights)
//       grouped, forms 1 and 0: Ms = rows of each group (comma separated); form 2: Ms = tokens of each group, padded to
//       blocks of 128, N x K = the size of each group's result
//   ck_profiler block_quantize        <X 1 fp16|2 bf16|3 fp32> <block 1 1x128|2 128x1|3 128x128> <verify> <init> <log> <time> M N
//   ck_profiler layernorm_fwd         <X 1 fp16|2 bf16|3 fp32> <out 1 y|2 8-bit|3 both> <verify> <init> <log> <time> M N
//   ck_profiler layernorm_bwd         <X 1 fp16|2 bf16|3 fp32> <verify> <init> <log> <time> M N
// 8-bit values are e4m3, weights of layer norm fp32.
#pragma once
#include "ck/library/reference_tensor_operation/cpu/reference_block_quantize.hpp"
#include "ck/library/reference_tensor_operation/cpu/reference_gemm_ab_scale.hpp"
#include "ck/library/reference_tensor_operation/cpu/reference_layernorm.hpp"
#include "ck/tensor_operation/gpu/device/device_block_quantize.hpp"
#include "ck/tensor_operation/gpu/device/device_gemm_ab_scale.hpp"
#include "ck/tensor_operation/gpu/device/device_grouped_gemm_ab_scale.hpp"
#include "ck/tensor_operation/gpu/device/device_layernorm_bwd.hpp"
#include "ck/tensor_operation/gpu/device/device_layernorm_fwd.hpp"

namespace block_scale {

using ck::type_convert;
using F8 = ck::f8_t;

// half a step of a type, relative to the value
template <typename T>
constexpr double half_step()
{
    return std::is_same<T, ck::half_t>::value ? 0x1p-11 : std::is_same<T, ck::bhalf_t>::value ? 0x1p-8 : 0x1p-24;
}

// |out - ref| <= the rounding of `out` plus `sums`, the error of the 32-bit arithmetic before it
template <typename T>
bool within(const char* what, std::size_t i, T out, double ref, double sums)
{
    const double o = type_convert<float>(out), bound = half_step<T>() * (std::abs(ref) + sums + 0x1p-14) + sums;
    if(std::abs(o - ref) <= bound)
        return true;
    std::cout << what << "[" << i << "] = " << o << ", reference " << ref << ", bound " << bound << std::endl;
    return false;
}

template <typename T>
Tensor<T> random_tensor(const HostTensorDescriptor& d, int init)
{
    Tensor<T> t(d);
    if(init == 1)
        t.GenerateTensorValue(GeneratorTensor_2<T>{-5, 5});
    else if(init == 2)
        t.GenerateTensorValue(GeneratorTensor_3<T>{-1.0, 1.0});
    return t;
}
inline Tensor<float> random_scales(std::size_t rows, std::size_t cols, int init)
{
    Tensor<float> t(std::vector<std::size_t>{rows, cols});
    if(init != 0)
        t.GenerateTensorValue(GeneratorTensor_3<float>{0.5, 2.0});
    return t;
}

// every element of a matrix from its indexes
template <typename T, typename F>
void fill(Tensor<T>& t, F&& f)
{
    t.ForEach([&](Tensor<T>& self, const std::vector<std::size_t>& i) { self(i) = f(i[0], i[1]); });
}

template <typename T>
struct OnDevice : DeviceMem
{
    explicit OnDevice(const Tensor<T>& t) : DeviceMem(sizeof(T) * t.mData.size()) { this->ToDevice(t.mData.data()); }
    T* get() { return static_cast<T*>(this->GetDeviceBuffer()); }
};

inline std::size_t pad16(std::size_t n) { return (n + 15) / 16 * 16; }
inline std::size_t blocks(std::size_t n) { return (n + 127) / 128; }

// The tiles the profiler compares: the library's own choice first.
inline std::vector<int32_t> tiles(bool ksplit)
{
    std::vector<int32_t> t{0};
    for(const int cols : {128, 192, 224, 256})
        t.push_back(CKB_SCALED_TILE(cols, 2, 1));
    for(const int cols : {16, 32, 64, 128})
        for(int ks = 1; ks <= (ksplit ? 8 : 1); ks *= 2)
            t.push_back(CKB_SCALED_TILE(cols, 1, ks));
    return t;
}

// One product (groups == 0) or one over groups; rows[g] = rows of A (forms 0, 1) or K values (form 2) of group g.
template <typename E, typename ALayout, typename BLayout, int BlockM, int BlockN>
bool product(bool verify, int init, bool time, const std::vector<std::size_t>& rows, bool grouped, bool k_groups, std::size_t M,
             std::size_t N, std::size_t K)
{
    const std::size_t G = grouped ? rows.size() : 1;
    const std::size_t nb = grouped && !k_groups ? G : 1, ne = k_groups ? G : 1; // matrices of B and of E
    const bool a_row = std::is_same<ALayout, Row>::value, b_row = std::is_same<BLayout, Row>::value;
    const std::size_t lda = pad16(a_row ? K : M), ldb = pad16(b_row ? N : K), b_size = ldb * (b_row ? K : N);
    const std::size_t kb = blocks(K), bn = (N + BlockN - 1) / BlockN;
    const auto a  = random_tensor<F8>(example::matrix_descriptor(M, K, lda, ALayout{}), init);
    const auto as = random_scales(kb, (M + BlockM - 1) / BlockM, init); // [K block][row block]
    std::vector<Tensor<F8>> b;
    std::vector<Tensor<float>> bs;
    for(std::size_t g = 0; g < nb; ++g)
    {
        b.push_back(random_tensor<F8>(example::matrix_descriptor(K, N, ldb, BLayout{}), init));
        bs.push_back(random_scales(kb, bn, init));
    }
    std::vector<int32_t> offsets{0};
    for(const std::size_t r : rows)
        offsets.push_back(offsets.back() + static_cast<int32_t>(k_groups ? blocks(r) : r));
    OnDevice<F8> a_dev(a);
    OnDevice<float> as_dev(as);
    DeviceMem b_dev(nb * b_size), bs_dev(sizeof(float) * nb * kb * bn), e_dev(sizeof(E) * ne * M * N), o_dev(sizeof(int32_t) * offsets.size());
    std::vector<F8> b_all(nb * b_size);
    std::vector<float> bs_all;
    for(std::size_t g = 0; g < nb; ++g)
    {
        std::copy(b[g].begin(), b[g].end(), b_all.begin() + g * b_size);
        bs_all.insert(bs_all.end(), bs[g].begin(), bs[g].end());
    }
    b_dev.ToDevice(b_all.data());
    bs_dev.ToDevice(bs_all.data());
    o_dev.ToDevice(offsets.data());

    Tensor<double> ref(std::vector<std::size_t>{ne * M, N}), size(std::vector<std::size_t>{ne * M, N});
    if(verify)
        for(std::size_t g = 0; g < G; ++g)
        {
            // the group's part as a problem of its own
            const std::size_t m0 = grouped && !k_groups ? offsets[g] : 0, m1 = grouped && !k_groups ? offsets[g + 1] : M;
            const std::size_t k0 = k_groups ? offsets[g] * 128 : 0, k1 = k_groups ? std::min<std::size_t>(K, offsets[g + 1] * 128) : K;
            if(m0 == m1)
                continue;
            const std::size_t bg = nb > 1 ? g : 0, e0 = k_groups ? g * M : m0;
            Tensor<double> r(std::vector<std::size_t>{m1 - m0, N}), s(std::vector<std::size_t>{m1 - m0, N});
            if(k1 > k0)
            {
                Tensor<F8> pa(std::vector<std::size_t>{m1 - m0, k1 - k0}), pb(std::vector<std::size_t>{k1 - k0, N});
                Tensor<float> pas(std::vector<std::size_t>{(m1 - m0 + BlockM - 1) / BlockM, blocks(k1 - k0)}), pbs(std::vector<std::size_t>{blocks(k1 - k0), bn});
                fill(pa, [&](std::size_t m, std::size_t k) { return a(m0 + m, k0 + k); });
                fill(pb, [&](std::size_t k, std::size_t n) { return b[bg](k0 + k, n); });
                fill(pas, [&](std::size_t m, std::size_t k) { return as(k0 / 128 + k, m0 / BlockM + m); });
                fill(pbs, [&](std::size_t k, std::size_t n) { return bs[bg](k0 / 128 + k, n); });
                ck::tensor_operation::host::ReferenceGemmABScale<F8, F8>::Run(pa, pb, pas, pbs, BlockM, BlockN, r, s);
            }
            std::copy(r.begin(), r.end(), ref.begin() + e0 * N);
            std::copy(s.begin(), s.end(), size.begin() + e0 * N);
        }

    const dev::BlockScaleStrides sa{1, static_cast<long long>(as.mDesc.GetStrides()[0])}, sb{1, static_cast<long long>(bn)};
    const std::size_t flop = 2 * M * N * K, bytes = a_dev.GetBufferSize() + b_dev.GetBufferSize() + e_dev.GetBufferSize() + as_dev.GetBufferSize() + bs_dev.GetBufferSize();
    Best best;
    bool pass = true;
    std::vector<E> out(ne * M * N);
    const float* p_as = as_dev.get();
    const float* p_bs = static_cast<const float*>(bs_dev.GetDeviceBuffer());
    auto one          = [&](auto& op, auto&& make, int32_t tile) {
        op.SetTileConfig(tile);
        auto arg = make(op);
        if(!op.IsSupportedArgument(arg.get()))
            return;
        e_dev.SetZero();
        const float ms = op.MakeInvokerPointer()->Run(arg.get(), StreamConfig{nullptr, time});
        const std::string name = op.GetTypeString() + " [" + op.GetBackendString() + "]";
        if(time)
            best.offer(name, ms, flop, bytes);
        else
            best.name = name;
        if(verify)
        {
            e_dev.FromDevice(out.data());
            bool ok = true;
            // 32-bit sums: a step per product on the tensor core, half a step per block and scaling
            for(std::size_t i = 0; i < out.size() && ok; ++i)
                ok = within("E", i, out[i], ref.mData[i], size.mData[i] * (128 * 0x1p-23 + (kb + 4) * 0x1p-24));
            pass = pass && ok;
        }
    };
    for(const int32_t tile : tiles(!grouped))
    {
        if(grouped)
        {
            constexpr bool by_k = !std::is_same<ALayout, Row>::value;
            dev::DeviceGroupedGemmABScale<by_k ? CKB_GROUP_K_BLOCKS : CKB_GROUP_ROWS, ALayout, BLayout, F8, F8, E, BlockM, BlockN> op;
            one(op, [&](auto& o) {
                return o.MakeArgumentPointer(a_dev.get(), b_dev.GetDeviceBuffer(), p_as, p_bs, e_dev.GetDeviceBuffer(),
                                             static_cast<const int32_t*>(o_dev.GetDeviceBuffer()), static_cast<int>(G), M, N, K, lda, ldb, N,
                                             sa, sb, b_size, kb * bn, M * N);
            }, tile);
        }
        else
        {
            dev::DeviceGemmABScale<ALayout, BLayout, F8, F8, E, BlockM, BlockN> op;
            one(op, [&](auto& o) {
                return o.MakeArgumentPointer(a_dev.get(), b_dev.GetDeviceBuffer(), p_as, p_bs, e_dev.GetDeviceBuffer(), M, N, K, lda, ldb, N,
                                             sa, sb);
            }, tile);
        }
    }
    best.report(grouped ? "grouped_gemm_ab_scale" : "gemm_ab_scale");
    return pass && !best.name.empty();
}

inline int profile_product(int argc, char* argv[], bool grouped)
{
    if(argc != 11)
    {
        std::printf("arg2: type of E (1: fp16; 2: bf16; 3: fp32)\n"
                    "arg3: form (1: A[m, k] * B[n, k]; 0: A[m, k] * B[k, n]; 2: A[k, m] * B[k, n])\n"
                    "arg4: verification (0: no; 1: yes)\narg5: initialization (0: no init; 1: integer value; 2: decimal value)\n"
                    "arg6: print tensor value (0: no; 1: yes)\narg7: time kernel (0=no, 1=yes)\narg8 to 10: %s, N, K\n",
                    grouped ? "Ms (comma separated)" : "M");
        return 1;
    }
    const int type = std::stoi(argv[2]), form = std::stoi(argv[3]), init = std::stoi(argv[5]);
    const bool verify = std::stoi(argv[4]), time = std::stoi(argv[7]);
    std::vector<std::size_t> rows;
    std::stringstream list(argv[8]);
    for(std::string item; std::getline(list, item, ',');)
        rows.push_back(std::stoul(item));
    std::size_t sum = 0, n = std::stoul(argv[9]), k = std::stoul(argv[10]);
    const bool k_groups = grouped && form == 2;
    for(const std::size_t r : rows)
        sum += k_groups ? blocks(r) * 128 : r;
    if(type < 1 || type > 3 || form < 0 || form > 2 || rows.empty() || sum == 0 || n == 0 || k == 0)
    {
        std::cout << "no instance for type " << type << ", form " << form << ", or an empty problem" << std::endl;
        return 1;
    }
    std::size_t M = sum;
    if(k_groups) // the result is N x K of the command line, the groups cut the summed extent
        M = n, n = k, k = sum;
    auto run = [&](auto e) {
        using E = decltype(e);
        if(form == 1)
            return product<E, Row, Col, 1, 128>(verify, init, time, rows, grouped, false, M, n, k);
        if(form == 0)
            return product<E, Row, Row, 1, 128>(verify, init, time, rows, grouped, false, M, n, k);
        return product<E, Col, Row, 1, 1>(verify, init, time, rows, grouped, k_groups, M, n, k);
    };
    const bool ok = type == 1 ? run(ck::half_t{}) : type == 2 ? run(ck::bhalf_t{}) : run(float{});
    return ok ? 0 : 1;
}

template <typename X, int BlockM, int BlockN>
bool quantize(bool verify, int init, bool time, std::size_t M, std::size_t N)
{
    const auto x = random_tensor<X>(HostTensorDescriptor(std::vector<std::size_t>{M, N}), init);
    Tensor<F8> q(std::vector<std::size_t>{M, N}), q_ref(q.mDesc);
    Tensor<float> s(std::vector<std::size_t>{(M + BlockM - 1) / BlockM, (N + BlockN - 1) / BlockN}), s_ref(s.mDesc);
    OnDevice<X> x_dev(x);
    OnDevice<F8> q_dev(q);
    OnDevice<float> s_dev(s);
    dev::DeviceBlockQuantize<X, F8, BlockM, BlockN> op;
    auto arg = op.MakeArgumentPointer(x_dev.get(), q_dev.get(), s_dev.get(), M, N, N, N, {static_cast<long long>(s.mDesc.GetStrides()[0]), 1});
    if(!op.IsSupportedArgument(arg.get()))
        return false;
    const float ms = op.MakeInvokerPointer()->Run(arg.get(), StreamConfig{nullptr, time});
    Best best;
    best.name = op.GetTypeString();
    if(time)
        best.offer(op.GetTypeString(), ms, M * N, x_dev.GetBufferSize() + q_dev.GetBufferSize() + s_dev.GetBufferSize());
    best.report("block_quantize");
    if(!verify)
        return true;
    ck::tensor_operation::host::ReferenceBlockQuantize<X, F8>::Run(x, q_ref, s_ref, BlockM, BlockN);
    q_dev.FromDevice(q.mData.data());
    s_dev.FromDevice(s.mData.data());
    for(std::size_t i = 0; i < s.mData.size(); ++i) // both are one correctly rounded division
        if(s.mData[i] != s_ref.mData[i])
            return std::cout << "scale[" << i << "] = " << s.mData[i] << ", reference " << s_ref.mData[i] << std::endl, false;
    for(std::size_t i = 0; i < q.mData.size(); ++i)
        if(type_convert<float>(q.mData[i]) != type_convert<float>(q_ref.mData[i]))
            return std::cout << "q[" << i << "] = " << type_convert<float>(q.mData[i]) << ", reference " << type_convert<float>(q_ref.mData[i]) << std::endl, false;
    return true;
}

inline int profile_block_quantize(int argc, char* argv[])
{
    if(argc != 10)
    {
        std::printf("arg2: type of X (1: fp16; 2: bf16; 3: fp32)\narg3: block (1: 1 x 128; 2: 128 x 1; 3: 128 x 128)\n"
                    "arg4: verification\narg5: initialization\narg6: print tensor value\narg7: time kernel\narg8 to 9: M, N\n");
        return 1;
    }
    const int type = std::stoi(argv[2]), block = std::stoi(argv[3]), init = std::stoi(argv[5]);
    const bool verify = std::stoi(argv[4]), time = std::stoi(argv[7]);
    const std::size_t M = std::stoul(argv[8]), N = std::stoul(argv[9]);
    if(type < 1 || type > 3 || block < 1 || block > 3 || M == 0 || N == 0)
    {
        std::cout << "no instance for type " << type << ", block " << block << ", or an empty problem" << std::endl;
        return 1;
    }
    auto run = [&](auto x) {
        using X = decltype(x);
        return block == 1 ? quantize<X, 1, 128>(verify, init, time, M, N)
                          : block == 2 ? quantize<X, 128, 1>(verify, init, time, M, N) : quantize<X, 128, 128>(verify, init, time, M, N);
    };
    const bool ok = type == 1 ? run(ck::half_t{}) : type == 2 ? run(ck::bhalf_t{}) : run(float{});
    return ok ? 0 : 1;
}

// What 32-bit layer norm may be off before its rounding, as a multiple of 2^-24 of the terms' magnitudes: the sums run over
// at most N / 32 + 16 additions in a row per thread and its partners, each quotient and root adds a few.
template <typename X>
bool layernorm_fwd(int outputs, bool verify, int init, bool time, std::size_t M, std::size_t N)
{
    const auto x     = random_tensor<X>(HostTensorDescriptor(std::vector<std::size_t>{M, N}), init);
    const auto gamma = random_scales(1, N, 1), beta = random_scales(1, N, 1);
    Tensor<float> g(std::vector<std::size_t>{N}), b(std::vector<std::size_t>{N});
    g.mData = gamma.mData;
    b.mData = beta.mData;
    Tensor<X> y(x.mDesc);
    Tensor<F8> q(std::vector<std::size_t>{M, N});
    Tensor<float> s(std::vector<std::size_t>{M, blocks(N)}), mean(std::vector<std::size_t>{M}), rstd(mean.mDesc);
    OnDevice<X> x_dev(x), y_dev(y);
    OnDevice<F8> q_dev(q);
    OnDevice<float> g_dev(g), b_dev(b), s_dev(s), mean_dev(mean), rstd_dev(rstd);
    const float eps = 1e-5f;
    const bool to_y = outputs & 1, to_q = outputs & 2;
    dev::DeviceLayernormFwd<X, float> op;
    auto arg = op.MakeArgumentPointer(x_dev.get(), g_dev.get(), b_dev.get(), to_y ? y_dev.get() : nullptr, mean_dev.get(), rstd_dev.get(),
                                      M, N, N, N, eps, to_q ? q_dev.get() : nullptr, to_q ? s_dev.get() : nullptr, N,
                                      {static_cast<long long>(blocks(N)), 1});
    if(!op.IsSupportedArgument(arg.get()))
        return false;
    const float ms = op.MakeInvokerPointer()->Run(arg.get(), StreamConfig{nullptr, time});
    Best best;
    best.name = op.GetTypeString();
    if(time)
        best.offer(op.GetTypeString(), ms, 8 * M * N, x_dev.GetBufferSize() + (to_y ? y_dev.GetBufferSize() : 0) + (to_q ? q_dev.GetBufferSize() + s_dev.GetBufferSize() : 0));
    best.report("layernorm_fwd");
    if(!verify)
        return true;
    Tensor<double> y_ref(std::vector<std::size_t>{M, N}), mean_ref(std::vector<std::size_t>{M}), rstd_ref(mean_ref.mDesc);
    ck::tensor_operation::host::ReferenceLayernormFwd<X, float>::Run(x, g, b, eps, y_ref, mean_ref, rstd_ref);
    y_dev.FromDevice(y.mData.data());
    q_dev.FromDevice(q.mData.data());
    s_dev.FromDevice(s.mData.data());
    mean_dev.FromDevice(mean.mData.data());
    rstd_dev.FromDevice(rstd.mData.data());
    const double steps = (N / 32 + 32) * 0x1p-24;
    bool ok            = true;
    for(std::size_t m = 0; m < M && ok; ++m)
    {
        double most = 0;
        for(std::size_t n = 0; n < N; ++n)
            most = std::max(most, std::abs(static_cast<double>(type_convert<float>(x(m, n)))));
        ok = within("mean", m, mean(m), mean_ref(m), steps * most) && within("rstd", m, rstd(m), rstd_ref(m), steps * rstd_ref(m));
        for(std::size_t n = 0; n < N && ok; ++n)
        {
            const double sums = steps * (2 * most * rstd_ref(m) * std::abs(g(n)) + std::abs(y_ref(m, n)) + std::abs(b(n)));
            if(to_y)
                ok = within("y", m * N + n, y(m, n), y_ref(m, n), sums);
            // an 8-bit value reads back as y to half a step of its binade (or of the subnormals, 2^-10 of a unit)
            if(to_q && ok)
            {
                const double sc = s(m, n / 128), back = sc * type_convert<float>(q(m, n));
                ok = std::abs(back - y_ref(m, n)) <= sums * 1.125 + std::abs(y_ref(m, n)) * 0x1.01p-4 + sc * 0x1p-10;
                if(!ok)
                    std::cout << "q[" << m << ", " << n << "] reads back as " << back << ", reference " << y_ref(m, n) << std::endl;
            }
        }
    }
    return ok;
}

template <typename X>
bool layernorm_bwd(bool verify, int init, bool time, std::size_t M, std::size_t N)
{
    const auto x = random_tensor<X>(HostTensorDescriptor(std::vector<std::size_t>{M, N}), init), dy = random_tensor<X>(x.mDesc, init);
    Tensor<float> g(std::vector<std::size_t>{N}), zero(g.mDesc), mean(std::vector<std::size_t>{M}), rstd(mean.mDesc), dg(g.mDesc), db(g.mDesc);
    g.GenerateTensorValue(GeneratorTensor_3<float>{0.5, 2.0});
    Tensor<double> y_ref(std::vector<std::size_t>{M, N}), mean_ref(std::vector<std::size_t>{M}), rstd_ref(mean_ref.mDesc);
    ck::tensor_operation::host::ReferenceLayernormFwd<X, float>::Run(x, g, zero, 1e-5f, y_ref, mean_ref, rstd_ref);
    std::copy(mean_ref.begin(), mean_ref.end(), mean.begin());
    std::copy(rstd_ref.begin(), rstd_ref.end(), rstd.begin());
    Tensor<X> dx(x.mDesc);
    OnDevice<X> x_dev(x), dy_dev(dy), dx_dev(dx);
    OnDevice<float> g_dev(g), mean_dev(mean), rstd_dev(rstd), dg_dev(dg), db_dev(db);
    dev::DeviceLayernormBwd<X, float> op;
    auto arg = op.MakeArgumentPointer(dy_dev.get(), x_dev.get(), g_dev.get(), mean_dev.get(), rstd_dev.get(), dx_dev.get(), dg_dev.get(),
                                      db_dev.get(), M, N, N, N, N);
    if(!op.IsSupportedArgument(arg.get()))
        return false;
    DeviceMem workspace(op.GetWorkSpaceSize(arg.get()));
    op.SetWorkSpacePointer(arg.get(), workspace.GetDeviceBuffer());
    const float ms = op.MakeInvokerPointer()->Run(arg.get(), StreamConfig{nullptr, time});
    Best best;
    best.name = op.GetTypeString();
    if(time)
        best.offer(op.GetTypeString(), ms, 15 * M * N, 3 * x_dev.GetBufferSize());
    best.report("layernorm_bwd");
    if(!verify)
        return true;
    Tensor<double> dx_ref(std::vector<std::size_t>{M, N}), dg_ref(std::vector<std::size_t>{N}), db_ref(dg_ref.mDesc);
    ck::tensor_operation::host::ReferenceLayernormBwd<X, float>::Run(dy, x, g, mean, rstd, dx_ref, dg_ref, db_ref);
    dx_dev.FromDevice(dx.mData.data());
    dg_dev.FromDevice(dg.mData.data());
    db_dev.FromDevice(db.mData.data());
    bool ok = true;
    auto xh = [&](std::size_t m, std::size_t n) { return (static_cast<double>(type_convert<float>(x(m, n))) - mean(m)) * rstd(m); };
    for(std::size_t m = 0; m < M && ok; ++m)
    {
        double top = 0, top_w = 0; // largest (|x| + |mean|) * rstd and |dy * gamma| of the row
        for(std::size_t n = 0; n < N; ++n)
        {
            top   = std::max(top, (std::abs(type_convert<float>(x(m, n))) + std::abs(mean(m))) * static_cast<double>(rstd(m)));
            top_w = std::max(top_w, std::abs(static_cast<double>(type_convert<float>(dy(m, n))) * g(n)));
        }
        const double sums = (N / 32 + 32) * 0x1p-24 * rstd(m) * top_w * (2 + top * top);
        for(std::size_t n = 0; n < N && ok; ++n)
            ok = within("dx", m * N + n, dx(m, n), dx_ref(m, n), sums);
    }
    for(std::size_t n = 0; n < N && ok; ++n)
    {
        double sg = 0, sb = 0;
        for(std::size_t m = 0; m < M; ++m)
        {
            const double d = std::abs(type_convert<float>(dy(m, n)));
            sg += d * (std::abs(xh(m, n)) + 2 * std::abs(mean(m)) * rstd(m));
            sb += d;
        }
        ok = within("dgamma", n, dg(n), dg_ref(n), (M + 8) * 0x1p-24 * sg) && within("dbeta", n, db(n), db_ref(n), (M + 8) * 0x1p-24 * sb);
    }
    return ok;
}

// `extra`: an argument between the type and the flags (the outputs of the forward pass)
inline int profile_layernorm(int argc, char* argv[], bool backward)
{
    const int extra = backward ? 0 : 1;
    if(argc != 9 + extra)
    {
        std::printf("arg2: type of X (1: fp16; 2: bf16; 3: fp32)\n%sthen: verification, initialization, print tensor value, time kernel, M, N\n",
                    backward ? "" : "arg3: outputs (1: y; 2: 8-bit; 3: both)\n");
        return 1;
    }
    const int type = std::stoi(argv[2]), outputs = backward ? 0 : std::stoi(argv[3]);
    char** rest = argv + 3 + extra;
    const bool verify = std::stoi(rest[0]), time = std::stoi(rest[3]);
    const int init      = std::stoi(rest[1]);
    const std::size_t M = std::stoul(rest[4]), N = std::stoul(rest[5]);
    if(type < 1 || type > 3 || (!backward && (outputs < 1 || outputs > 3)) || M == 0 || N == 0)
    {
        std::cout << "no instance for type " << type << ", outputs " << outputs << ", or an empty problem" << std::endl;
        return 1;
    }
    auto run = [&](auto x) {
        using X = decltype(x);
        return backward ? layernorm_bwd<X>(verify, init, time, M, N) : layernorm_fwd<X>(outputs, verify, init, time, M, N);
    };
    const bool ok = type == 1 ? run(ck::half_t{}) : type == 2 ? run(ck::bhalf_t{}) : run(float{});
    return ok ? 0 : 1;
}

} // namespace block_scale
