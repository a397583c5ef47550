// CPU reference operators of the operations in block_scale_ops.hpp: one output element (or row, or block) per call, sums in
// 64 bits, work split over the host's threads.
#pragma once
#include <algorithm>
#include <cmath>
#include <thread>

#include "ck/b200/block_scale_ops.hpp"
#include "ck/b200/host_tensor.hpp"

namespace ck {
namespace tensor_operation {
namespace host {

// E and, per element, the sum of the magnitudes of its terms (what rounding errors of a 32-bit sum are measured by).
// a[m, k] with scales as[m / block_m, k / 128], b[k, n] with bs[k / 128, n / block_n].
template <typename ADataType, typename BDataType>
struct ReferenceGemmABScale
{
    static void Run(const Tensor<ADataType>& a, const Tensor<BDataType>& b, const Tensor<float>& as, const Tensor<float>& bs,
                    int block_m, int block_n, Tensor<double>& e, Tensor<double>& size)
    {
        const int K = static_cast<int>(a.mDesc.GetLengths()[1]);
        auto f      = [&](auto m, auto n) {
            double sum = 0, mag = 0;
            for(int k = 0; k < K; ++k)
            {
                const double t = static_cast<double>(type_convert<float>(a(m, k))) * type_convert<float>(b(k, n)) *
                                 as(m / block_m, k / 128) * bs(k / 128, n / block_n);
                sum += t;
                mag += std::abs(t);
            }
            e(m, n)    = sum;
            size(m, n) = mag;
        };
        make_ParallelTensorFunctor(f, e.mDesc.GetLengths()[0], e.mDesc.GetLengths()[1])(std::thread::hardware_concurrency());
    }
};

// scale = largest magnitude / largest 8-bit value (at least 2^-126, 1 for zeros), q = x / scale
template <typename XDataType, typename QDataType>
struct ReferenceBlockQuantize
{
    static void Run(const Tensor<XDataType>& x, Tensor<QDataType>& q, Tensor<float>& scale, int block_m, int block_n)
    {
        const float qmax = b200::row_dtype<QDataType>::value == CKB_F8_E4M3 ? 448.f : 57344.f;
        const std::size_t M = x.mDesc.GetLengths()[0], N = x.mDesc.GetLengths()[1];
        auto f = [&](auto bm, auto bn) {
            const std::size_t m1 = std::min<std::size_t>(M, (bm + 1) * block_m), n1 = std::min<std::size_t>(N, (bn + 1) * block_n);
            float amax = 0;
            for(std::size_t m = bm * block_m; m < m1; ++m)
                for(std::size_t n = bn * block_n; n < n1; ++n)
                    amax = std::max(amax, std::fabs(type_convert<float>(x(m, n))));
            const float s = amax == 0.f ? 1.f : std::max(amax / qmax, std::ldexp(1.f, -126));
            scale(bm, bn) = s;
            for(std::size_t m = bm * block_m; m < m1; ++m)
                for(std::size_t n = bn * block_n; n < n1; ++n)
                    q(m, n) = type_convert<QDataType>(type_convert<float>(x(m, n)) / s);
        };
        make_ParallelTensorFunctor(f, scale.mDesc.GetLengths()[0],
                                   scale.mDesc.GetLengths()[1])(std::thread::hardware_concurrency());
    }
};

// y, mean and rstd of each row
template <typename XDataType, typename WDataType>
struct ReferenceLayernormFwd
{
    static void Run(const Tensor<XDataType>& x, const Tensor<WDataType>& gamma, const Tensor<WDataType>& beta, float eps,
                    Tensor<double>& y, Tensor<double>& mean, Tensor<double>& rstd)
    {
        const std::size_t N = x.mDesc.GetLengths()[1];
        auto f              = [&](auto m) {
            double s = 0, ss = 0;
            for(std::size_t n = 0; n < N; ++n)
                s += type_convert<float>(x(m, n));
            const double mu = s / N;
            for(std::size_t n = 0; n < N; ++n)
                ss += std::pow(type_convert<float>(x(m, n)) - mu, 2);
            const double r = 1 / std::sqrt(ss / N + eps);
            for(std::size_t n = 0; n < N; ++n)
                y(m, n) = (type_convert<float>(x(m, n)) - mu) * r * type_convert<float>(gamma(n)) + type_convert<float>(beta(n));
            mean(m) = mu;
            rstd(m) = r;
        };
        make_ParallelTensorFunctor(f, x.mDesc.GetLengths()[0])(std::thread::hardware_concurrency());
    }
};

// dx of each row; dgamma and dbeta of each column
template <typename XDataType, typename WDataType>
struct ReferenceLayernormBwd
{
    static void Run(const Tensor<XDataType>& dy, const Tensor<XDataType>& x, const Tensor<WDataType>& gamma,
                    const Tensor<float>& mean, const Tensor<float>& rstd, Tensor<double>& dx, Tensor<double>& dgamma,
                    Tensor<double>& dbeta)
    {
        const std::size_t M = x.mDesc.GetLengths()[0], N = x.mDesc.GetLengths()[1];
        auto xhat = [&](auto m, auto n) { return (static_cast<double>(type_convert<float>(x(m, n))) - mean(m)) * rstd(m); };
        auto row  = [&](auto m) {
            double w0 = 0, w1 = 0;
            for(std::size_t n = 0; n < N; ++n)
            {
                const double w = static_cast<double>(type_convert<float>(dy(m, n))) * type_convert<float>(gamma(n));
                w0 += w;
                w1 += w * xhat(m, n);
            }
            for(std::size_t n = 0; n < N; ++n)
            {
                const double w = static_cast<double>(type_convert<float>(dy(m, n))) * type_convert<float>(gamma(n));
                dx(m, n)       = rstd(m) * (w - w0 / N - xhat(m, n) * w1 / N);
            }
        };
        auto col = [&](auto n) {
            double g = 0, b = 0;
            for(std::size_t m = 0; m < M; ++m)
            {
                g += type_convert<float>(dy(m, n)) * xhat(m, n);
                b += type_convert<float>(dy(m, n));
            }
            dgamma(n) = g;
            dbeta(n)  = b;
        };
        make_ParallelTensorFunctor(row, M)(std::thread::hardware_concurrency());
        make_ParallelTensorFunctor(col, N)(std::thread::hardware_concurrency());
    }
};

} // namespace host
} // namespace tensor_operation
} // namespace ck
