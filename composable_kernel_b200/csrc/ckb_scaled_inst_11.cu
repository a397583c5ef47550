#include "ckb_scaled_launch.cuh"

namespace ckb {
template cudaError_t launch_scaled<1, 1>(int, const ScaledParams&, int, cudaStream_t, int, int*);
}
