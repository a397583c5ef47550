#include "ckb_scaled_launch.cuh"

namespace ckb {
template cudaError_t launch_scaled<0, 1>(int, const ScaledParams&, int, cudaStream_t, int, int*);
}
