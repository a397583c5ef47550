// What the host sides of the library share (defined in ckb_api.cu): error text, device information, tensor maps,
// launch and timing.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/ckb200.h"

namespace ckb {

// Sets the calling thread's error message and returns `code`.
int host_fail(int code, const char* fmt, ...);

struct HostDevice
{
    int sm_count;
    uint32_t* status; // device status word of the bounded waits
    uint64_t wait_limit_ns;
};
int host_device(HostDevice* out);

// The SMs that a process may use of a device with `sm_count` of them (CKB_SM_LIMIT).
int host_limited_sms(int sm_count);

// Refuses a pointer that kernels of the current device cannot read: host memory, or memory of another device.
// nullptr passes (optional tensors).
int host_check_pointer(const void* p, const char* what);

// 8-bit matrix [rows][inner] (pitch in bytes; `batch` matrices `batch_pitch` bytes apart when batch >= 1) -> tensor
// map with a box of 128 bytes x box_rows, 128-byte swizzle.  The maps are cached per thread.
int host_encode_8bit(CUtensorMap* tm, const void* ptr, int64_t rows, int64_t inner, int64_t pitch, int box_rows,
                     int64_t batch, int64_t batch_pitch, const char* what);

// CKB_NO_PDL (see programmatic_launch_enabled): kernels are launched with the programmatic-stream-serialization
// attribute and wait (griddepcontrol.wait) before they touch global memory.
void host_add_pdl(cudaLaunchAttribute* attrs, int* n);

void host_note_plan(const char* fmt, ...); // ckb_last_plan
void host_count_launches(uint64_t n);      // ckb_launch_count

// One launch, or the reference's timing protocol (kernel_launch.hpp:12-74): a warm-up, then n_rep between two events.
// `once` issues the call's launches and returns a cudaError_t; `launches` = how many kernels that is.
template <typename Once>
int host_run_timed(Once once, int launches, cudaStream_t stream, int n_rep, float* avg_ms)
{
    if(avg_ms)
        *avg_ms = 0.f;
    auto failed = [](cudaError_t e) { return host_fail(CKB_ERR_CUDA, "kernel launch failed: %s", cudaGetErrorString(e)); };
    cudaError_t e = once();
    if(e != cudaSuccess)
        return failed(e);
    host_count_launches(launches);
    if(n_rep <= 0)
        return CKB_OK;
    cudaEvent_t start = nullptr, stop = nullptr;
    float total = 0.f;
    e = cudaEventCreate(&start);
    if(e == cudaSuccess)
        e = cudaEventCreate(&stop);
    if(e == cudaSuccess)
        e = cudaDeviceSynchronize();
    if(e == cudaSuccess)
        e = cudaEventRecord(start, stream);
    for(int i = 0; i < n_rep && e == cudaSuccess; ++i)
    {
        e = once();
        host_count_launches(launches);
    }
    if(e == cudaSuccess)
        e = cudaEventRecord(stop, stream);
    if(e == cudaSuccess)
        e = cudaEventSynchronize(stop);
    if(e == cudaSuccess)
        e = cudaEventElapsedTime(&total, start, stop);
    if(start)
        cudaEventDestroy(start);
    if(stop)
        cudaEventDestroy(stop);
    if(e != cudaSuccess)
        return failed(e);
    if(avg_ms)
        *avg_ms = total / n_rep;
    return CKB_OK;
}

} // namespace ckb
