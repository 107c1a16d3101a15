// Host helpers that the C ABI's translation units share: errors, device properties, launches.  Defined in hogatt_api.cu where they
// are more than a line.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>

#include "../../include/hogatt.h"

namespace hogatt {

extern thread_local int tl_last_cuda_error;

#define HOGATT_CUDA_OK(expr)                         \
    do {                                             \
        cudaError_t err__ = (expr);                  \
        if (err__ != cudaSuccess) {                  \
            tl_last_cuda_error = (int)err__;         \
            (void)cudaGetLastError();                \
            return HOGATT_ERR_CUDA;                  \
        }                                            \
    } while (0)

constexpr int kMaxDevices = 64;

int current_device_info(int* dev, int* sms, int* smem_optin);

// cudaFuncSetAttribute(MaxDynamicSharedMemorySize) once per (kernel instantiation, device).
template <class Kernel>
int ensure_smem_limit(Kernel kernel, int dev, size_t bytes, std::atomic<size_t>* granted /*[kMaxDevices]*/) {
    if (bytes <= 48 * 1024) return HOGATT_OK;
    if (granted[dev].load(std::memory_order_acquire) >= bytes) return HOGATT_OK;
    HOGATT_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    granted[dev].store(bytes, std::memory_order_release);
    return HOGATT_OK;
}

// Launch with the programmatic-stream-serialization attribute: the kernel may be scheduled while its
// stream predecessor is still running (each of our kernels calls griddepcontrol.wait before it touches
// global memory that earlier work may write -- everything except the K/V rows of fragments the caller
// declared stable).  On unless HOGATT_PDL=0 is set in the environment when the library is first used.
bool pdl_enabled();

template <class... KArgs, class... Args>
cudaError_t launch_kernel(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
}

// A tiled tensor map with the 128-byte swizzle over a dense row-major tensor of 16-bit elements: dims[0] is the contiguous one, box[0] = 64
// elements = 128 bytes.
int encode_map(CUtensorMap* out, const void* base, int dtype, int rank, const cuuint64_t* dims, const cuuint32_t* box);

bool paged_mma_disabled();  // HOGATT_PAGED_MMA=0: the paged operators stay on the CUDA cores
bool dense_disabled();      // HOGATT_DENSE=0: AUTO keeps away from the tcgen05 kernels

inline size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }
inline size_t dtype_size(int dtype) { return dtype == HOGATT_F32 ? 4 : 2; }
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

}  // namespace hogatt
