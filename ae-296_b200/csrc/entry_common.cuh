// What the entry points share (lora_api.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <initializer_list>

namespace b200lora {

int cuda_fail(cudaError_t e);             // keeps the error's text for b200_lora_last_cuda_error; returns B200_LORA_ERR_CUDA
int sm_count();                           // of the current device
bool encode_map(CUtensorMap* out, const void* base, std::initializer_list<uint64_t> extents, std::initializer_list<uint64_t> strides,
                std::initializer_list<uint32_t> box);

// Dynamic shared memory beyond 48 KB has to be allowed once per kernel and device: all that the kernel's own leaves of a block's, so
// that threads which launch it with different sizes set the same.
constexpr int kSmemLimit = 232448;        // of a block
template <auto KERNEL>
inline cudaError_t allow_smem() {
    static std::atomic<bool> allowed[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev >= 0 && dev < 64 && allowed[dev].load(std::memory_order_relaxed))) return e;
    cudaFuncAttributes own;
    e = cudaFuncGetAttributes(&own, KERNEL);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit - (int)own.sharedSizeBytes);
    if (e == cudaSuccess && dev >= 0 && dev < 64) allowed[dev].store(true, std::memory_order_relaxed);
    return e;
}

}  // namespace b200lora
