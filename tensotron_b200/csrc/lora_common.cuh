// Device helpers shared by the adapter kernels.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "ptx.cuh"

namespace tt {
namespace lora {

__device__ __forceinline__ float act_apply(float v, int act)
{
    if (act == 1) return v > 0.f ? v : 0.f;
    if (act == 2) return tanhf(v);
    return v;
}

// Asynchronous copies, global -> shared: one float, or four consecutive ones of which the first `n` exist (the others
// become 0; nothing is read when n <= 0, but `src` has to be a valid address).
__device__ __forceinline__ void copy1(float* dst, const float* src, bool there)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 4 : 0) : "memory");
}

__device__ __forceinline__ void copy4(float* dst, const float* src, int n, bool vec)
{
    if (vec) {
        // (a vector copy never meets a partial group: the rows are a multiple of four long)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(n > 0 ? 16 : 0) : "memory");
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) copy1(dst + i, i < n ? src + i : src, i < n);
    }
}

// Sixteen bytes, all there.
__device__ __forceinline__ void copy16(float* dst, const float* src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// Waits until at most N of the calling thread's copy groups are unfinished.
template <int N>
__device__ __forceinline__ void wait_copies()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

}  // namespace lora
}  // namespace tt
