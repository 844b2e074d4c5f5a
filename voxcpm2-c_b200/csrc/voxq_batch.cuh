// voxq_batch.cuh -- element types and argument checks shared by the operators
// of a batched decoder step (rotary cache append, paged attention, low-rank
// adapters, fused norms).
#pragma once

#include <cuda_bf16.h>

#include "voxq_common.cuh"
#include "voxq_internal.h"

namespace voxq {

using bf16 = __nv_bfloat16;

inline int elem_bytes(int dtype) { return dtype == VOXQ_F32 ? 4 : 2; }
inline bool elem_ok(int dtype) { return dtype == VOXQ_F32 || dtype == VOXQ_F16 || dtype == VOXQ_BF16; }

// base address and a stride (in elements) both multiples of 16 bytes
inline bool rows16(const void* p, int64_t stride, int dtype) {
    return ((uintptr_t)p & 15) == 0 && (stride * elem_bytes(dtype)) % 16 == 0;
}

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(bf16 x) { return __bfloat162float(x); }
// round to nearest even, the one rounding of a result held in fewer bits
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ bf16 from_f<bf16>(float x) { return __float2bfloat16_rn(x); }

// Launches with programmatic stream serialization (see pdl_enabled): the
// kernel may start while its predecessor drains and must execute pdl_wait()
// before its first access to global memory.
template <typename... P, typename... A>
inline cudaError_t launch_pdl(void (*kern)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, P(args)...);
}

// Calls f with a value of the element type that `dtype` names.
template <typename F>
auto with_elem(int dtype, F f) {
    if (dtype == VOXQ_F16) return f(__half{});
    if (dtype == VOXQ_BF16) return f(bf16{});
    return f(float{});
}

}  // namespace voxq
