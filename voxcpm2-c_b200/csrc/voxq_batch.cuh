// voxq_batch.cuh -- element types and argument checks shared by the operators
// of a batched decoder step (rotary cache append, paged attention, low-rank
// adapters, fused norms).
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

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

template <typename T>
constexpr bool is_f32 = std::is_same<T, float>::value;

// Four elements of a 16-byte row as fp32.
template <typename T>
__device__ __forceinline__ void load4(float (&x)[4], const T* p) {
    T e[4];
    if constexpr (is_f32<T>) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        memcpy(e, &v, 16);
    } else {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        memcpy(e, &v, 8);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = to_f(e[i]);
}

// 16 bytes to shared memory, zeros when !ok (the source is then not read).
__device__ __forceinline__ void cp_async16_or_zero(void* dst, const void* src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(ok ? 16 : 0) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma8(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x as a sum of two TF32 values, the high one rounded to nearest, the low one cut: what is left out is below 2^-22 of it.
// In integer operations, as conversions run at a fraction of their rate (5 sequences of 80 fp32 tokens on 1200 keys: 80 us,
// 94 with conversions).  A NaN whose bits the rounding carries over stays one in the low part.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}

// Calls f with a value of the element type that `dtype` names.
template <typename F>
auto with_elem(int dtype, F f) {
    if (dtype == VOXQ_F16) return f(__half{});
    if (dtype == VOXQ_BF16) return f(bf16{});
    return f(float{});
}

// The request (or sequence) whose rows fill tile `tile` of a ragged batch, when
// the items of request s own tiles cu[s] * mul / TM + s on: as many as they can
// need, with gaps, so no scan is needed -- it is the last s whose first tile is
// not past this one.  All threads of the block take part; batch > 0.
template <int TM>
__device__ __forceinline__ int tile_owner(const int32_t* __restrict__ cu, int batch, int mul, int tile) {
    int s = -1;
    for (int i0 = 0; i0 < batch; i0 += blockDim.x) {
        const int i = i0 + threadIdx.x;
        s += __syncthreads_count(i < batch && __ldg(cu + i) * mul / TM + i <= tile);
    }
    return max(s, 0);
}

}  // namespace voxq
