// voxq_paged.cuh -- what the paged-attention kernels share: the call's sizes,
// the walk through the block table, the causal limit and the output types.
#pragma once

#include "voxq_batch.cuh"

namespace voxq {

constexpr float kLog2e = 1.4426950408889634f;

// The call's sizes as the kernels take them.
struct PagedArgs {
    voxq_paged_attn d;
    int group;        // query heads per kv head
    int page_shift;   // log2(page_size), or -1
    int split_len;    // keys per split (a multiple of the key tile)
    int splits;       // most splits a row can have; 1: none
    float scale2;     // scale * log2(e): the softmax runs in base 2
    float2* ml;       // [total_q][heads][splits] running maximum and sum
    float* acc;       // [total_q][heads][splits][head_dim] unnormalised sums
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Offset of cache position j of a sequence (its block-table row `table`) at
// kv head kh, in elements.
__device__ __forceinline__ int64_t cache_row(const PagedArgs& p, const int32_t* table, int j, int kh) {
    const int e = p.page_shift >= 0 ? j >> p.page_shift : (int)((uint32_t)j / (uint32_t)p.d.page_size);
    const int page = __ldg(table + e);
    return (int64_t)((uint32_t)page < (uint32_t)p.d.pages ? page : 0) * p.d.page_stride +
           (int64_t)(j - e * p.d.page_size) * p.d.row_stride + (int64_t)kh * p.d.head_stride;
}

// Positions that row i of a sequence's n sees.
__device__ __forceinline__ int visible(const PagedArgs& p, int len, int n, int i) {
    return p.d.causal ? max(min(len, len - n + i + 1), 0) : len;
}

template <typename T>
__device__ __forceinline__ void store_pair(const PagedArgs& p, int64_t at, float x, float y) {
    if (is_f32<T> || p.d.out_dtype == VOXQ_F32) {
        *reinterpret_cast<float2*>((float*)p.d.out + at) = make_float2(x, y);
    } else {
        T e[2] = {from_f<T>(x), from_f<T>(y)};
        uint32_t v;
        memcpy(&v, e, 4);
        *reinterpret_cast<uint32_t*>((T*)p.d.out + at) = v;
    }
}

// Attention on the tcgen05 tensor cores (voxq_paged_tc.cu): 16-bit types, head_dim 64 or 128, page_size a multiple
// of 8, scale > 0.  Launches the main kernel only.
constexpr int kTcRows = 256;  // rows of a CTA
bool paged_tc_takes(const voxq_paged_attn& d);
VoxCPMError paged_tc_launch(const PagedArgs& a, cudaStream_t st);

}  // namespace voxq
