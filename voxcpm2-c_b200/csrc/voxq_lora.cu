// voxq_lora.cu -- low-rank adapters of many requests beside a shared projection.
#include "voxq_batch.cuh"
#include "voxq_internal.h"

namespace voxq {

constexpr int kLoraThreads = 256;
constexpr int kLoraMaxRank = 128;

// The request that owns row m: the last s with cu[s] <= m.
__device__ __forceinline__ int owner(const int32_t* __restrict__ cu, int batch, int m) {
    int lo = 0, hi = batch - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (cu[mid] <= m) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// One row per CTA: h = scale A x in shared memory (a warp per rank), then every
// thread its output columns.
template <typename T, typename W>
__global__ void __launch_bounds__(kLoraThreads) lora_kernel(const voxq_lora d) {
    __shared__ float h[kLoraMaxRank];
    const int m = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int w = d.batch ? d.adapter[owner(d.cu, d.batch, m)] : -1;
    const bool on = w >= 0 && w < d.adapters;
    const int rank = !on ? 0 : d.ranks ? min(max(d.ranks[w], 0), d.rank) : d.rank;
    const T* x = (const T*)d.x + m * d.ldx;
    for (int r = warp; r < rank; r += kLoraThreads / 32) {
        const W* a = (const W*)d.a + ((int64_t)w * d.rank + r) * d.K;
        float s = 0.0f;
        for (int k = lane; k < d.K; k += 32) s = fmaf(to_f(x[k]), to_f(a[k]), s);
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) h[r] = s * d.scale[w];
    }
    __syncthreads();
    for (int n = threadIdx.x; n < d.N; n += kLoraThreads) {
        float s = 0.0f;
        for (int r = 0; r < rank; r++) s = fmaf(h[r], to_f(((const W*)d.b)[((int64_t)w * d.N + n) * d.rank + r]), s);
        if (d.base) s += to_f(((const T*)d.base)[m * d.ldb + n]);
        ((T*)d.out)[m * d.ldo + n] = from_f<T>(s);
    }
}

}  // namespace voxq

using namespace voxq;

extern "C" VoxCPMError voxq_lora_forward(const voxq_lora* d, void* stream) {
    if (!d) return VOXCPM_ERR_INTERNAL;
    if (d->rows < 0 || d->batch < 0 || d->K < 0 || d->N < 0 || d->rank < 0 || d->adapters < 0 || (d->rows && !d->batch))
        return VOXCPM_ERR_SHAPE_MISMATCH;
    if (!elem_ok(d->dtype) || !elem_ok(d->w_dtype) || (d->dtype != VOXQ_F32 && d->dtype != d->w_dtype) || d->K % 8 ||
        d->N % 8 || d->rank % 8 || d->rank > kLoraMaxRank)
        return VOXCPM_ERR_UNSUPPORTED;
    if (d->rows == 0 || d->N == 0) return VOXCPM_SUCCESS;
    const bool weights = d->adapters && d->rank && d->K;
    if (!d->out || !d->cu || !d->adapter || (weights && (!d->x || !d->a || !d->b || !d->scale))) return VOXCPM_ERR_INTERNAL;
    if (!rows16(d->out, d->ldo, d->dtype) || (d->base && !rows16(d->base, d->ldb, d->dtype)) ||
        (weights && (!rows16(d->x, d->ldx, d->dtype) || !rows16(d->a, 0, d->w_dtype) || !rows16(d->b, 0, d->w_dtype))))
        return VOXCPM_ERR_UNSUPPORTED;
    voxq_lora p = *d;
    if (!weights) p.adapters = 0;
    cudaStream_t st = (cudaStream_t)stream;
    with_elem(p.dtype, [&](auto x) {
        with_elem(p.w_dtype, [&](auto w) { lora_kernel<decltype(x), decltype(w)><<<p.rows, kLoraThreads, 0, st>>>(p); });
    });
    VOXQ_CUDA_TRY(cudaGetLastError());
    return VOXCPM_SUCCESS;
}
