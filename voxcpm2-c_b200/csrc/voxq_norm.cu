// voxq_norm.cu -- the norms around a block, its gate and its residual scale in
// one pass over the rows.
#include "voxq_batch.cuh"
#include "voxq_internal.h"

namespace voxq {

constexpr int kNormThreads = 256;
constexpr int kNormMaxD = 16384;

__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.0f;
    for (int w = 0; w < kNormThreads / 32; w++) s += red[w];
    return s;
}

// One row per CTA, held in registers between the passes.
template <typename T>
__global__ void __launch_bounds__(kNormThreads) norm_residual_kernel(const voxq_norm d) {
    __shared__ float red[kNormThreads / 32];
    const int m = blockIdx.x;
    const T* y = (const T*)d.y + m * d.ldy;
    const T* x = (const T*)d.x + m * d.ldx;
    const T* g = nullptr;
    if (d.gate) {
        const int r = d.gate_index ? min(max(d.gate_index[m], 0), d.gate_rows - 1) : d.gate_rows == 1 ? 0 : m;
        g = (const T*)d.gate + r * d.ldg;
    }
    float inv = 1.0f;
    if (d.w_post) {
        float s = 0.0f;
        for (int i = threadIdx.x; i < d.D; i += kNormThreads) s += to_f(y[i]) * to_f(y[i]);
        inv = rsqrtf(block_sum(s, red) / d.D + d.eps);
    }
    constexpr int PER = kNormMaxD / kNormThreads;
    float hr[PER];
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const int i = threadIdx.x + j * kNormThreads;
        hr[j] = 0.0f;
        if (i >= d.D) continue;
        float z = to_f(y[i]);
        if (d.w_post) z = z * inv * d.w_post[i];
        if (g) z *= to_f(g[i]);
        hr[j] = to_f(x[i]) + d.alpha * z;
        s += hr[j] * hr[j];
    }
    inv = d.n_out ? rsqrtf(block_sum(s, red) / d.D + d.eps) : 0.0f;
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const int i = threadIdx.x + j * kNormThreads;
        if (i >= d.D) continue;
        if (d.h_out) ((T*)d.h_out + m * d.ldh)[i] = from_f<T>(hr[j]);
        if (d.n_out) ((T*)d.n_out + m * d.ldn)[i] = from_f<T>(hr[j] * inv * d.w_pre[i]);
    }
}

}  // namespace voxq

using namespace voxq;

extern "C" VoxCPMError voxq_norm_residual(const voxq_norm* d, void* stream) {
    if (!d) return VOXCPM_ERR_INTERNAL;
    if (d->rows < 0 || d->D < 0 || d->gate_rows < 0) return VOXCPM_ERR_SHAPE_MISMATCH;
    if (!elem_ok(d->dtype) || d->D > kNormMaxD) return VOXCPM_ERR_UNSUPPORTED;
    if (d->rows == 0 || d->D == 0) return VOXCPM_SUCCESS;
    if (!d->y || !d->x || (!d->h_out && !d->n_out) || (d->n_out && !d->w_pre)) return VOXCPM_ERR_INTERNAL;
    if (d->gate && (d->gate_rows == 0 || (!d->gate_index && d->gate_rows != 1 && d->gate_rows != d->rows)))
        return VOXCPM_ERR_SHAPE_MISMATCH;
    with_elem(d->dtype, [&](auto x) {
        norm_residual_kernel<decltype(x)><<<d->rows, kNormThreads, 0, (cudaStream_t)stream>>>(*d);
    });
    VOXQ_CUDA_TRY(cudaGetLastError());
    return VOXCPM_SUCCESS;
}
