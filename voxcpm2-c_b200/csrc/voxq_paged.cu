// voxq_paged.cu -- attention of a ragged batch's new tokens over a paged KV cache.
#include <math.h>

#include "voxq_batch.cuh"
#include "voxq_internal.h"

namespace voxq {

constexpr int kPagedThreads = 128;
constexpr int kPagedMaxHeadDim = 256;

// The sequence that owns token t: the last s with cu[s] <= t.
__device__ __forceinline__ int owner_seq(const int32_t* __restrict__ cu, int batch, int t) {
    int lo = 0, hi = batch - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (cu[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// One query row of one head per CTA.  Running maximum m and sum l of the
// softmax over tiles of 128 keys: a thread scores one key, then owns the
// output dimensions threadIdx.x and threadIdx.x + 128.
template <typename T>
__global__ void __launch_bounds__(kPagedThreads) paged_attn_kernel(const voxq_paged_attn d) {
    __shared__ float qs[kPagedMaxHeadDim], ps[kPagedThreads], red[kPagedThreads / 32];
    __shared__ int64_t rows[kPagedThreads];
    const int t = blockIdx.x, h = blockIdx.y, kh = h / (d.heads / d.kv_heads);
    const int s = owner_seq(d.cu_q, d.batch, t);
    const int n = d.cu_q[s + 1] - d.cu_q[s], i = t - d.cu_q[s];
    const int len = min(max(d.kv_len[s], 0), d.max_kv);
    const int seen = i < 0 || i >= n ? 0 : d.causal ? min(len, len - n + i + 1) : len;
    const T* q = (const T*)d.q + t * d.q_stride + h * d.q_head_stride;
    for (int c = threadIdx.x; c < d.head_dim; c += kPagedThreads) qs[c] = to_f(q[c]) * d.scale;
    float m = -INFINITY, l = 0.0f, acc[2] = {0.0f, 0.0f};
    for (int t0 = 0; t0 < seen; t0 += kPagedThreads) {
        __syncthreads();
        const int j = t0 + threadIdx.x;
        float v = -INFINITY;
        if (j < seen) {
            int page = d.block_table[s * d.table_stride + j / d.page_size];
            if (page < 0 || page >= d.pages) page = 0;
            const int64_t row = page * d.page_stride + (j % d.page_size) * d.row_stride + kh * d.head_stride;
            rows[threadIdx.x] = row;
            const T* k = (const T*)d.k + row;
            v = 0.0f;
            for (int c = 0; c < d.head_dim; c++) v = fmaf(qs[c], to_f(k[c]), v);
        }
        float mx = v;
#pragma unroll
        for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = mx;
        __syncthreads();
        const float mn = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
        ps[threadIdx.x] = j < seen ? expf(v - mn) : 0.0f;
        __syncthreads();
        const float f = m == -INFINITY ? 0.0f : expf(m - mn);
        m = mn;
        l *= f;
        acc[0] *= f;
        acc[1] *= f;
        for (int jj = 0; jj < min(kPagedThreads, seen - t0); jj++) {
            l += ps[jj];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int c = threadIdx.x + e * kPagedThreads;
                if (c < d.head_dim) acc[e] = fmaf(ps[jj], to_f(((const T*)d.v)[rows[jj] + c]), acc[e]);
            }
        }
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const int c = threadIdx.x + e * kPagedThreads;
        if (c >= d.head_dim) continue;
        const int64_t at = t * d.o_stride + h * d.o_head_stride + c;
        if (d.out_dtype == VOXQ_F32) ((float*)d.out)[at] = seen > 0 ? acc[e] * inv : 0.0f;
        else ((T*)d.out)[at] = from_f<T>(seen > 0 ? acc[e] * inv : 0.0f);
    }
}

static VoxCPMError paged_check(const voxq_paged_attn* d) {
    if (!d) return VOXCPM_ERR_INTERNAL;
    if (d->batch < 0 || d->heads < 0 || d->kv_heads < 0 || d->head_dim < 0 || d->pages < 0 || d->page_size < 0 ||
        d->total_q < 0 || d->max_q < 0 || d->max_kv < 0)
        return VOXCPM_ERR_SHAPE_MISMATCH;
    if (!elem_ok(d->dtype) || (d->out_dtype != d->dtype && d->out_dtype != VOXQ_F32) || d->head_dim % 8 ||
        d->head_dim > kPagedMaxHeadDim)
        return VOXCPM_ERR_UNSUPPORTED;
    if (d->total_q == 0 || d->heads == 0 || d->head_dim == 0) return VOXCPM_SUCCESS;
    if (d->batch == 0 || d->kv_heads == 0 || d->heads % d->kv_heads) return VOXCPM_ERR_SHAPE_MISMATCH;
    if (d->max_kv && (d->page_size == 0 || d->pages == 0 || d->table_stride < (d->max_kv + (int64_t)d->page_size - 1) / d->page_size))
        return VOXCPM_ERR_SHAPE_MISMATCH;
    return VOXCPM_SUCCESS;
}

}  // namespace voxq

using namespace voxq;

extern "C" size_t voxq_paged_attention_workspace(const voxq_paged_attn* d) { return 0; }

extern "C" VoxCPMError voxq_paged_attention(const voxq_paged_attn* d, void* stream) {
    const VoxCPMError e = paged_check(d);
    if (e != VOXCPM_SUCCESS || d->total_q == 0 || d->heads == 0 || d->head_dim == 0) return e;
    if (!d->q || !d->out || !d->cu_q || !d->kv_len || (d->max_kv && (!d->k || !d->v || !d->block_table))) return VOXCPM_ERR_INTERNAL;
    if (!rows16(d->q, d->q_stride, d->dtype) || !rows16(d->q, d->q_head_stride, d->dtype) ||
        !rows16(d->out, d->o_stride, d->out_dtype) || !rows16(d->out, d->o_head_stride, d->out_dtype) ||
        (d->max_kv && (!rows16(d->k, d->page_stride, d->dtype) || !rows16(d->v, d->row_stride, d->dtype) || !rows16(d->k, d->head_stride, d->dtype))))
        return VOXCPM_ERR_UNSUPPORTED;
    voxq_paged_attn p = *d;
    if (p.scale == 0.0f) p.scale = 1.0f / sqrtf((float)p.head_dim);
    with_elem(p.dtype, [&](auto x) {
        paged_attn_kernel<decltype(x)><<<dim3(p.total_q, p.heads), kPagedThreads, 0, (cudaStream_t)stream>>>(p);
    });
    VOXQ_CUDA_TRY(cudaGetLastError());
    return VOXCPM_SUCCESS;
}
