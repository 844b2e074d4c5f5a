// voxq_rope.cu -- rotary tables, and the rotation of new tokens fused with
// their write into a paged KV cache.
#include <math.h>

#include "voxq_batch.cuh"
#include "voxq_internal.h"

namespace voxq {

struct RopeFreqs {
    double inv[128];  // angle per position of each pair
    float* out;
    int n_pos, half;
    double attn;
};

// Angles in fp64: a position of 10^5 times a frequency rounded to fp32 would
// already be off by 6e-3 radians.  Runs once per model.
__global__ void __launch_bounds__(256) rope_table_kernel(const __grid_constant__ RopeFreqs p) {
    const int64_t n = (int64_t)p.n_pos * p.half;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
        double s, c;
        sincos((double)(i / p.half) * p.inv[i % p.half], &s, &c);
        reinterpret_cast<float2*>(p.out)[i] = make_float2((float)(c * p.attn), (float)(s * p.attn));
    }
}

// One element pair per thread.
template <typename T, typename C>
__global__ void __launch_bounds__(128) rope_append_kernel(const voxq_rope d) {
    const int t = blockIdx.x, slot_h = blockIdx.y;
    const int half = d.rot_dim / 2, H = d.heads, KVH = d.kv_heads;
    const T* src;
    C* dst;
    bool turn = d.freqs != nullptr;
    if (slot_h < H) {
        src = (const T*)d.q + t * d.q_stride + slot_h * d.q_head_stride;
        dst = (C*)d.q_out + t * d.qo_stride + slot_h * d.qo_head_stride;
    } else {
        const int64_t slot = d.slots[t];
        if (slot < 0 || slot >= (int64_t)d.pages * d.page_size) return;
        const bool key = slot_h < H + KVH;
        const int h = key ? slot_h - H : slot_h - H - KVH;
        src = key ? (const T*)d.k + t * d.k_stride + h * d.k_head_stride : (const T*)d.v + t * d.v_stride + h * d.v_head_stride;
        dst = (C*)(key ? d.cache_k : d.cache_v) + (slot / d.page_size) * d.page_stride +
              (slot % d.page_size) * d.row_stride + h * d.head_stride;
        turn = turn && key;
    }
    const int rot = turn ? d.rot_dim : 0;
    const float* f = d.freqs;
    if (turn) f += (int64_t)min(max(d.positions[t], 0), d.n_pos - 1) * d.rot_dim;
    for (int i = threadIdx.x; i < rot / 2; i += 128) {
        const int i0 = d.interleaved ? 2 * i : i, i1 = d.interleaved ? 2 * i + 1 : i + half;
        const float x0 = to_f(src[i0]), x1 = to_f(src[i1]), c = f[2 * i], s = f[2 * i + 1];
        dst[i0] = from_f<C>(x0 * c - x1 * s);
        dst[i1] = from_f<C>(x0 * s + x1 * c);
    }
    for (int i = rot + threadIdx.x; i < d.head_dim; i += 128) dst[i] = from_f<C>(to_f(src[i]));
}

}  // namespace voxq

using namespace voxq;

extern "C" VoxCPMError voxq_rope_freqs(const voxq_rope_table* d, void* stream) {
    if (!d || !d->out) return VOXCPM_ERR_INTERNAL;
    if (d->n_pos < 0 || d->rot_dim < 0 || d->rot_dim % 2) return VOXCPM_ERR_SHAPE_MISMATCH;
    if (d->rot_dim > 256 || d->scaling < VOXQ_ROPE_PLAIN || d->scaling > VOXQ_ROPE_LONG) return VOXCPM_ERR_UNSUPPORTED;
    if (!(d->theta > 1.0) || !isfinite(d->theta)) return VOXCPM_ERR_SHAPE_MISMATCH;
    const bool scaled = d->scaling == VOXQ_ROPE_LINEAR || d->scaling == VOXQ_ROPE_NTK || d->scaling == VOXQ_ROPE_YARN;
    if (scaled && (!(d->factor > 0.0) || !isfinite(d->factor))) return VOXCPM_ERR_SHAPE_MISMATCH;
    if (d->scaling == VOXQ_ROPE_NTK && d->rot_dim == 2) return VOXCPM_ERR_SHAPE_MISMATCH;
    if (d->scaling == VOXQ_ROPE_YARN && d->original_len <= 0) return VOXCPM_ERR_SHAPE_MISMATCH;
    if (d->scaling == VOXQ_ROPE_LONG && !d->long_factors) return VOXCPM_ERR_INTERNAL;
    if (d->n_pos == 0 || d->rot_dim == 0) return VOXCPM_SUCCESS;
    RopeFreqs p{};
    p.out = d->out;
    p.n_pos = d->n_pos;
    p.half = d->rot_dim / 2;
    p.attn = d->attn_factor != 0.0 ? d->attn_factor : 1.0;
    double theta = d->theta;
    if (d->scaling == VOXQ_ROPE_NTK) theta *= pow(d->factor, (double)d->rot_dim / (d->rot_dim - 2));
    double lo = 0, hi = 0;
    if (d->scaling == VOXQ_ROPE_YARN) {
        const double bf = d->beta_fast != 0.0 ? d->beta_fast : 32.0, bs = d->beta_slow != 0.0 ? d->beta_slow : 1.0;
        if (!(bf > 0.0) || !(bs > 0.0)) return VOXCPM_ERR_SHAPE_MISMATCH;
        auto at = [&](double turns) { return d->rot_dim * log(d->original_len / (turns * 2 * M_PI)) / (2 * log(theta)); };
        lo = fmin(fmax(floor(at(bf)), 0.0), d->rot_dim - 1.0);
        hi = fmin(fmax(ceil(at(bs)), 0.0), d->rot_dim - 1.0);
        if (hi <= lo) hi = lo + 1e-3;  // both ends in one pair: a step there
    }
    for (int i = 0; i < p.half; i++) {
        double f = pow(theta, -2.0 * i / d->rot_dim);
        if (d->scaling == VOXQ_ROPE_LINEAR) f /= d->factor;
        if (d->scaling == VOXQ_ROPE_YARN) {
            const double g = 1.0 - fmin(fmax((i - lo) / (hi - lo), 0.0), 1.0);
            f = f * (1.0 - g) / d->factor + f * g;
        }
        if (d->scaling == VOXQ_ROPE_LONG) {
            if (!(d->long_factors[i] > 0.0)) return VOXCPM_ERR_SHAPE_MISMATCH;
            f /= d->long_factors[i];
        }
        p.inv[i] = f;
    }
    const int64_t n = (int64_t)p.n_pos * p.half;
    rope_table_kernel<<<(int)(n / 256 + 1 < 2048 ? n / 256 + 1 : 2048), 256, 0, (cudaStream_t)stream>>>(p);
    VOXQ_CUDA_TRY(cudaGetLastError());
    return VOXCPM_SUCCESS;
}

extern "C" VoxCPMError voxq_rope_append(const voxq_rope* d, void* stream) {
    if (!d) return VOXCPM_ERR_INTERNAL;
    if (d->tokens < 0 || d->heads < 0 || d->kv_heads < 0 || d->head_dim < 0 || d->rot_dim < 0 || d->pages < 0 ||
        d->page_size < 0 || d->rot_dim > d->head_dim || d->rot_dim % 2)
        return VOXCPM_ERR_SHAPE_MISMATCH;
    if (!elem_ok(d->in_dtype) || !elem_ok(d->cache_dtype) || (d->in_dtype != VOXQ_F32 && d->in_dtype != d->cache_dtype) ||
        d->head_dim % 8 || d->head_dim > 256)
        return VOXCPM_ERR_UNSUPPORTED;
    const bool turn = d->freqs && d->rot_dim;
    if (turn && d->n_pos <= 0) return VOXCPM_ERR_SHAPE_MISMATCH;
    if (!turn && d->rot_dim) return VOXCPM_ERR_INTERNAL;
    const bool store = d->kv_heads > 0 && d->pages > 0 && d->page_size > 0;
    const int heads = d->q_out ? d->heads : 0;
    if (d->tokens == 0 || d->head_dim == 0 || (heads == 0 && !store)) return VOXCPM_SUCCESS;
    if ((turn && !d->positions) || (heads && !d->q) || (store && (!d->k || !d->v || !d->cache_k || !d->cache_v || !d->slots)))
        return VOXCPM_ERR_INTERNAL;
    const int it = d->in_dtype, ct = d->cache_dtype;
    if (heads && !(rows16(d->q, d->q_stride, it) && rows16(d->q, d->q_head_stride, it) && rows16(d->q_out, d->qo_stride, ct) &&
                   rows16(d->q_out, d->qo_head_stride, ct)))
        return VOXCPM_ERR_UNSUPPORTED;
    if (store && !(rows16(d->k, d->k_stride, it) && rows16(d->k, d->k_head_stride, it) && rows16(d->v, d->v_stride, it) &&
                   rows16(d->v, d->v_head_stride, it) && rows16(d->cache_k, d->page_stride, ct) &&
                   rows16(d->cache_v, d->row_stride, ct) && rows16(d->cache_k, d->head_stride, ct)))
        return VOXCPM_ERR_UNSUPPORTED;
    voxq_rope p = *d;
    p.heads = heads;
    if (!turn) p.freqs = nullptr;
    if (!store) p.kv_heads = 0;
    const dim3 grid(p.tokens, p.heads + 2 * p.kv_heads);
    cudaStream_t st = (cudaStream_t)stream;
    with_elem(it, [&](auto x) {
        with_elem(ct, [&](auto y) { rope_append_kernel<decltype(x), decltype(y)><<<grid, 128, 0, st>>>(p); });
    });
    VOXQ_CUDA_TRY(cudaGetLastError());
    return VOXCPM_SUCCESS;
}
