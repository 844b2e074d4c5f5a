// voxq_rope.cu -- rotary tables, and the rotation of new tokens fused with
// their write into a paged KV cache.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "voxq_batch.cuh"
#include "voxq_internal.h"

namespace voxq {

constexpr int kRopeThreads = 256;

struct RopeFreqs {
    double inv[128];  // angle per position of each pair
    float* out;
    int n_pos, half;
    double attn;
};

// Angles in fp64: a position of 10^5 times a frequency rounded to fp32 would
// already be off by 6e-3 radians.  Bound by fp64 sincos; runs once per model.
__global__ void __launch_bounds__(256) rope_table_kernel(const __grid_constant__ RopeFreqs p) {
    const int64_t n = (int64_t)p.n_pos * p.half;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
        double s, c;
        sincos((double)(i / p.half) * p.inv[i % p.half], &s, &c);
        reinterpret_cast<float2*>(p.out)[i] = make_float2((float)(c * p.attn), (float)(s * p.attn));
    }
}

// N contiguous elements as fp32 and back, in 16-byte (or, for runs of four
// 16-bit elements, 8-byte) accesses; N = 1 for odd rotary halves.
template <int N, typename T>
__device__ __forceinline__ void load_run(float (&x)[N], const T* p) {
    if constexpr (N == 1) {
        x[0] = to_f(p[0]);
    } else {
        constexpr int W = N * sizeof(T) >= 16 ? 16 : 8;  // bytes per access
        using V = typename std::conditional<W == 16, uint4, uint2>::type;
        constexpr int E = W / sizeof(T);
#pragma unroll
        for (int j = 0; j < N / E; j++) {
            const V v = reinterpret_cast<const V*>(p)[j];
            T e[E];
            memcpy(e, &v, W);
#pragma unroll
            for (int i = 0; i < E; i++) x[j * E + i] = to_f(e[i]);
        }
    }
}
template <int N, typename T>
__device__ __forceinline__ void store_run(T* p, const float (&x)[N]) {
    if constexpr (N == 1) {
        p[0] = from_f<T>(x[0]);
    } else {
        constexpr int W = N * sizeof(T) >= 16 ? 16 : 8;
        using V = typename std::conditional<W == 16, uint4, uint2>::type;
        constexpr int E = W / sizeof(T);
#pragma unroll
        for (int j = 0; j < N / E; j++) {
            T e[E];
#pragma unroll
            for (int i = 0; i < E; i++) e[i] = from_f<T>(x[j * E + i]);
            V v;
            memcpy(&v, e, W);
            reinterpret_cast<V*>(p)[j] = v;
        }
    }
}

// One pass over q, k and v, bound by HBM for prompts and by the latency of its one chain (position -> table row -> store)
// for a step.  Thread (x, y, z) takes CH pairs of heads y, y + blockDim.y, .. of the block's z-th token: two runs of CH
// elements half a rotary width apart, or one of 2 CH when interleaved, so every access is a full vector.  The elements
// behind rot_dim are items of 2 CH elements as well.  The inputs do not wait for the position: their loads are issued
// before it is needed.  10 100 tokens of 24 heads of 128 in bf16: 28 us, 4.5 TB/s (2 and 4 heads a thread, which read
// the table less often, 28.4 and 36.6 us); 48 tokens: 2.5 us.
template <typename T, typename C, int CH, bool INTER>
__global__ void __launch_bounds__(kRopeThreads) rope_append_kernel(const __grid_constant__ voxq_rope d) {
    const int t = blockIdx.x * blockDim.z + threadIdx.z, item = threadIdx.x;
    const int half = d.rot_dim / 2, H = d.heads, heads = H + 2 * d.kv_heads;
    const int turning = half / CH;  // items that rotate
    const bool turn = item < turning;
    const int i0 = !turn ? d.rot_dim + (item - turning) * 2 * CH : INTER ? item * 2 * CH : item * CH;
    const int i1 = turn && !INTER ? i0 + half : i0 + CH;
    pdl_wait();
    pdl_launch_dependents();
    if (t >= d.tokens) return;
    const int p = d.freqs ? __ldg(d.positions + t) : 0;
    const int64_t slot = d.kv_heads ? __ldg(d.slots + t) : -1;
    float a[CH], b[CH];
    auto fetch = [&](int h) {
        const int kh = h - H < d.kv_heads ? h - H : h - H - d.kv_heads;
        const T* src = h < H ? (const T*)d.q + t * d.q_stride + h * d.q_head_stride
                       : h - H < d.kv_heads ? (const T*)d.k + t * d.k_stride + kh * d.k_head_stride
                                            : (const T*)d.v + t * d.v_stride + kh * d.v_head_stride;
        load_run<CH>(a, src + i0);
        load_run<CH>(b, src + i1);
    };
    int h = threadIdx.y;
    fetch(h);
    float c[CH], s[CH];
    if (turn) {
        const float2* f = reinterpret_cast<const float2*>(d.freqs) + (int64_t)min(max(p, 0), d.n_pos - 1) * half + item * CH;
        if constexpr (CH == 1) {
            c[0] = __ldg(f).x;
            s[0] = __ldg(f).y;
        } else {
#pragma unroll
            for (int j = 0; j < CH; j += 2) {
                const float4 v = __ldg(reinterpret_cast<const float4*>(f + j));
                c[j] = v.x;
                s[j] = v.y;
                c[j + 1] = v.z;
                s[j + 1] = v.w;
            }
        }
    }
    const bool live = slot >= 0 && slot < (int64_t)d.pages * d.page_size;
    const uint32_t row = live ? (uint32_t)slot : 0u, page = d.page_size ? row / (uint32_t)d.page_size : 0u;
    const int64_t place = page * d.page_stride + (row - page * d.page_size) * d.row_stride;
    while (true) {
        const int kh = h - H < d.kv_heads ? h - H : h - H - d.kv_heads;
        if (turn && h - H < d.kv_heads) {
            if (INTER) {  // a holds pairs 0 .. CH/2 - 1 side by side, b the rest
#pragma unroll
                for (int j = 0; j < CH; j++) {
                    float& x0 = 2 * j < CH ? a[2 * j % CH] : b[2 * j % CH];
                    float& x1 = 2 * j + 1 < CH ? a[(2 * j + 1) % CH] : b[(2 * j + 1) % CH];
                    const float y0 = x0 * c[j] - x1 * s[j], y1 = x0 * s[j] + x1 * c[j];
                    x0 = y0;
                    x1 = y1;
                }
            } else {
#pragma unroll
                for (int j = 0; j < CH; j++) {
                    const float y0 = a[j] * c[j] - b[j] * s[j], y1 = a[j] * s[j] + b[j] * c[j];
                    a[j] = y0;
                    b[j] = y1;
                }
            }
        }
        if (h < H || live) {
            C* dst = h < H ? (C*)d.q_out + t * d.qo_stride + h * d.qo_head_stride
                           : (C*)(h - H < d.kv_heads ? d.cache_k : d.cache_v) + place + kh * d.head_stride;
            store_run<CH>(dst + i0, a);
            store_run<CH>(dst + i1, b);
        }
        h += blockDim.y;
        if (h >= heads) return;
        fetch(h);
    }
}

template <typename T, typename C, int CH>
static cudaError_t rope_launch(const voxq_rope& p, cudaStream_t st) {
    const int items = p.head_dim / (2 * CH), heads = p.heads + 2 * p.kv_heads;
    const int y = std::min(heads, std::max(1, kRopeThreads / items));
    const int z = std::min(64, std::max(1, kRopeThreads / (items * y)));  // 64: a block's limit along z
    auto kern = p.interleaved ? rope_append_kernel<T, C, CH, true> : rope_append_kernel<T, C, CH, false>;
    return launch_pdl(kern, dim3((p.tokens + z - 1) / z), dim3(items, y, z), 0, st, p);
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
    if ((uintptr_t)d->out & 7) return VOXCPM_ERR_UNSUPPORTED;  // pairs in one access
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
    if ((int64_t)d->pages * d->page_size > INT32_MAX) return VOXCPM_ERR_UNSUPPORTED;
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
    if (turn && ((uintptr_t)d->freqs & 7)) return VOXCPM_ERR_UNSUPPORTED;  // pairs in one access
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
    if (!turn) p.rot_dim = 0;
    cudaStream_t st = (cudaStream_t)stream;
    // the widest run that divides both the rotary half and the rest of the head
    const int half = p.rot_dim / 2, rest = p.head_dim - p.rot_dim;
    cudaError_t e = cudaSuccess;
    with_elem(it, [&](auto x) {
        with_elem(ct, [&](auto y) {
            using T = decltype(x);
            using C = decltype(y);
            if constexpr (std::is_same<T, float>::value || std::is_same<T, C>::value) {
                // (and vectors of the table want its rows aligned)
                const bool aligned = ((uintptr_t)p.freqs & 15) == 0;
                if (aligned && half % 8 == 0 && rest % 16 == 0) e = rope_launch<T, C, 8>(p, st);
                else if (aligned && half % 4 == 0 && rest % 8 == 0) e = rope_launch<T, C, 4>(p, st);
                else e = rope_launch<T, C, 1>(p, st);
            }
        });
    });
    VOXQ_CUDA_TRY(e);
    return VOXCPM_SUCCESS;
}
