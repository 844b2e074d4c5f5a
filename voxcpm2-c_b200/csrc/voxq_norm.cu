// voxq_norm.cu -- the norms around a block, its gate and its residual scale in
// one pass over the rows.
#include "voxq_batch.cuh"
#include "voxq_internal.h"

namespace voxq {

constexpr int kNormMaxD = 16384;

// V contiguous elements in one access: 16 bytes, or two elements or one where a
// row or its width is not aligned to more.
template <int BYTES>
struct VecAccess {
    using type = typename std::conditional<BYTES == 16, uint4, typename std::conditional<BYTES == 8, uint2, typename std::conditional<BYTES == 4, uint32_t, uint16_t>::type>::type>::type;
};
template <typename T, int V>
struct Vec {
    T e[V];
};
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T* p) {
    Vec<T, V> r;
    using A = typename VecAccess<V * sizeof(T)>::type;
    const A v = *reinterpret_cast<const A*>(p);
    memcpy(&r, &v, sizeof(A));
    return r;
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, V>& r) {
    using A = typename VecAccess<V * sizeof(T)>::type;
    A v;
    memcpy(&v, &r, sizeof(A));
    *reinterpret_cast<A*>(p) = v;
}

// The norm weights go through the read-only path, so that their loads may be
// issued ahead of the stores of h, which the compiler cannot tell apart.
template <int V>
__device__ __forceinline__ void load_weights(float (&w)[V], const float* p) {
    if constexpr (V == 1) {
        w[0] = __ldg(p);
    } else if constexpr (V == 2) {
        const float2 v = __ldg(reinterpret_cast<const float2*>(p));
        w[0] = v.x;
        w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < V / 4; i++) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(p) + i);
            w[4 * i] = v.x;
            w[4 * i + 1] = v.y;
            w[4 * i + 2] = v.z;
            w[4 * i + 3] = v.w;
        }
    }
}

// Sum over the WR warps of a row, the same value in every thread.
template <int WR>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (WR > 1) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < WR; w++) v += red[w];
    }
    return v;
}

// h = x + alpha g z and n = RMSNorm(h) w_pre, z = y or RMSNorm(y) w_post.
// 2 reads and 2 writes per element and a few flops: bound by HBM for many
// rows, by the latency of one load and two reductions for a few.  WR warps
// hold a whole row in registers, PER vectors of V elements a thread, so the
// second norm needs no second read; all of a row's loads are issued before the
// first reduction.  h stays fp32 from its sum to the norm.  8191 bf16 rows of
// 1024, gated, with both norms: 18.4 us, 3.6 TB/s with inputs partly in L2; 2
// fp32 rows of 2048: 2.3 us.
template <typename T, int V, int WR, int PER>
__global__ void __launch_bounds__(WR == 1 ? 128 : 32 * WR) norm_residual_kernel(const __grid_constant__ voxq_norm d) {
    __shared__ float red[2][WR];
    const int m = WR == 1 ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (WR == 1 && m >= d.rows) return;
    const int tid = WR == 1 ? threadIdx.x & 31 : threadIdx.x;
    const T* y = (const T*)d.y + m * d.ldy;
    const T* x = (const T*)d.x + m * d.ldx;
    pdl_wait();
    pdl_launch_dependents();
    Vec<T, V> yv[PER], xv[PER], gv[PER];
    const T* g = nullptr;
    if (d.gate) g = (const T*)d.gate + (d.gate_index ? min(max(__ldg(d.gate_index + m), 0), d.gate_rows - 1) : d.gate_rows == 1 ? 0 : m) * d.ldg;
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const int i = (tid + j * 32 * WR) * V;
        if (i < d.D) {
            yv[j] = load_vec<T, V>(y + i);
            xv[j] = load_vec<T, V>(x + i);
        }
    }
    if (g)
#pragma unroll
        for (int j = 0; j < PER; j++)
            if ((tid + j * 32 * WR) * V < d.D) gv[j] = load_vec<T, V>(g + (tid + j * 32 * WR) * V);
    float inv = 1.0f;
    if (d.w_post) {
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < PER; j++)
            if ((tid + j * 32 * WR) * V < d.D)
#pragma unroll
                for (int e = 0; e < V; e++) s = fmaf(to_f(yv[j].e[e]), to_f(yv[j].e[e]), s);
        inv = rsqrtf(row_sum<WR>(s, red[0]) / d.D + d.eps);
    }
    float h[PER][V], s = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const int i = (tid + j * 32 * WR) * V;
        if (i >= d.D) continue;
        float w[V];
        if (d.w_post) load_weights<V>(w, d.w_post + i);
#pragma unroll
        for (int e = 0; e < V; e++) {
            float z = to_f(yv[j].e[e]);
            if (d.w_post) z = z * inv * w[e];
            if (g) z *= to_f(gv[j].e[e]);
            h[j][e] = fmaf(d.alpha, z, to_f(xv[j].e[e]));
            s = fmaf(h[j][e], h[j][e], s);
        }
    }
    if (d.h_out)
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int i = (tid + j * 32 * WR) * V;
            if (i >= d.D) continue;
            Vec<T, V> hv;
#pragma unroll
            for (int e = 0; e < V; e++) hv.e[e] = from_f<T>(h[j][e]);
            store_vec<T, V>((T*)d.h_out + m * d.ldh + i, hv);
        }
    if (!d.n_out) return;
    inv = rsqrtf(row_sum<WR>(s, red[1]) / d.D + d.eps);
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const int i = (tid + j * 32 * WR) * V;
        if (i >= d.D) continue;
        float w[V];
        load_weights<V>(w, d.w_pre + i);
        Vec<T, V> nv;
#pragma unroll
        for (int e = 0; e < V; e++) nv.e[e] = from_f<T>(h[j][e] * inv * w[e]);
        store_vec<T, V>((T*)d.n_out + m * d.ldn + i, nv);
    }
}

template <typename T, int V, int WR, int PER>
static cudaError_t norm_launch(const voxq_norm& d, cudaStream_t st) {
    const int blocks = WR == 1 ? (d.rows + 3) / 4 : d.rows;
    return launch_pdl(norm_residual_kernel<T, V, WR, PER>, dim3(blocks), dim3(WR == 1 ? 128 : 32 * WR), 0, st, d);
}

// Widths and alignments that are not 16-byte: two elements or one an access, so several a thread, and room for no more than
// the row needs.  (3289 gated rows of 2162 in fp16, both norms: 32 us; 160 with one element an access and room for 16 384.)
template <typename T, int V>
static cudaError_t norm_narrow(const voxq_norm& d, cudaStream_t st) {
    const int nv = (d.D + V - 1) / V;
    if (nv <= 256) return norm_launch<T, V, 4, 2>(d, st);
    if (nv <= 512) return norm_launch<T, V, 4, 4>(d, st);
    if (nv <= 1024) return norm_launch<T, V, 8, 4>(d, st);
    if (nv <= 2048) return norm_launch<T, V, 16, 4>(d, st);
    if (nv <= 4096) return norm_launch<T, V, 16, 8>(d, st);
    return norm_launch<T, V, 16, kNormMaxD / 512 / V>(d, st);
}

// One vector a thread as far as 512 threads go: the shortest chains and the most rows in flight.  (8191 rows of 1024 in
// bf16, gated, with both norms: 24.6 us from cold caches with 4 warps of one vector a row, 26.6 with one warp of four,
// 28.7 with 4 warps and room for two.)
template <typename T>
static cudaError_t norm_dispatch(const voxq_norm& d, int width, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    if (width < V) return width == 2 ? norm_narrow<T, 2>(d, st) : norm_narrow<T, 1>(d, st);
    const int nv = d.D / V;
    if (nv <= 32) return norm_launch<T, V, 1, 1>(d, st);
    if (nv <= 64) return norm_launch<T, V, 2, 1>(d, st);
    if (nv <= 128) return norm_launch<T, V, 4, 1>(d, st);
    if (nv <= 256) return norm_launch<T, V, 8, 1>(d, st);
    if (nv <= 512) return norm_launch<T, V, 16, 1>(d, st);
    if (nv <= 1024) return norm_launch<T, V, 16, 2>(d, st);
    return norm_launch<T, V, 16, 8>(d, st);
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
    const int dt = d->dtype;
    // elements per access: the most that divide the width and to which all rows are aligned
    auto fits = [&](int v) {
        const int64_t by = (int64_t)v * elem_bytes(dt);
        auto rows = [&](const void* p, int64_t ld) { return !p || ((uintptr_t)p % by == 0 && ld * elem_bytes(dt) % by == 0); };
        auto weights = [&](const float* w) { return (uintptr_t)w % (v < 4 ? 4 * v : 16) == 0; };
        return d->D % v == 0 && rows(d->y, d->ldy) && rows(d->x, d->ldx) && rows(d->gate, d->ldg) && rows(d->h_out, d->ldh) &&
               rows(d->n_out, d->ldn) && weights(d->w_post) && weights(d->w_pre);
    };
    if (!fits(1)) return VOXCPM_ERR_UNSUPPORTED;  // elements themselves out of line
    const int wide = 16 / elem_bytes(dt), width = fits(wide) ? wide : fits(2) ? 2 : 1;
    VOXQ_CUDA_TRY(with_elem(dt, [&](auto x) { return norm_dispatch<decltype(x)>(*d, width, (cudaStream_t)stream); }));
    return VOXCPM_SUCCESS;
}
