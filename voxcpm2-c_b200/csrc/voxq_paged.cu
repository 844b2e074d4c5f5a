// voxq_paged.cu -- attention of a ragged batch's new tokens over a paged KV cache.
#include <math.h>

#include <algorithm>

#include "voxq_internal.h"
#include "voxq_paged.cuh"

namespace voxq {

// Splits of the keys.  Down to kMinSplit keys while there is less than a CTA an SM: 8 fp32 tokens on 2000 keys took 31 us with
// splits of 256, 16 with 64.  Down to kMinSplitMore while there are fewer than kSplitCtas an SM: 16 sequences of 32 fp32 tokens
// on 1000 keys took 150 us with 2 an SM, 98 with 4, 96 with 8; finer, the records cost more than they save (12 tokens on 8000
// keys, bf16 x 128: 22.5 us with 32 splits, 39 with 126).  The tcgen05 kernel, one CTA of which fills an SM, lasts as long for
// 64 keys as for 200: 4 prompts of 200 tokens took 39 us split, 21 whole.
constexpr int kMinSplit = 64, kMinSplitMore = 256, kSplitCtas = 4;
constexpr int kTcWork = 36 * 1024;  // keys x head dims of 64-row tiles per SM from which the tcgen05 kernel pays
constexpr int kMaxSplits = 128;

constexpr int kMmaThreads = 256;

// Shape of the kernel for element type T and head dims up to HD.
template <typename T, int HD>
struct PagedShape {
    static constexpr int TR = 64;                          // rows of a tile
    static constexpr int BK = is_f32<T> ? 32 : 64;         // keys of a tile
    static constexpr int ST = HD > 128 ? 2 : 3;            // cp.async stages
    static constexpr int P = HD + 16 / (int)sizeof(T);     // shared pitch: 16 bytes more than a row
    static constexpr int stage = 2 * BK * P * (int)sizeof(T);
    static constexpr int MP = HD + 4;                      // pitch of the rows' sums while the two halves are joined
    static constexpr int bytes = TR * P * (int)sizeof(T) + ST * stage;
    static_assert(bytes <= 227 * 1024 && TR * MP * 4 <= ST * stage, "shared memory");
};

// Attention of more than 16 rows a sequence on warp-level MMAs: fp32, calls with little to do, and the head dims and page
// sizes that the tcgen05 kernel does not take; and any number of rows where a tensor map cannot describe the caches.
//
// The rows of a tile are the pairs (token, query head of the kv head's group), so a key is read once for all heads that
// share it.  Two warps own each 16 rows and take half of a tile's keys each, with their own maximum and sums, joined at the
// end: a lone warp on a quarter of an SM waits for its own MMAs.  Keys and values of BK positions arrive by
// cp.async, three stages deep, each thread following the block table for its own rows of the tile (a page may end
// anywhere inside it); rows past the end are zeros in shared memory, whatever the cache holds.  One pass, base-2 softmax
// with running maximum m and sum l per row.  With few tiles the keys are split over CTAs (blockIdx.z); a row with more
// than one split leaves (m, l, sums) for paged_combine_kernel.
// 5 sequences of 21..133 fp32 tokens on 300..1500 keys, 16 query heads over 2 x 64: 40 us, 23 TFLOP/s of fp32-accurate
// products (58 with one warp a row group, all of a tile's keys and conversions for the split).  Bound by the latency of its
// MMAs and, in fp32, by splitting every operand into two TF32 parts on its way to them.
template <typename T, int HD>
__global__ void __launch_bounds__(kMmaThreads) paged_mma_kernel(const __grid_constant__ PagedArgs p) {
    using S = PagedShape<T, HD>;
    constexpr int TR = S::TR, BK = S::BK, P = S::P, ST = S::ST, NB = HD / 8, KW = BK / 2;  // keys of a warp
    extern __shared__ __align__(16) uint8_t paged_sh[];
    T* qs = reinterpret_cast<T*>(paged_sh);
    T* kv = qs + TR * P;
    const voxq_paged_attn& d = p.d;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int wm = warp & 3, wk = warp >> 2, kh = blockIdx.y, G = p.group;
    pdl_wait();
    pdl_launch_dependents();
    const int s = tile_owner<TR>(d.cu_q, d.batch, G, blockIdx.x);
    const int first = __ldg(d.cu_q + s), n = min(__ldg(d.cu_q + s + 1), d.total_q) - first;
    const int r0 = ((int)blockIdx.x - (first * G / TR + s)) * TR, rows = min(n * G - r0, TR);
    if (first < 0 || n <= 0 || r0 < 0 || rows <= 0) return;
    const int len = min(max(__ldg(d.kv_len + s), 0), d.max_kv);
    const int k_end = visible(p, len, n, (r0 + rows - 1) / G);  // the tile's last row sees most
    const int k_beg = blockIdx.z * p.split_len, k_stop = min(k_end, k_beg + p.split_len);
    if (k_beg >= k_end && blockIdx.z > 0) return;
    const int32_t* table = d.block_table + s * d.table_stride;

    constexpr int E = 16 / sizeof(T), CPR = HD / E, RP = kMmaThreads / CPR;  // vectors per row, rows per pass
    const int lc = threadIdx.x % CPR * E, lr = threadIdx.x / CPR;
    auto fetch = [&](int t0, int stage) {
        T* ks = kv + stage * 2 * BK * P + lr * P + lc;
        int64_t at[BK / RP];
#pragma unroll
        for (int j = 0; j < BK / RP; j++) {
            const int key = t0 + lr + j * RP;
            at[j] = key < k_stop && lc < d.head_dim ? cache_row(p, table, key, kh) + lc : -1;
        }
#pragma unroll
        for (int j = 0; j < BK / RP; j++) {
            const int64_t o = at[j] < 0 ? 0 : at[j];
            cp_async16_or_zero(ks + j * RP * P, (const T*)d.k + o, at[j] >= 0);
            cp_async16_or_zero(ks + (BK + j * RP) * P, (const T*)d.v + o, at[j] >= 0);
        }
    };
    for (int i = threadIdx.x; i < TR * CPR; i += kMmaThreads) {
        const int r = i / CPR, c = i % CPR * E, row = r0 + r;
        const bool ok = r < rows && c < d.head_dim;
        cp_async16_or_zero(qs + r * P + c, (const T*)d.q + (ok ? (first + row / G) * d.q_stride + (kh * G + row % G) * d.q_head_stride + c : 0), ok);
    }
#pragma unroll
    for (int j = 0; j < ST - 1; j++) {
        if (k_beg + j * BK < k_stop) fetch(k_beg + j * BK, j);
        cp_async_commit();
    }

    // this lane's rows: g and g + 8 of the warp's 16
    int vis[2], row[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
        row[e] = r0 + wm * 16 + g + 8 * e;
        vis[e] = row[e] < n * G ? min(visible(p, len, n, row[e] / G), k_stop) : 0;
    }
    float o[NB][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < NB; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
    constexpr bool QREG = !is_f32<T> && HD <= 128;  // queries stay in registers
    uint32_t qf[QREG ? HD / 16 : 1][4];

    int stage = 0;
    for (int t0 = k_beg; t0 < k_stop; t0 += BK) {
        cp_async_wait<ST - 2>();
        __syncthreads();  // the tile has landed; the stage that is refilled next is read
        {
            const int ahead = t0 + (ST - 1) * BK, to = stage == 0 ? ST - 1 : stage - 1;
            if (ahead < k_stop) fetch(ahead, to);
            cp_async_commit();
        }
        const T* ks = kv + stage * 2 * BK * P;
        const T* qw = qs + wm * 16 * P;
        stage = stage + 1 == ST ? 0 : stage + 1;
        if constexpr (QREG) {
            if (t0 == k_beg)
#pragma unroll
                for (int k = 0; k < HD / 16; k++) ldsm4(qf[k], smem_u32(qw + (lane & 15) * P + k * 16 + (lane >> 4) * 8));
        }

        const PaddedRows<T, P> kr{smem_u32(ks + wk * KW * P)}, vr{smem_u32(ks + (BK + wk * KW) * P)};
        attend_keys<T, HD, KW / 8>(p, qw, qf, kr, vr, t0 + wk * KW + 2 * t, vis, m, l, o);
    }
    cp_async_wait<0>();
#pragma unroll
    for (int e = 0; e < 2; e++) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    }

    // join the two halves of the keys
    __shared__ float2 half_ml[S::TR];
    float* half_o = reinterpret_cast<float*>(kv);
    __syncthreads();  // every stage is read
    if (wk == 1)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int r = wm * 16 + g + 8 * e;
            if (t == 0) half_ml[r] = make_float2(m[e], l[e]);
#pragma unroll
            for (int j = 0; j < NB; j++)
                *reinterpret_cast<float2*>(half_o + r * S::MP + j * 8 + 2 * t) = make_float2(o[j][2 * e], o[j][2 * e + 1]);
        }
    __syncthreads();
    if (wk == 1) return;
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const int r = wm * 16 + g + 8 * e;
        const float2 other = half_ml[r];
        const float mm = fmaxf(m[e], other.x);
        const float f0 = m[e] == -INFINITY ? 0.0f : ex2(m[e] - mm), f1 = other.x == -INFINITY ? 0.0f : ex2(other.x - mm);
        m[e] = mm;
        l[e] = l[e] * f0 + other.y * f1;
#pragma unroll
        for (int j = 0; j < NB; j++) {
            const float2 x = *reinterpret_cast<const float2*>(half_o + r * S::MP + j * 8 + 2 * t);
            o[j][2 * e] = o[j][2 * e] * f0 + x.x * f1;
            o[j][2 * e + 1] = o[j][2 * e + 1] * f0 + x.y * f1;
        }
    }
    // A row's result goes to out, or, when its keys fill more than one split, to this split's record.
    bool again[2] = {false, false}, weights[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const int r = row[e];
        if (r >= n * G) continue;
        const int tok = first + r / G, h = kh * G + r % G, seen = visible(p, len, n, r / G);
        float chk = 0.0f;
#pragma unroll
        for (int j = 0; j < NB; j++) chk = fmaf(o[j][2 * e], 0.0f, fmaf(o[j][2 * e + 1], 0.0f, chk));
        again[e] = not_finite<T>(chk, l[e]);
        weights[e] = l[e] == l[e];
        if (seen <= p.split_len) {
            if (blockIdx.z > 0) {
                again[e] = false;
                continue;
            }
            const float inv = seen > 0 ? 1.0f / l[e] : 0.0f;
            const int64_t at = tok * d.o_stride + h * d.o_head_stride;
#pragma unroll
            for (int j = 0; j < NB; j++)
                if (j * 8 < d.head_dim) store_pair<T>(p, at + j * 8 + 2 * t, o[j][2 * e] * inv, o[j][2 * e + 1] * inv);
        } else if (k_beg < seen) {
            const int64_t rec = ((int64_t)tok * d.heads + h) * p.splits + blockIdx.z;
            if (t == 0) p.ml[rec] = make_float2(m[e], l[e]);
#pragma unroll
            for (int j = 0; j < NB; j++)
                if (j * 8 < d.head_dim)
                    *reinterpret_cast<float2*>(p.acc + rec * d.head_dim + j * 8 + 2 * t) = make_float2(o[j][2 * e], o[j][2 * e + 1]);
        } else {
            again[e] = false;
        }
    }
    uint32_t rows_again = 0;  // bit 8 e + g: a lane of row g + 8 e found something; bit 16 more: its weights are not finite
#pragma unroll
    for (int e = 0; e < 2; e++)
        if (again[e]) rows_again |= (weights[e] ? 1u : 0x10001u) << (8 * e + g);
    rows_again = __reduce_or_sync(0xffffffffu, rows_again);
    if (rows_again == 0) return;
    __syncwarp();  // what this warp wrote is read
    RowsAgain<T> found(k_beg);
    for (int i = 0; i < 16; i++) {
        const int r = r0 + wm * 16 + i, seen = visible(p, len, n, r / G);
        const int64_t rec = ((int64_t)(first + r / G) * d.heads + kh * G + r % G) * p.splits + blockIdx.z;
        if (rows_again >> i & 1) found.row(p, s, first, r, kh, k_beg, min(seen, k_stop), seen <= p.split_len ? -1 : rec, !(rows_again >> (16 + i) & 1));
    }
}

// Joins a row's splits in their order: M = max m_z, out = sum_z acc_z 2^(m_z - M) / sum_z l_z 2^(m_z - M).  One CTA per
// token and head, its warps along the splits: with a thread per element that walked all of them, 50 splits took longer
// than the attention itself.  Latency bound: 4 us behind the attention, most of it the start and two dependent loads.
template <typename T>
__global__ void __launch_bounds__(kPagedThreads) paged_combine_kernel(const __grid_constant__ PagedArgs p) {
    constexpr int W = kPagedThreads / 32;
    __shared__ float weight[kMaxSplits];
    __shared__ __align__(16) float part[W][kPagedMaxHeadDim];
    __shared__ float red[2][W];
    const voxq_paged_attn& d = p.d;
    const int tok = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // (the batch's integers were complete before the attention let this kernel start)
    int s = -1;
    for (int i0 = 0; i0 < d.batch; i0 += kPagedThreads) {
        const int i = i0 + threadIdx.x;
        s += __syncthreads_count(i < d.batch && __ldg(d.cu_q + i) <= tok);
    }
    s = max(s, 0);
    const int first = __ldg(d.cu_q + s), n = min(__ldg(d.cu_q + s + 1), d.total_q) - first;
    const int len = min(max(__ldg(d.kv_len + s), 0), d.max_kv);
    const int seen = tok >= first && tok < first + n ? visible(p, len, n, tok - first) : 0;
    pdl_wait();
    pdl_launch_dependents();
    if (seen <= p.split_len) return;
    const int z = (seen + p.split_len - 1) / p.split_len;
    const int64_t rec = ((int64_t)tok * d.heads + h) * p.splits;
    static_assert(kMaxSplits <= kPagedThreads, "a thread per split");
    const float2 ml = threadIdx.x < z ? p.ml[rec + threadIdx.x] : make_float2(-INFINITY, 0.0f);
    float m = ml.x;
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) red[0][warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; w++) m = fmaxf(m, red[0][w]);
    const float f = ml.x == -INFINITY ? 0.0f : ex2(ml.x - m);
    if (threadIdx.x < z) weight[threadIdx.x] = f;
    float l = ml.y * f;
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) red[1][warp] = l;
    __syncthreads();
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < W; w++) l += red[1][w];
    // warp w: splits w, w + W, ...; a lane four elements at a time
    for (int c = lane * 4; c < d.head_dim; c += 128) {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const float* a = p.acc + rec * d.head_dim + c;
#pragma unroll 8
        for (int j = warp; j < z; j += W) {
            const float4 x = *reinterpret_cast<const float4*>(a + (int64_t)j * d.head_dim);
            const float g = weight[j];
            v.x = fmaf(x.x, g, v.x);
            v.y = fmaf(x.y, g, v.y);
            v.z = fmaf(x.z, g, v.z);
            v.w = fmaf(x.w, g, v.w);
        }
        *reinterpret_cast<float4*>(&part[warp][c]) = v;
    }
    __syncthreads();
    const int64_t at = tok * d.o_stride + h * d.o_head_stride;
    for (int c = threadIdx.x * 2; c < d.head_dim; c += 2 * kPagedThreads) {
        float x = 0.0f, y = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) {
            x += part[w][c];
            y += part[w][c + 1];
        }
        store_pair<T>(p, at + c, x / l, y / l);
    }
}

// What a call runs: rows per tile, and the keys per split.  A pure function of
// the descriptor's integers, so that the workspace is known beforehand.
struct PagedPlan {
    bool tc;        // tcgen05 kernel
    bool step;      // the kernel for at most 16 rows a sequence
    int split_len, splits;
    size_t bytes;   // workspace
};

static PagedPlan paged_plan(const voxq_paged_attn& d) {
    PagedPlan r;
    const int G = d.heads / d.kv_heads;
    r.step = (int64_t)d.max_q * G <= 16 && paged_maps_take(d);
    if (r.step) {
        r.tc = false;
        r.splits = 1;
        r.split_len = INT32_MAX;
        r.bytes = paged_step_bytes(d);
        return r;
    }
    // The tcgen05 kernel starts up more slowly and is faster by key, so it takes the calls with much to do; sooner where the
    // tiles alone come near one an SM.  us, this kernel against the MMAs, kv heads of 8 query heads x 128: a prompt of 50
    // tokens 16 : 12, of 400 33 : 29, 4 prompts of 200 20 : 29; 16 sequences of 3 tokens on 1500 keys 31 : 35, 64 of them
    // 45 : 80, 64 of 4 on 300 22 : 35.  x 64: 16 of 8 on 1500 29 : 25, of 12 31 : 33, 64 of 12 37 : 59.
    const int64_t small = paged_tiles(d, 64), sms = device_sm_count();
    r.tc = paged_tc_takes(d) && (double)small * d.max_kv * d.head_dim >= (double)kTcWork * sms / (4 * small > 3 * sms ? 3 : 1);
    const int64_t tiles = paged_tiles(d, r.tc ? paged_tc_rows(d) : 64);
    auto splits = [&](int ctas, int keys) { return std::min(ctas * sms / tiles, ((int64_t)d.max_kv + keys - 1) / keys); };
    const int64_t most = r.tc ? splits(1, kMinSplitMore) : std::max(splits(1, kMinSplit), splits(kSplitCtas, kMinSplitMore));
    const int64_t z = std::min(std::max<int64_t>(1, most), (int64_t)kMaxSplits);
    const int step = r.tc ? 128 : 64;  // whole key tiles
    r.split_len = (int)(((d.max_kv + z - 1) / z + step - 1) / step * step);
    r.splits = r.split_len ? (d.max_kv + r.split_len - 1) / r.split_len : 1;
    if (r.splits <= 1) {
        r.splits = 1;
        r.split_len = INT32_MAX;
    }
    r.bytes = r.splits > 1 ? (size_t)d.total_q * d.heads * r.splits * (8 + 4 * (size_t)d.head_dim) : 0;
    return r;
}

template <typename T, int HD>
static VoxCPMError paged_mma_launch(const PagedArgs& a, cudaStream_t st) {
    using S = PagedShape<T, HD>;
    auto kern = paged_mma_kernel<T, HD>;
    static std::atomic<uint64_t> asked{0};
    VOXQ_CUDA_TRY(allow_shared((const void*)kern, S::bytes, asked));
    const dim3 grid((int)((int64_t)a.d.total_q * a.group / S::TR) + a.d.batch, a.d.kv_heads, a.splits);
    VOXQ_CUDA_TRY(launch_pdl(kern, grid, dim3(kMmaThreads), S::bytes, st, a));
    return VOXCPM_SUCCESS;
}

template <typename T>
static VoxCPMError paged_run(const PagedArgs& a, const PagedPlan& plan, cudaStream_t st) {
    const int hd = a.d.head_dim;
    VoxCPMError e = plan.tc ? paged_tc_launch(a, st) : plan.step ? paged_step_launch(a, st) : VOXCPM_ERR_UNSUPPORTED;
    if (e == VOXCPM_ERR_UNSUPPORTED)
        e = hd <= 64 ? paged_mma_launch<T, 64>(a, st) : hd <= 128 ? paged_mma_launch<T, 128>(a, st) : paged_mma_launch<T, 256>(a, st);
    if (e != VOXCPM_SUCCESS || a.splits == 1) return e;
    VOXQ_CUDA_TRY(launch_pdl(paged_combine_kernel<T>, dim3(a.d.total_q, a.d.heads), dim3(kPagedThreads), 0, st, a));
    return VOXCPM_SUCCESS;
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
    // row and tile numbers are 32-bit, and so are the launch grid's limits
    if ((int64_t)d->total_q * d->heads + (int64_t)d->batch * d->kv_heads > INT32_MAX || d->heads > 65535 || d->max_kv > 1 << 30)
        return VOXCPM_ERR_UNSUPPORTED;
    return VOXCPM_SUCCESS;
}

static bool paged_empty(const voxq_paged_attn* d) { return d->total_q == 0 || d->heads == 0 || d->head_dim == 0; }

}  // namespace voxq

using namespace voxq;

extern "C" size_t voxq_paged_attention_workspace(const voxq_paged_attn* d) {
    return paged_check(d) != VOXCPM_SUCCESS || paged_empty(d) ? 0 : paged_plan(*d).bytes;
}

extern "C" VoxCPMError voxq_paged_attention(const voxq_paged_attn* d, void* stream) {
    const VoxCPMError e = paged_check(d);
    if (e != VOXCPM_SUCCESS || paged_empty(d)) return e;
    if (!d->q || !d->out || !d->cu_q || !d->kv_len || (d->max_kv && (!d->k || !d->v || !d->block_table))) return VOXCPM_ERR_INTERNAL;
    if (!rows16(d->q, d->q_stride, d->dtype) || !rows16(d->q, d->q_head_stride, d->dtype) ||
        !rows16(d->out, d->o_stride, d->out_dtype) || !rows16(d->out, d->o_head_stride, d->out_dtype) ||
        (d->max_kv && (!rows16(d->k, d->page_stride, d->dtype) || !rows16(d->v, d->row_stride, d->dtype) || !rows16(d->k, d->head_stride, d->dtype))))
        return VOXCPM_ERR_UNSUPPORTED;
    const PagedPlan plan = paged_plan(*d);
    if (plan.bytes) {
        if (!d->workspace) return VOXCPM_ERR_INTERNAL;
        if (d->workspace_bytes < plan.bytes) return VOXCPM_ERR_OOM;
        if ((uintptr_t)d->workspace & 255) return VOXCPM_ERR_UNSUPPORTED;
    }
    PagedArgs a{};
    a.d = *d;
    a.group = d->heads / d->kv_heads;
    a.page_shift = d->page_size > 0 && (d->page_size & (d->page_size - 1)) == 0 ? __builtin_ctz(d->page_size) : -1;
    a.err = device_error_word();
    if (!a.err) return VOXCPM_ERR_INTERNAL;
    a.split_len = plan.split_len;
    a.splits = plan.splits;
    a.scale2 = (d->scale != 0.0f ? d->scale : 1.0f / sqrtf((float)d->head_dim)) * kLog2e;
    a.acc = (float*)d->workspace;
    a.ml = (float2*)(a.acc + (size_t)d->total_q * d->heads * plan.splits * d->head_dim);
    return with_elem(d->dtype, [&](auto x) { return paged_run<decltype(x)>(a, plan, (cudaStream_t)stream); });
}
