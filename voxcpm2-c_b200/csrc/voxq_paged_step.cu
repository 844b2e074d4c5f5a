// voxq_paged_step.cu -- paged attention of at most 16 rows a sequence and kv head: the next-token step.
#include <mutex>

#include "voxq_internal.h"
#include "voxq_paged.cuh"

namespace voxq {

// Shape of the kernel: stages of 8 KB (16 KB for head dims over 128), SW for each consumer warp.
template <typename T, int HD>
struct StepShape {
    static constexpr int KT = HD > 128 ? 32 / (int)sizeof(T) : 4096 / (HD * (int)sizeof(T));  // keys of a stage
    static constexpr int BL = HD * (int)sizeof(T) / 128;     // 128-byte blocks of a row
    static constexpr int P = HD + 16 / (int)sizeof(T);       // shared pitch of the queries
    static constexpr int W = 4, SW = HD > 128 ? 1 : 3, ST = W * SW;  // consumer warps, stages of each
    static constexpr int stage = 2 * KT * HD * (int)sizeof(T);
    static constexpr int merge = W * 16 * (HD + 4) * 4;
    static constexpr int bytes = 1024 + (ST * stage > merge ? ST * stage : merge) + 16 * P * (int)sizeof(T);
    static_assert(2 * (bytes + 2048) <= 228 * 1024, "two blocks an SM");
};
constexpr int kStepThreads = 160;

// KT rows as 128-byte blocks of 128-byte-swizzled rows.
template <typename T, int KT>
struct SwizzledRows {
    uint32_t base;
    __device__ __forceinline__ uint32_t operator()(int row, int dim) const {
        const int b = dim * (int)sizeof(T);
        return base + (b / 128) * (KT * 128) + row * 128 + (((b % 128 / 16) ^ (row & 7)) << 4) + b % 16;
    }
};

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// Up to 16 rows -- pairs (token, query head of the kv head's group) -- against a split of a sequence's keys: the
// next-token step.  It reads the cache once and computes little, so it is bound by HBM, and by how early and how evenly
// the copies are issued.  A producer warp does nothing else: per tile of KT positions each of its lanes looks the page
// of one box up and issues its TMA copy; boxes past the last key are left out.  (The same stages by cp.async, from this
// warp or from all, took 150 and 65 us where this takes STEPUS: a warp has few of those in flight.)  Each of four
// consumer warps takes every fourth key tile by itself, with its own running maximum m, sum l and outputs for the 16 rows,
// so no warp waits for another until they are joined at the end.  Two blocks share an SM: one's start and end hide
// behind the other's stream.
template <typename T, int HD>
__global__ void __launch_bounds__(kStepThreads, 2) paged_step_kernel(const __grid_constant__ PagedArgs p, const __grid_constant__ PagedMaps maps) {
    using S = StepShape<T, HD>;
    constexpr int KT = S::KT, P = S::P, ST = S::ST, W = S::W, NB = HD / 8, KN = KT / 8;
    extern __shared__ uint8_t step_sh[];
    __shared__ uint64_t full[ST], empty[ST];
    const uint32_t ring = (smem_u32(step_sh) + 1023) & ~1023u;
    uint8_t* ring_p = step_sh + (ring - smem_u32(step_sh));
    T* qs = reinterpret_cast<T*>(ring_p + (ST * S::stage > S::merge ? ST * S::stage : S::merge));
    const voxq_paged_attn& d = p.d;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int kh = blockIdx.y, G = p.group;
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; i++) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, 1);
        }
        mbar_fence_init();
    }
    pdl_wait();
    pdl_launch_dependents();
    const int s = tile_owner<16>(d.cu_q, d.batch, G, blockIdx.x);  // (a block barrier: the stages' barriers are ready)
    const int first = __ldg(d.cu_q + s), n = min(__ldg(d.cu_q + s + 1), d.total_q) - first;
    const int r0 = ((int)blockIdx.x - (first * G / 16 + s)) * 16, rows = min(n * G - r0, 16);
    if (first < 0 || n <= 0 || r0 < 0 || rows <= 0) return;
    const int len = min(max(__ldg(d.kv_len + s), 0), d.max_kv);
    const int k_end = visible(p, len, n, (r0 + rows - 1) / G);
    const int k_beg = blockIdx.z * p.split_len, k_stop = min(k_end, k_beg + p.split_len);
    if (k_beg >= k_end && blockIdx.z > 0) return;
    const int tiles = k_stop > k_beg ? (k_stop - k_beg + KT - 1) / KT : 0;

    // Stage of key tile c: a warp has stages of its own, because a barrier's phases can only be told apart by who has
    // seen each of them, and copies may land out of order.
    auto slot_of = [](int c) { return c % W * S::SW + c / W % S::SW; };
    if (warp == W) {
        const int32_t* table = d.block_table + s * d.table_stride;
        // A tile has `boxes` boxes: KT / R for each 128-byte block of its keys and values.  The lanes take as many tiles
        // at a time as they have boxes for, and look the next ones' pages up before they wait for these ones' stages.
        const int R = maps.box_rows, per = KT / R, boxes = 2 * per * S::BL, at_once = 32 / boxes;
        const int mine = lane / boxes, box = lane % boxes, block = box / per % S::BL, row = box % per * R;
        const bool value = box >= per * S::BL;
        bool ok = true;
        int c = 0, page = 0, off = 0;
        auto look_up = [&](int tile) {
            const int key = k_beg + tile * KT + row;
            if (key >= k_stop) return;
            const int e = p.page_shift >= 0 ? key >> p.page_shift : (int)((uint32_t)key / (uint32_t)d.page_size);
            page = __ldg(table + e);
            off = key - e * d.page_size;
        };
        look_up(mine);
        while (c < tiles && ok) {
            const int now_page = (uint32_t)page < (uint32_t)d.pages ? page : 0, now_off = off, first_c = c;
            look_up(c + at_once + mine);
            for (int u = 0; u < at_once && c < tiles; u++, c++) {
                const int slot = slot_of(c);
                if (c >= ST) ok = __all_sync(0xffffffffu, mbar_wait_bounded(empty + slot, (c / ST - 1) & 1, VOXQ_DEVERR_WAIT_EMPTY, p.err));
                if (!ok) break;
                const bool live = first_c + mine == c && k_beg + c * KT + row < k_stop;
                const int count = __popc(__ballot_sync(0xffffffffu, live));
                if (lane == 0) mbar_arrive_expect_tx(full + slot, count * R * 128);
                __syncwarp();
                if (live)
                    tma_page(ring + slot * S::stage + (value ? S::stage / 2 : 0) + block * (KT * 128) + row * 128, maps, value ? &maps.v : &maps.k,
                             block * (128 / (int)sizeof(T)), now_off, kh, now_page, full + slot);
            }
        }
        if (!ok)  // nothing of this block may still be writing its shared memory when it ends
            for (int i = max(0, c - ST); i < c; i++) mbar_wait_bounded(full + slot_of(i), (i / ST) & 1, VOXQ_DEVERR_NONE, p.err);
        return;
    }

    // queries, and this lane's rows: g and g + 8
    constexpr int QC = HD * (int)sizeof(T) / 16;
    for (int i = threadIdx.x; i < 16 * QC; i += 128) {
        const int r = i / QC, c = i % QC * (16 / (int)sizeof(T)), row = r0 + r;
        const bool live = r < rows && c < d.head_dim;
        cp_async16_or_zero(qs + r * P + c, (const T*)d.q + (live ? (first + row / G) * d.q_stride + (kh * G + row % G) * d.q_head_stride + c : 0), live);
    }
    cp_async_commit();
    cp_async_wait<0>();
    consumers_sync();
    constexpr bool QREG = !is_f32<T> && HD <= 128;
    uint32_t qf[QREG ? HD / 16 : 1][4];
    if constexpr (QREG) {
#pragma unroll
        for (int k = 0; k < HD / 16; k++) ldsm4(qf[k], smem_u32(qs + (lane & 15) * P + k * 16 + (lane >> 4) * 8));
    }
    int vis[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const int row = r0 + g + 8 * e;
        vis[e] = row < n * G ? min(visible(p, len, n, row / G), k_stop) : 0;
    }
    float o[NB][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < NB; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
    for (int c = warp; c < tiles; c += W) {
        const int slot = slot_of(c);
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(full + slot, (c / ST) & 1, VOXQ_DEVERR_WAIT_FULL, p.err))) break;
        const SwizzledRows<T, KT> ks{ring + slot * S::stage}, vs{ring + slot * S::stage + S::stage / 2};
        const int valid = k_stop - (k_beg + c * KT);
        if (valid < KT) {
            // values past the last key may be anything, and 0 * NaN is NaN
            for (int i = lane; i < (KT - valid) * S::BL * 8; i += 32)
                sts128(vs.base + i / ((KT - valid) * 8) * (KT * 128) + valid * 128 + i % ((KT - valid) * 8) * 16, make_uint4(0, 0, 0, 0));
            __syncwarp();
        }
        attend_keys<T, HD, KN>(p, qs, qf, ks, vs, k_beg + c * KT + 2 * t, vis, m, l, o);
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + slot);
    }
#pragma unroll
    for (int e = 0; e < 2; e++) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    }
    consumers_sync();  // every stage is read
    // join the warps' shares of the keys: 8 threads a row
    constexpr int MP = HD + 4;
    __shared__ float2 wml[W][16];
    float* mo = reinterpret_cast<float*>(ring_p);
#pragma unroll
    for (int e = 0; e < 2; e++) {
        if (t == 0) wml[warp][g + 8 * e] = make_float2(m[e], l[e]);
#pragma unroll
        for (int j = 0; j < NB; j++)
            *reinterpret_cast<float2*>(mo + (warp * 16 + g + 8 * e) * MP + j * 8 + 2 * t) = make_float2(o[j][2 * e], o[j][2 * e + 1]);
    }
    consumers_sync();
    const int r = threadIdx.x >> 3, rr = r0 + r;
    if (r >= rows) return;
    float mm = -INFINITY, ll = 0.0f, f[W];
#pragma unroll
    for (int w = 0; w < W; w++) mm = fmaxf(mm, wml[w][r].x);
#pragma unroll
    for (int w = 0; w < W; w++) {
        f[w] = wml[w][r].x == -INFINITY ? 0.0f : ex2(wml[w][r].x - mm);
        ll = fmaf(wml[w][r].y, f[w], ll);
    }
    // to out, or, when the row's keys fill more than one split, to this split's record
    const int seen = visible(p, len, n, rr / G), tok = first + rr / G, h = kh * G + rr % G;
    const bool all = seen <= p.split_len;
    if (all ? blockIdx.z > 0 : k_beg >= seen) return;
    const float inv = !all ? 1.0f : seen > 0 ? 1.0f / ll : 0.0f;
    const int64_t rec = ((int64_t)tok * d.heads + h) * p.splits + blockIdx.z, at = tok * d.o_stride + h * d.o_head_stride;
    if (!all && (threadIdx.x & 7) == 0) p.ml[rec] = make_float2(mm, ll);
    for (int c = (threadIdx.x & 7) * 2; c < d.head_dim; c += 16) {
        float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float2 x = *reinterpret_cast<const float2*>(mo + (w * 16 + r) * MP + c);
            v.x = fmaf(x.x, f[w], v.x);
            v.y = fmaf(x.y, f[w], v.y);
        }
        if (all) store_pair<T>(p, at + c, v.x * inv, v.y * inv);
        else *reinterpret_cast<float2*>(p.acc + rec * d.head_dim + c) = v;
    }
}

template <typename T, int HD>
static VoxCPMError step_launch(const PagedArgs& a, cudaStream_t st) {
    using S = StepShape<T, HD>;
    auto kern = paged_step_kernel<T, HD>;
    static std::once_flag once;
    static cudaError_t attr = cudaSuccess;
    std::call_once(once, [&] { attr = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::bytes); });
    VOXQ_CUDA_TRY(attr);
    PagedMaps m;
    const VoxCPMError e = paged_maps(a.d, S::KT, &m);
    if (e != VOXCPM_SUCCESS) return e;
    const dim3 grid((int)((int64_t)a.d.total_q * a.group / 16) + a.d.batch, a.d.kv_heads, a.splits);
    VOXQ_CUDA_TRY(launch_pdl(kern, grid, dim3(kStepThreads), S::bytes, st, a, m));
    return VOXCPM_SUCCESS;
}

VoxCPMError paged_step_launch(const PagedArgs& a, cudaStream_t st) {
    return with_elem(a.d.dtype, [&](auto x) {
        using T = decltype(x);
        const int hd = a.d.head_dim;
        return hd <= 64 ? step_launch<T, 64>(a, st) : hd <= 128 ? step_launch<T, 128>(a, st) : step_launch<T, 256>(a, st);
    });
}

}  // namespace voxq
