// voxq_paged_step.cu -- paged attention of at most 16 rows a sequence and kv head: the next-token step.
#include <algorithm>
#include <mutex>

#include "voxq_internal.h"
#include "voxq_paged.cuh"

namespace voxq {

// Shape of the kernel: stages of 16 KB, SW for each consumer warp.
template <typename T, int HD>
struct StepShape {
    static constexpr int KT = 8192 / (HD * (int)sizeof(T));  // keys of a tile
    static constexpr int BL = HD * (int)sizeof(T) / 128;     // 128-byte blocks of a row
    static constexpr int P = HD + 16 / (int)sizeof(T);       // shared pitch of the queries
    static constexpr int W = 4, SW = 1, ST = W * SW;         // consumer warps, stages of each
    static constexpr int stage = 2 * KT * HD * (int)sizeof(T);
    static constexpr int MP = HD + 4;                        // pitch of the warps' outputs while they are joined
    static constexpr int bytes = 1024 + ST * stage + W * 16 * MP * 4 + 16 * P * (int)sizeof(T);
    static constexpr int per_sm = HD > 128 ? 1 : 2;          // blocks that share an SM
    static_assert(per_sm * (bytes + 2048) <= 228 * 1024, "shared memory");
};
constexpr int kStepThreads = 160;
constexpr int kWholeTiles = 16;   // a row's keys stay in one block up to here
constexpr int kMinTiles = 8;      // tiles that are worth a block of their own
constexpr int kStepPieces = 512;  // most blocks, and so most pieces of one row

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

// The work of a call as one line of key tiles: sequence by sequence, within it row tile by row tile (16 rows), kv head by
// kv head, tile by tile.  The blocks take equal stretches of it, whatever the lengths are; a stretch that ends inside a
// row's keys leaves a piece, and the pieces are joined afterwards.  Where all rows have few keys (step_whole), the items
// themselves stand on the line, one step each, and nothing is cut.
struct StepSeq {
    int first, n, len;  // first row in the batch, rows (tokens), positions
    int tiles;          // key tiles of each of its items (row tile, kv head); 1 for no keys
    int line;           // steps of an item on the line
    int64_t units;      // steps of all its items
};
template <int KT>
__device__ __forceinline__ StepSeq step_seq(const PagedArgs& p, int s) {
    StepSeq q;
    q.first = __ldg(p.d.cu_q + s);
    q.n = q.first < 0 ? 0 : max(min(__ldg(p.d.cu_q + s + 1), p.d.total_q) - q.first, 0);
    q.len = min(max(__ldg(p.d.kv_len + s), 0), p.d.max_kv);
    q.tiles = max((q.len + KT - 1) / KT, 1);
    q.line = p.step_whole ? 1 : q.tiles;
    q.units = (int64_t)((q.n * p.group + 15) / 16) * p.d.kv_heads * q.line;
    return q;
}
// Units before each thread's sequences tid * per .. and in total, over the block's THREADS threads.
template <int THREADS, int KT>
__device__ __forceinline__ int64_t step_scan(const PagedArgs& p, int per, int64_t& before) {
    __shared__ int64_t sums[THREADS / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int64_t mine = 0;
    for (int i = 0; i < per; i++) {
        const int s = threadIdx.x * per + i;
        if (s < p.d.batch) mine += step_seq<KT>(p, s).units;
    }
    int64_t run = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int64_t v = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += v;
    }
    if (lane == 31) sums[warp] = run;
    __syncthreads();
    int64_t total = 0;
    before = run - mine;
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) {
        if (w < warp) before += sums[w];
        total += sums[w];
    }
    return total;
}
__device__ __forceinline__ int step_blocks(const PagedArgs& p, int64_t total) {
    return (int)max((int64_t)1, min((int64_t)p.step_blocks, p.step_whole ? total : total / kMinTiles));
}

// Up to 16 rows -- pairs (token, query head of the kv head's group) -- against a sequence's keys: the next-token step.
// It reads the cache once and computes little, so it is bound by HBM, by how early and how evenly the copies are issued
// and by an even share for every block.  A producer warp does nothing but copy: its lanes look the pages of several
// tiles' boxes up at once and issue their TMA copies, on into the next stretch of keys while the last is still at work;
// boxes past the last key are left out.  (The same stages by cp.async, from this warp or from all, took 150 and 65 us
// where this takes STEPUS for 64 sequences: a warp has few of those in flight.)  Each of four consumer warps takes every
// fourth tile by itself, with its own running maximum m, sum l and outputs for the 16 rows, so no warp waits for another
// until they are joined.  Two blocks share an SM: one's start and joins hide behind the other's stream.
template <typename T, int HD>
__global__ void __launch_bounds__(kStepThreads, StepShape<T, HD>::per_sm) paged_step_kernel(const __grid_constant__ PagedArgs p, const __grid_constant__ PagedMaps maps) {
    using S = StepShape<T, HD>;
    constexpr int KT = S::KT, P = S::P, ST = S::ST, W = S::W, NB = HD / 8, KN = KT / 8, MP = S::MP;
    extern __shared__ uint8_t step_sh[];
    __shared__ uint64_t full[ST], empty[ST];
    __shared__ float2 wml[W][16];
    __shared__ int64_t start_base;
    __shared__ int start_seq;
    const uint32_t ring = (smem_u32(step_sh) + 1023) & ~1023u;
    float* mo = reinterpret_cast<float*>(step_sh + (ring - smem_u32(step_sh)) + ST * S::stage);
    T* qs = reinterpret_cast<T*>(mo + W * 16 * MP);
    const voxq_paged_attn& d = p.d;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, G = p.group;
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; i++) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, 1);
        }
        mbar_fence_init();
    }
    pdl_wait();
    pdl_launch_dependents();

    // this block's stretch [pos, end), and the sequence that it begins in
    const int per = (d.batch + kStepThreads - 1) / kStepThreads;
    int64_t before;
    const int64_t total = step_scan<kStepThreads, KT>(p, per, before);
    const int blocks = step_blocks(p, total);
    if ((int)blockIdx.x >= blocks || total == 0) return;
    int64_t pos = blockIdx.x * total / blocks;
    const int64_t end = (blockIdx.x + 1) * total / blocks;
    for (int i = 0; i < per; i++) {
        const int s = threadIdx.x * per + i;
        if (s >= d.batch) break;
        const int64_t units = step_seq<KT>(p, s).units;
        if (pos >= before && pos < before + units) {
            start_seq = s;
            start_base = before;
        }
        before += units;
    }
    __syncthreads();
    int s = start_seq;
    int64_t base = start_base;

    // Stage of the block's c-th tile: a warp has stages of its own, because a barrier's phases can only be told apart by
    // who has seen each of them, and copies may land out of order.
    auto slot_of = [](int c) { return c % W * S::SW + c / W % S::SW; };
    // The part of the stretch at pos that lies in one item: tiles a .. b - 1 of row tile rt and kv head kh.
    StepSeq q = step_seq<KT>(p, s);
    int a, b, rt, kh;
    auto part = [&] {
        while (pos >= base + q.units) {
            base += q.units;
            q = step_seq<KT>(p, ++s);
        }
        const int64_t in = pos - base;
        const int item = (int)(in / q.line);
        a = (int)(in - (int64_t)item * q.line);
        b = p.step_whole ? q.tiles : (int)min((int64_t)q.tiles, a + (end - pos));
        kh = item % d.kv_heads;
        rt = item / d.kv_heads;
    };
    auto past = [&] { return p.step_whole ? 1 : b - a; };
    int c = 0;  // tiles before this part

    if (warp == W) {
        // A tile has `boxes` boxes: KT / R for each 128-byte block of its keys and values.  The lanes take as many tiles
        // at a time as they have boxes for, and look the next ones' pages up before they wait for these ones' stages.
        const int R = maps.box_rows, rows_per = KT / R, boxes = 2 * rows_per * S::BL, at_once = 32 / boxes;
        const int mine = lane / boxes, box = lane % boxes, block = box / rows_per % S::BL, row = box % rows_per * R;
        const bool value = box >= rows_per * S::BL;
        bool ok = true;
        for (; pos < end && ok; pos += past()) {
            part();
            const int32_t* table = d.block_table + s * d.table_stride;
            const int k_stop = min(b * KT, q.len);
            int page = 0, off = 0;
            auto look_up = [&](int tile) {
                const int key = tile * KT + row;
                if (key >= k_stop) return;
                const int e = p.page_shift >= 0 ? key >> p.page_shift : (int)((uint32_t)key / (uint32_t)d.page_size);
                page = __ldg(table + e);
                off = key - e * d.page_size;
            };
            look_up(a + mine);
            for (int i = a; i < b && ok;) {
                const int now_page = (uint32_t)page < (uint32_t)d.pages ? page : 0, now_off = off, from = i;
                look_up(i + at_once + mine);
                for (int u = 0; u < at_once && i < b; u++, i++, c++) {
                    const int slot = slot_of(c);
                    if (c >= ST) ok = __all_sync(0xffffffffu, mbar_wait_bounded(empty + slot, (c / ST - 1) & 1, VOXQ_DEVERR_WAIT_EMPTY, p.err));
                    if (!ok) break;
                    const bool live = from + mine == i && i * KT + row < k_stop;
                    const int count = __popc(__ballot_sync(0xffffffffu, live));
                    if (lane == 0) mbar_arrive_expect_tx(full + slot, count * R * 128);
                    __syncwarp();
                    if (live)
                        tma_page(ring + slot * S::stage + (value ? S::stage / 2 : 0) + block * (KT * 128) + row * 128, maps,
                                 value ? &maps.v : &maps.k, block * (128 / (int)sizeof(T)), now_off, kh, now_page, full + slot);
                }
            }
        }
        if (!ok)  // nothing of this block may still be writing its shared memory when it ends
            for (int i = max(0, c - ST); i < c; i++) mbar_wait_bounded(full + slot_of(i), (i / ST) & 1, VOXQ_DEVERR_NONE, p.err);
        return;
    }

    constexpr int QC = HD * (int)sizeof(T) / 16;
    constexpr bool QREG = !is_f32<T> && HD <= 128;
    bool ok = true;
    for (bool again = false; pos < end; pos += past(), again = true) {
        part();
        const int r0 = rt * 16, rows = min(q.n * G - r0, 16), k_stop = min(b * KT, q.len);
        // queries, and this lane's rows: g and g + 8
        for (int i = threadIdx.x; i < 16 * QC; i += 128) {
            const int r = i / QC, x = i % QC * (16 / (int)sizeof(T)), row = r0 + r;
            const bool live = r < rows && x < d.head_dim;
            cp_async16_or_zero(qs + r * P + x, (const T*)d.q + (live ? (q.first + row / G) * d.q_stride + (kh * G + row % G) * d.q_head_stride + x : 0), live);
        }
        cp_async_commit();
        cp_async_wait<0>();
        consumers_sync();
        uint32_t qf[QREG ? HD / 16 : 1][4];
        if constexpr (QREG) {
#pragma unroll
            for (int k = 0; k < HD / 16; k++) ldsm4(qf[k], smem_u32(qs + (lane & 15) * P + k * 16 + (lane >> 4) * 8));
        }
        int vis[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int row = r0 + g + 8 * e;
            vis[e] = row < q.n * G ? min(visible(p, q.len, q.n, row / G), k_stop) : 0;
        }
        float o[NB][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < NB; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
        // (without keys there is one tile with nothing in it)
        for (int i = a + ((warp - c) & (W - 1)); i < b && ok; i += W) {
            const int x = c + i - a, slot = slot_of(x);
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(full + slot, (x / ST) & 1, VOXQ_DEVERR_WAIT_FULL, p.err));
            if (!ok) break;
            const SwizzledRows<T, KT> ks{ring + slot * S::stage}, vs{ring + slot * S::stage + S::stage / 2};
            const int valid = max(k_stop - i * KT, 0);
            if (valid < KT) {
                // values past the last key may be anything, and 0 * NaN is NaN
                for (int j = lane; j < (KT - valid) * S::BL * 8; j += 32)
                    sts128(vs.base + j / ((KT - valid) * 8) * (KT * 128) + valid * 128 + j % ((KT - valid) * 8) * 16, make_uint4(0, 0, 0, 0));
                // written before the copy of a later tile into this stage
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
            attend_keys<T, HD, KN>(p, qs, qf, ks, vs, i * KT + 2 * t, vis, m, l, o);
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + slot);
        }
        c += b - a;
        // join the warps' shares of the keys
#pragma unroll
        for (int e = 0; e < 2; e++) {
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
            if (t == 0) wml[warp][g + 8 * e] = make_float2(m[e], l[e]);
#pragma unroll
            for (int j = 0; j < NB; j++)
                *reinterpret_cast<float2*>(mo + (warp * 16 + g + 8 * e) * MP + j * 8 + 2 * t) = make_float2(o[j][2 * e], o[j][2 * e + 1]);
        }
        consumers_sync();
        const int r = threadIdx.x >> 3, row = r0 + r;  // 8 threads a row
        if (r < rows && ok) {
            float mm = -INFINITY, ll = 0.0f, f[W];
#pragma unroll
            for (int w = 0; w < W; w++) mm = fmaxf(mm, wml[w][r].x);
#pragma unroll
            for (int w = 0; w < W; w++) {
                f[w] = wml[w][r].x == -INFINITY ? 0.0f : ex2(wml[w][r].x - mm);
                ll = fmaf(wml[w][r].y, f[w], ll);
            }
            // all of the row's keys: to out; else the block's first piece (0) or its last (1)
            const bool all = a == 0 && b == q.tiles;
            const float inv = !all ? 1.0f : visible(p, q.len, q.n, row / G) > 0 ? 1.0f / ll : 0.0f;
            const int64_t rec = (blockIdx.x * 2 + (again ? 1 : 0)) * 16 + r;
            const int64_t at = (q.first + row / G) * d.o_stride + (kh * G + row % G) * d.o_head_stride;
            if (!all && (threadIdx.x & 7) == 0) p.ml[rec] = make_float2(mm, ll);
            for (int x = (threadIdx.x & 7) * 2; x < d.head_dim; x += 16) {
                float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < W; w++) {
                    const float2 y = *reinterpret_cast<const float2*>(mo + (w * 16 + r) * MP + x);
                    v.x = fmaf(y.x, f[w], v.x);
                    v.y = fmaf(y.y, f[w], v.y);
                }
                if (all) store_pair<T>(p, at + x, v.x * inv, v.y * inv);
                else *reinterpret_cast<float2*>(p.acc + rec * d.head_dim + x) = v;
            }
        }
        consumers_sync();  // the joined outputs and the queries are read
    }
}

// Joins the pieces of a row that several blocks worked on, in their order: M = max m, out = sum acc 2^(m - M) / sum l 2^(m - M).
// One CTA per token and query head, its warps along the pieces.
template <typename T, int KT>
__global__ void __launch_bounds__(kPagedThreads) step_combine_kernel(const __grid_constant__ PagedArgs p) {
    constexpr int W = kPagedThreads / 32, PER = kStepPieces / kPagedThreads;
    __shared__ float weight[kStepPieces];
    __shared__ __align__(16) float part[W][kPagedMaxHeadDim];
    __shared__ float red[2][W];
    __shared__ int64_t seq_base;
    const voxq_paged_attn& d = p.d;
    const int tok = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = p.group;
    pdl_wait();
    pdl_launch_dependents();
    const int per = (d.batch + kPagedThreads - 1) / kPagedThreads;
    int64_t before;
    const int64_t total = step_scan<kPagedThreads, KT>(p, per, before);
    int s = -1;
    for (int i0 = 0; i0 < d.batch; i0 += kPagedThreads) {
        const int i = i0 + threadIdx.x;
        s += __syncthreads_count(i < d.batch && __ldg(d.cu_q + i) <= tok);
    }
    s = max(s, 0);
    if (s / per == (int)threadIdx.x) {
        for (int i = threadIdx.x * per; i < s; i++) before += step_seq<KT>(p, i).units;
        seq_base = before;
    }
    __syncthreads();
    const StepSeq q = step_seq<KT>(p, s);
    if (tok < q.first || tok >= q.first + q.n) return;
    // the row's tiles, and the blocks a .. b that worked on them: block x has [x total / blocks, (x + 1) total / blocks)
    const int blocks = step_blocks(p, total), row = (tok - q.first) * G + h % G;
    const int64_t at0 = seq_base + ((int64_t)(row / 16) * d.kv_heads + h / G) * q.tiles;
    auto owner = [&](int64_t x) { return (int)(((x + 1) * blocks - 1) / total); };
    const int a = owner(at0), b = owner(at0 + q.tiles - 1), z = b - a + 1;
    if (z == 1) return;
    const int later = a * total / blocks < at0 ? 1 : 0;  // the first of them came to this row after another
    auto record = [&](int j) { return (int64_t)((a + j) * 2 + (j == 0 ? later : 0)) * 16 + row % 16; };
    float2 ml[PER];
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int j = threadIdx.x + i * kPagedThreads;
        ml[i] = j < z ? p.ml[record(j)] : make_float2(-INFINITY, 0.0f);
        m = fmaxf(m, ml[i].x);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) red[0][warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; w++) m = fmaxf(m, red[0][w]);
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int j = threadIdx.x + i * kPagedThreads;
        const float f = ml[i].x == -INFINITY ? 0.0f : ex2(ml[i].x - m);
        if (j < z) weight[j] = f;
        l = fmaf(ml[i].y, f, l);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) red[1][warp] = l;
    __syncthreads();
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < W; w++) l += red[1][w];
    for (int c = lane * 4; c < d.head_dim; c += 128) {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
        for (int j = warp; j < z; j += W) {
            const float4 x = *reinterpret_cast<const float4*>(p.acc + record(j) * d.head_dim + c);
            const float f = weight[j];
            v.x = fmaf(x.x, f, v.x);
            v.y = fmaf(x.y, f, v.y);
            v.z = fmaf(x.z, f, v.z);
            v.w = fmaf(x.w, f, v.w);
        }
        *reinterpret_cast<float4*>(&part[warp][c]) = v;
    }
    __syncthreads();
    const float inv = visible(p, q.len, q.n, tok - q.first) > 0 ? 1.0f / l : 0.0f;
    const int64_t at = tok * d.o_stride + h * d.o_head_stride;
    for (int c = threadIdx.x * 2; c < d.head_dim; c += 2 * kPagedThreads) {
        float x = 0.0f, y = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) {
            x += part[w][c];
            y += part[w][c + 1];
        }
        store_pair<T>(p, at + c, x * inv, y * inv);
    }
}

static int step_keys(const voxq_paged_attn& d) {  // StepShape's KT
    const int hd = d.head_dim <= 64 ? 64 : d.head_dim <= 128 ? 128 : 256;
    return 8192 / (hd * elem_bytes(d.dtype));
}

int paged_step_blocks(const voxq_paged_attn& d, int* whole) {
    const int kt = step_keys(d), group = d.heads / d.kv_heads;
    // as many items and tiles as the bounds admit
    const int64_t items = ((int64_t)d.total_q * group / 16 + std::min(d.batch, d.total_q)) * d.kv_heads;
    const int64_t tiles = std::max<int64_t>((d.max_kv + (int64_t)kt - 1) / kt, 1);
    const int64_t resident = std::min<int64_t>((d.head_dim > 128 ? 1 : 2) * device_sm_count(), kStepPieces);
    *whole = tiles <= kWholeTiles;
    return (int)std::max<int64_t>(1, std::min(resident, *whole ? items : items * tiles / kMinTiles));
}

size_t paged_step_bytes(const voxq_paged_attn& d) {
    int whole;
    const int blocks = paged_step_blocks(d, &whole);
    return whole ? 0 : (size_t)blocks * 2 * 16 * (8 + 4 * (size_t)d.head_dim);
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
    VOXQ_CUDA_TRY(launch_pdl(kern, dim3(a.step_blocks), dim3(kStepThreads), S::bytes, st, a, m));
    if (!a.step_whole)
        VOXQ_CUDA_TRY(launch_pdl(step_combine_kernel<T, S::KT>, dim3(a.d.total_q, a.d.heads), dim3(kPagedThreads), 0, st, a));
    return VOXCPM_SUCCESS;
}

VoxCPMError paged_step_launch(const PagedArgs& call, cudaStream_t st) {
    PagedArgs a = call;
    a.step_blocks = paged_step_blocks(a.d, &a.step_whole);
    a.acc = (float*)a.d.workspace;
    a.ml = (float2*)(a.acc + (size_t)a.step_blocks * 2 * 16 * a.d.head_dim);
    return with_elem(a.d.dtype, [&](auto x) {
        using T = decltype(x);
        const int hd = a.d.head_dim;
        return hd <= 64 ? step_launch<T, 64>(a, st) : hd <= 128 ? step_launch<T, 128>(a, st) : step_launch<T, 256>(a, st);
    });
}

}  // namespace voxq
