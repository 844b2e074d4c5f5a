// voxq_paged_step.cu -- paged attention of at most 16 rows a sequence and kv head: the next-token step.
#include <algorithm>

#include "voxq_internal.h"
#include "voxq_paged.cuh"

namespace voxq {

constexpr int step_keys(int hd, int size) { return 8192 / (hd * size); }

// Shape of the kernel: stages of 16 KB, SW for each warp.  (8 KB stages, two a warp: 39.4 us where this takes 38.0.)
template <typename T, int HD>
struct StepShape {
    static constexpr int KT = step_keys(HD, sizeof(T));      // keys of a tile
    static constexpr int BL = HD * (int)sizeof(T) / 128;     // 128-byte blocks of a row
    static constexpr int P = HD + 16 / (int)sizeof(T);       // shared pitch of the queries
    static constexpr int W = 4, SW = 1, ST = W * SW;  // warps, stages of each
    static constexpr int stage = 2 * KT * HD * (int)sizeof(T);
    static constexpr int MP = HD + 4;                        // pitch of the warps' outputs while they are joined
    static constexpr int bytes = 1024 + ST * stage + W * 16 * MP * 4 + 16 * P * (int)sizeof(T);
    static constexpr int per_sm = HD > 128 ? 1 : 2;          // blocks that share an SM
    static_assert(per_sm * (bytes + 2048) <= 228 * 1024, "shared memory");
};
constexpr int kStepThreads = 128;
// A row's keys stay in one block up to kWholeTiles, or kWholeMany where the rows alone give half of the SMs a block: no join.
// us, whole against cut, kv heads of 128: 1 sequence of 200 keys (7 tiles) 14 : 18, of 900 (29) 23 : 16; 64 of 700 25 : 29;
// 128 of 1000 41 : 47.
constexpr int kWholeTiles = 12, kWholeMany = 40;
constexpr int kMinTiles = 4;  // tiles that are worth a block of their own: one sequence of 900 keys 16 us, 18 with 2 or 8, 25 with 16
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
__device__ __forceinline__ int step_blocks(const PagedArgs& p, int64_t total) {
    return (int)max((int64_t)1, min((int64_t)p.step_blocks, p.step_whole ? total : total / kMinTiles));
}

// Up to 16 rows -- pairs (token, query head of the kv head's group) -- against a sequence's keys: the next-token step.
// It reads the cache once and computes little, so it is bound by HBM, by how early and how evenly the copies are issued
// and by an even share for every block.  Each of four warps takes every fourth tile of the block's stretch by itself, with
// its own stages, running maximum m, sum l and outputs for the 16 rows, so no warp waits for another until they are
// joined.  It also issues its own TMA copies, a lane per box of a page, SW tiles ahead and on into the next row's keys;
// boxes past the last key are left out, and the pages of the tile after next are looked up meanwhile.  (One warp that
// issues for all took 700 clocks a tile, most of them for the copies' operands, and was the bound of short calls; the
// same stages by cp.async took 65 to 150 us where this takes 38 for 64 sequences of 600..4096 keys x 2 heads x 128, 3.9 TB/s,
// since a warp has few of those in flight.)  Two blocks share an SM: one's start and joins hide behind the other's
// stream (with 4 or 6, of smaller stages, 46 and 54 us).  Of the 38 us 1.5 pass before the first tile, blocks end
// between 24 and 32, and the join takes the rest.
template <typename T, int HD>
__global__ void __launch_bounds__(kStepThreads, StepShape<T, HD>::per_sm) paged_step_kernel(const __grid_constant__ PagedArgs p, const __grid_constant__ PagedMaps maps) {
    using S = StepShape<T, HD>;
    constexpr int KT = S::KT, P = S::P, ST = S::ST, W = S::W, NB = HD / 8, KN = KT / 8, MP = S::MP;
    extern __shared__ uint8_t step_sh[];
    __shared__ uint64_t full[ST];
    __shared__ float2 wml[W][16];
    __shared__ int64_t sums[kStepThreads / 32], start_base;
    __shared__ StepSeq start;
    __shared__ int start_seq;
    const uint32_t ring = (smem_u32(step_sh) + 1023) & ~1023u;
    float* mo = reinterpret_cast<float*>(step_sh + (ring - smem_u32(step_sh)) + ST * S::stage);
    T* qs = reinterpret_cast<T*>(mo + W * 16 * MP);
    const voxq_paged_attn& d = p.d;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, G = p.group;
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; i++) mbar_init(full + i, 1);
        mbar_fence_init();
    }
    pdl_wait();
    pdl_launch_dependents();

    // This block's stretch [pos, end), and the sequence that it begins in: an inclusive scan of the sequences' steps.
    const int per = (d.batch + kStepThreads - 1) / kStepThreads;
    int64_t mine = 0;
    for (int i = 0; i < per; i++) {
        const int s = threadIdx.x * per + i;
        if (s < d.batch) mine += step_seq<KT>(p, s).units;
    }
    int64_t before = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int64_t v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
    }
    if (lane == 31) sums[warp] = before;
    __syncthreads();
    before -= mine;
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < kStepThreads / 32; w++) {
        if (w < warp) before += sums[w];
        total += sums[w];
    }
    const int blocks = step_blocks(p, total);
    if ((int)blockIdx.x >= blocks || total == 0) {
        if (threadIdx.x == 0 && !p.step_whole) p.cut[blockIdx.x].pieces = 0;
        return;
    }
    int64_t pos = blockIdx.x * total / blocks;
    const int64_t end = (blockIdx.x + 1) * total / blocks;
    if (pos >= before && pos < before + mine) {
        int s = threadIdx.x * per;
        StepSeq q = step_seq<KT>(p, s);
        for (; pos >= before + q.units; q = step_seq<KT>(p, ++s)) before += q.units;
        start = q;
        start_seq = s;
        start_base = before;
    }
    __syncthreads();
    // A walk over the stretch: at pos, tiles a .. b - 1 of row tile rt and kv head kh of sequence s; c tiles before them.
    struct Walk {
        int64_t pos, base;
        StepSeq q;
        int s, a, b, rt, kh, c;
    };
    auto enter = [&](Walk& w) {
        while (w.pos >= w.base + w.q.units) {
            w.base += w.q.units;
            w.q = step_seq<KT>(p, ++w.s);
        }
        const int64_t in = w.pos - w.base;
        const int item = (int)(in / w.q.line);
        w.a = (int)(in - (int64_t)item * w.q.line);
        w.b = p.step_whole ? w.q.tiles : (int)min((int64_t)w.q.tiles, w.a + (end - w.pos));
        w.kh = item % d.kv_heads;
        w.rt = item / d.kv_heads;
    };
    auto leave = [&](Walk& w) {
        w.c += w.b - w.a;
        w.pos += p.step_whole ? 1 : w.b - w.a;
    };
    Walk it;
    it.pos = pos;
    it.base = start_base;
    it.q = start;
    it.s = start_seq;
    it.c = 0;
    enter(it);

    // The warp's copies run ahead of its products with a walk of their own: its k-th tile, the block's 4 k + warp-th, goes
    // to stage k % SW of its own.  (A barrier's phases can only be told apart by who has seen each of them, and copies may
    // land out of order: stages that warps shared would be read too early.)  A lane has one of the tile's boxes: KT / R
    // for each 128-byte block of its keys and values.
    const int R = maps.box_rows, rows_per = KT / R, boxes = 2 * rows_per * S::BL;
    const int block = lane / rows_per % S::BL, row_in = lane % rows_per * R;
    const bool value = lane >= rows_per * S::BL;
    const uint32_t box_at = ring + warp * S::SW * S::stage + (value ? S::stage / 2 : 0) + block * (KT * 128) + row_in * 128;
    uint64_t* const bars = full + warp * S::SW;
    Walk ahead = it;
    int issued = 0, page = 0, off = 0;
    bool more = true, live = false;
    auto look_up = [&] {  // tile 4 issued + warp
        const int x = issued * W + warp;
        while (x >= ahead.c + ahead.b - ahead.a) {
            leave(ahead);
            more = ahead.pos < end;
            if (!more) return;
            enter(ahead);
        }
        const int key = (ahead.a + x - ahead.c) * KT + row_in;
        live = lane < boxes && key < min(ahead.b * KT, ahead.q.len);
        if (live) {
            const int e = p.page_shift >= 0 ? key >> p.page_shift : (int)((uint32_t)key / (uint32_t)d.page_size);
            page = __ldg(d.block_table + ahead.s * d.table_stride + e);
            off = key - e * d.page_size;
        }
    };
    auto issue = [&] {
        if (!more) return;
        const int k = issued % S::SW, count = __popc(__ballot_sync(0xffffffffu, live));
        if (lane == 0) mbar_arrive_expect_tx(bars + k, count * R * 128);
        __syncwarp();
        if (live)
            tma_page(box_at + k * S::stage, maps, value ? &maps.v : &maps.k, block * (128 / (int)sizeof(T)), off, ahead.kh,
                     (uint32_t)page < (uint32_t)d.pages ? page : 0, bars + k);
        issued++;
        look_up();
    };
    look_up();
#pragma unroll
    for (int k = 0; k < S::SW; k++) issue();

    // The block with the last piece of a cut item -- its first part, which does not begin the item but ends it -- notes
    // what joining the pieces takes.
    if (threadIdx.x == 0 && !p.step_whole) {
        const int64_t at0 = pos - it.a;  // the item's first step
        const int from = (int)(((at0 + 1) * blocks - 1) / total);
        StepCut cut;
        cut.pieces = it.a > 0 && it.b == it.q.tiles ? (int)blockIdx.x - from + 1 : 0;
        cut.later = from * total / blocks < at0;
        cut.first = it.q.first;
        cut.n = it.q.n;
        cut.len = it.q.len;
        cut.row = it.rt * 16;
        cut.kh = it.kh;
        p.cut[blockIdx.x] = cut;
    }
    constexpr int QC = HD * (int)sizeof(T) / 16;
    constexpr bool QREG = !is_f32<T> && HD <= 128;
    bool ok = true;
    int done = 0;  // this warp's tiles
    for (bool again = false; it.pos < end; again = true) {
        if (again) enter(it);
        const StepSeq q = it.q;
        const int a = it.a, b = it.b, kh = it.kh, r0 = it.rt * 16, rows = min(q.n * G - r0, 16), k_stop = min(b * KT, q.len);
        // queries, and this lane's rows: g and g + 8
        for (int i = threadIdx.x; i < 16 * QC; i += 128) {
            const int r = i / QC, x = i % QC * (16 / (int)sizeof(T)), row = r0 + r;
            const bool live = r < rows && x < d.head_dim;
            cp_async16_or_zero(qs + r * P + x, (const T*)d.q + (live ? (q.first + row / G) * d.q_stride + (kh * G + row % G) * d.q_head_stride + x : 0), live);
        }
        cp_async_commit();
        cp_async_wait<0>();
        __syncthreads();
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
        for (int i = a + ((warp - it.c) & (W - 1)); i < b && ok; i += W) {
            const int k = done % S::SW;
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(bars + k, (done / S::SW) & 1, VOXQ_DEVERR_WAIT_FULL, p.err));
            if (!ok) break;
            const uint32_t at = ring + (warp * S::SW + k) * S::stage;
            const SwizzledRows<T, KT> ks{at}, vs{at + S::stage / 2};
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
            done++;
            issue();
        }
        leave(it);
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
        __syncthreads();
        const int r = threadIdx.x >> 3, row = r0 + r;  // 8 threads a row
        const bool all = a == 0 && b == q.tiles;
        uint32_t rows_again = 0;
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
            const float inv = !all ? 1.0f : visible(p, q.len, q.n, row / G) > 0 ? 1.0f / ll : 0.0f;
            const int64_t rec = (blockIdx.x * 2 + (again ? 1 : 0)) * 16 + r;
            const int64_t at = (q.first + row / G) * d.o_stride + (kh * G + row % G) * d.o_head_stride;
            if (!all && (threadIdx.x & 7) == 0) p.ml[rec] = make_float2(mm, ll);
            float chk = 0.0f;
            for (int x = (threadIdx.x & 7) * 2; x < d.head_dim; x += 16) {
                float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < W; w++) {
                    const float2 y = *reinterpret_cast<const float2*>(mo + (w * 16 + r) * MP + x);
                    v.x = fmaf(y.x, f[w], v.x);
                    v.y = fmaf(y.y, f[w], v.y);
                }
                chk = fmaf(v.x, 0.0f, fmaf(v.y, 0.0f, chk));
                if (all) store_pair<T>(p, at + x, v.x * inv, v.y * inv);
                else *reinterpret_cast<float2*>(p.acc + rec * d.head_dim + x) = v;
            }
            if (not_finite<T>(chk, ll)) rows_again = (ll == ll ? 1u : 0x10001u) << r;
        }
        rows_again = __reduce_or_sync(0xffffffffu, rows_again);
        if (rows_again) {  // (of this warp's four)
            __syncwarp();  // what this warp wrote is read
            RowsAgain<T> found(a * KT);
            for (int i = warp * 4; i < warp * 4 + 4; i++)
                if (rows_again >> i & 1)
                    found.row(p, it.s, q.first, r0 + i, kh, a * KT, min(visible(p, q.len, q.n, (r0 + i) / G), k_stop),
                              all ? -1 : (int64_t)(blockIdx.x * 2 + (again ? 1 : 0)) * 16 + i, !(rows_again >> (16 + i) & 1));
        }
        __syncthreads();  // the joined outputs and the queries are read
    }
    if (!ok)  // nothing of this block may still be writing its shared memory when it ends
        for (; done < issued; done++) mbar_wait_bounded(bars + done % S::SW, (done / S::SW) & 1, VOXQ_DEVERR_NONE, p.err);
}

// Joins the pieces of a row that several blocks worked on, in their order: M = max m, out = sum acc 2^(m - M) / sum l 2^(m - M).
// One CTA for each block of the attention and row of its first part, its warps along the pieces; most have nothing to do.
template <typename T>
__global__ void __launch_bounds__(kPagedThreads) step_combine_kernel(const __grid_constant__ PagedArgs p) {
    constexpr int W = kPagedThreads / 32, PER = kStepPieces / kPagedThreads;
    __shared__ float weight[kStepPieces];
    __shared__ __align__(16) float part[W][kPagedMaxHeadDim];
    __shared__ float red[2][W];
    const voxq_paged_attn& d = p.d;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = p.group;
    pdl_wait();
    pdl_launch_dependents();
    const StepCut cut = p.cut[blockIdx.x];
    const int z = cut.pieces, row = cut.row + blockIdx.y, a = blockIdx.x - z + 1;
    if (z < 2 || row >= cut.n * G) return;
    auto record = [&](int j) { return (int64_t)((a + j) * 2 + (j == 0 ? cut.later : 0)) * 16 + blockIdx.y; };
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
    const float inv = visible(p, cut.len, cut.n, row / G) > 0 ? 1.0f / l : 0.0f;
    const int64_t at = (cut.first + row / G) * d.o_stride + (cut.kh * G + row % G) * d.o_head_stride;
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

int paged_step_blocks(const voxq_paged_attn& d, int* whole) {
    const int kt = step_keys(d.head_dim <= 64 ? 64 : d.head_dim <= 128 ? 128 : 256, elem_bytes(d.dtype)), group = d.heads / d.kv_heads;
    // as many items and tiles as the bounds admit
    const int64_t items = ((int64_t)d.total_q * group / 16 + std::min(d.batch, d.total_q)) * d.kv_heads;
    const int64_t tiles = std::max<int64_t>((d.max_kv + (int64_t)kt - 1) / kt, 1);
    const int64_t resident = std::min<int64_t>((d.head_dim > 128 ? 1 : 2) * device_sm_count(), kStepPieces);
    *whole = tiles <= kWholeTiles || (tiles <= kWholeMany && items >= device_sm_count() / 2);
    return (int)std::max<int64_t>(1, std::min(resident, *whole ? items : items * tiles / kMinTiles));
}

size_t paged_step_bytes(const voxq_paged_attn& d) {
    int whole;
    const int blocks = paged_step_blocks(d, &whole);
    return whole ? 0 : (size_t)blocks * (2 * 16 * (8 + 4 * (size_t)d.head_dim) + sizeof(StepCut));
}

template <typename T, int HD>
static VoxCPMError step_launch(const PagedArgs& a, cudaStream_t st) {
    using S = StepShape<T, HD>;
    auto kern = paged_step_kernel<T, HD>;
    static std::atomic<uint64_t> asked{0};
    VOXQ_CUDA_TRY(allow_shared((const void*)kern, S::bytes, asked));
    PagedMaps m;
    const VoxCPMError e = paged_maps(a.d, S::KT, &m);
    if (e != VOXCPM_SUCCESS) return e;
    VOXQ_CUDA_TRY(launch_pdl(kern, dim3(a.step_blocks), dim3(kStepThreads), S::bytes, st, a, m));
    if (!a.step_whole)
        VOXQ_CUDA_TRY(launch_pdl(step_combine_kernel<T>, dim3(a.step_blocks, std::min<int64_t>(16, (int64_t)a.d.max_q * a.group)), dim3(kPagedThreads), 0, st, a));
    return VOXCPM_SUCCESS;
}

VoxCPMError paged_step_launch(const PagedArgs& call, cudaStream_t st) {
    PagedArgs a = call;
    a.step_blocks = paged_step_blocks(a.d, &a.step_whole);
    a.acc = (float*)a.d.workspace;
    a.ml = (float2*)(a.acc + (size_t)a.step_blocks * 2 * 16 * a.d.head_dim);
    a.cut = (StepCut*)(a.ml + (size_t)a.step_blocks * 2 * 16);
    return with_elem(a.d.dtype, [&](auto x) {
        using T = decltype(x);
        const int hd = a.d.head_dim;
        return hd <= 64 ? step_launch<T, 64>(a, st) : hd <= 128 ? step_launch<T, 128>(a, st) : step_launch<T, 256>(a, st);
    });
}

}  // namespace voxq
