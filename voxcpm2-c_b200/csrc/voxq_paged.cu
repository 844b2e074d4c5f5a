// voxq_paged.cu -- attention of a ragged batch's new tokens over a paged KV cache.
#include <math.h>

#include <algorithm>
#include <mutex>

#include "voxq_internal.h"
#include "voxq_paged.cuh"

namespace voxq {

constexpr int kPagedThreads = 128;
constexpr int kPagedMaxHeadDim = 256;
constexpr int kSplitCtas = 4;   // CTAs per SM that splitting the keys aims at
constexpr int kTcSplitCtas = 1;  // the same for the tcgen05 kernel, one CTA of which fills an SM
constexpr int kTcMinRows = 64;   // rows a sequence from which that kernel's 128-row tiles pay
constexpr int kMinSplit = 256;  // keys that are worth a CTA of their own
constexpr int kMaxSplits = 128;

// Shape of the kernel for element type T, head dims up to HD and WM warps
// along the rows (the other 4 / WM along the keys of a tile).
template <typename T, int HD, int WM>
struct PagedShape {
    static constexpr int WK = 4 / WM, TR = 16 * WM;       // rows of a tile
    static constexpr int BK = is_f32<T> ? 32 : 64;         // keys of a tile
    static constexpr int KW = BK / WK;                     // of a warp
    static constexpr int ST = HD > 128 ? 2 : 3;            // cp.async stages
    static constexpr int P = HD + 16 / (int)sizeof(T);     // shared pitch: 16 bytes more than a row
    static constexpr int stage = 2 * BK * P * (int)sizeof(T);
    static constexpr int merge = WK > 1 ? WK * 16 * (HD + 4) * 4 : 0;
    static constexpr int bytes = TR * P * (int)sizeof(T) + (ST * stage > merge ? ST * stage : merge);
    static_assert(bytes <= 227 * 1024, "shared memory");
};

// Attention on warp-level MMAs, for every element type, head dim and page
// size: few rows a sequence (steps, short chunks), fp32, and the head dims
// that the tcgen05 kernel does not take.
//
// The rows of a tile are the pairs (token, query head of the kv head's group),
// so a key is read once for all heads that share it.  Keys and values of BK
// positions arrive by cp.async, three stages deep, each thread following the
// block table for its own rows of the tile (a page may end anywhere inside
// it); rows past the end are zeros in shared memory, whatever the cache holds.
// One pass, base-2 softmax with running maximum m and sum l per row.
//   WM = 1  16 rows a tile, each warp a quarter of the tile's keys with its own
//           m, l and sums, joined in shared memory at the end.  A step reads
//           the cache once and computes little: bound by HBM.
//   WM = 4  64 rows a tile, each warp 16 rows and all keys.
// With few tiles the keys are split over CTAs (blockIdx.z); a row with more
// than one split leaves (m, l, sums) for paged_combine_kernel.
// 16-bit types: m16n8k16, fp32 accumulation; the weights p enter the second
// product as two 16-bit parts, since one would cost as much accuracy as the
// output's own rounding.  fp32: three TF32 products per operand pair (high and
// low parts), the second product's sums started afresh each tile and added in
// fp32, because MMA accumulation truncates.
template <typename T, int HD, int WM>
__global__ void __launch_bounds__(kPagedThreads) paged_mma_kernel(const __grid_constant__ PagedArgs p) {
    using S = PagedShape<T, HD, WM>;
    constexpr int WK = S::WK, TR = S::TR, BK = S::BK, KW = S::KW, P = S::P, ST = S::ST;
    constexpr int NB = HD / 8, KN = KW / 8;
    extern __shared__ __align__(16) uint8_t paged_sh[];
    T* qs = reinterpret_cast<T*>(paged_sh);
    T* kv = qs + TR * P;
    const voxq_paged_attn& d = p.d;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int wm = warp % WM, wk = warp / WM, kh = blockIdx.y, G = p.group;
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

    constexpr int E = 16 / sizeof(T), CPR = HD / E, RP = kPagedThreads / CPR;  // vectors per row, rows per pass
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
    for (int i = threadIdx.x; i < TR * CPR; i += kPagedThreads) {
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
        const T* ks = kv + stage * 2 * BK * P + wk * KW * P;
        const T* vs = ks + BK * P;
        const T* qw = qs + wm * 16 * P;
        stage = stage + 1 == ST ? 0 : stage + 1;
        if constexpr (QREG) {
            if (t0 == k_beg)
#pragma unroll
                for (int k = 0; k < HD / 16; k++) ldsm4(qf[k], smem_u32(qw + (lane & 15) * P + k * 16 + (lane >> 4) * 8));
        }

        float sc[KN][4];
#pragma unroll
        for (int j = 0; j < KN; j++) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.0f;
        if constexpr (!is_f32<T>) {
#pragma unroll
            for (int k = 0; k < HD / 16; k++) {
                uint32_t a[4];
                if constexpr (QREG) {
                    a[0] = qf[k][0], a[1] = qf[k][1], a[2] = qf[k][2], a[3] = qf[k][3];
                } else {
                    ldsm4(a, smem_u32(qw + (lane & 15) * P + k * 16 + (lane >> 4) * 8));
                }
#pragma unroll
                for (int j = 0; j < KN; j += 2) {
                    uint32_t b[4];
                    ldsm4(b, smem_u32(ks + (j * 8 + (lane & 7) + (lane >> 4) * 8) * P + k * 16 + ((lane >> 3) & 1) * 8));
                    mma16<T>(sc[j], a, b[0], b[1]);
                    mma16<T>(sc[j + 1], a, b[2], b[3]);
                }
            }
        } else {
#pragma unroll 4
            for (int k = 0; k < HD; k += 8) {
                uint32_t ah[4], al[4];
                split_tf32(qw[g * P + k + t], ah[0], al[0]);
                split_tf32(qw[(g + 8) * P + k + t], ah[1], al[1]);
                split_tf32(qw[g * P + k + t + 4], ah[2], al[2]);
                split_tf32(qw[(g + 8) * P + k + t + 4], ah[3], al[3]);
#pragma unroll
                for (int j = 0; j < KN; j++) {
                    uint32_t bh[2], bl[2];
                    split_tf32(ks[(j * 8 + g) * P + k + t], bh[0], bl[0]);
                    split_tf32(ks[(j * 8 + g) * P + k + t + 4], bh[1], bl[1]);
                    mma8(sc[j], al, bh[0], bh[1]);
                    mma8(sc[j], ah, bl[0], bl[1]);
                    mma8(sc[j], ah, bh[0], bh[1]);
                }
            }
        }

        // masks, the rows' maxima over the quad, weights
        const int base = t0 + wk * KW + 2 * t;
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < KN; j++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                sc[j][c] = base + j * 8 + (c & 1) < vis[c >> 1] ? sc[j][c] * p.scale2 : -INFINITY;
                mx[c >> 1] = fmaxf(mx[c >> 1], sc[j][c]);
            }
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
            mx[e] = fmaxf(fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2)), m[e]);
            f[e] = m[e] == -INFINITY ? 0.0f : ex2(m[e] - mx[e]);
            m[e] = mx[e];
            mx[e] = mx[e] == -INFINITY ? 0.0f : mx[e];  // no key so far: every weight is ex2(-inf) = 0
            l[e] *= f[e];
        }
#pragma unroll
        for (int j = 0; j < KN; j++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                sc[j][c] = ex2(sc[j][c] - mx[c >> 1]);
                l[c >> 1] += sc[j][c];
            }

        if constexpr (!is_f32<T>) {
#pragma unroll
            for (int j = 0; j < NB; j++) {
                o[j][0] *= f[0], o[j][1] *= f[0];
                o[j][2] *= f[1], o[j][3] *= f[1];
            }
#pragma unroll
            for (int k = 0; k < KN / 2; k++) {
                uint32_t ph[4], pl[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float x = sc[2 * k + e / 2][e % 2 * 2], y = sc[2 * k + e / 2][e % 2 * 2 + 1];
                    const T hi[2] = {from_f<T>(x), from_f<T>(y)};
                    const T lo[2] = {from_f<T>(x - to_f(hi[0])), from_f<T>(y - to_f(hi[1]))};
                    memcpy(&ph[e], hi, 4);
                    memcpy(&pl[e], lo, 4);
                }
#pragma unroll
                for (int j = 0; j < NB; j += 2) {
                    uint32_t b[4];
                    const T* at = vs + (k * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * P + j * 8 + (lane >> 4) * 8;
                    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(b[0]), "=r"(b[1]), "=r"(b[2]), "=r"(b[3]) : "r"(smem_u32(at)) : "memory");
                    mma16<T>(o[j], pl, b[0], b[1]);
                    mma16<T>(o[j + 1], pl, b[2], b[3]);
                    mma16<T>(o[j], ph, b[0], b[1]);
                    mma16<T>(o[j + 1], ph, b[2], b[3]);
                }
            }
        } else {
            constexpr int NG = NB < 8 ? NB : 8;  // head-dim blocks whose sums are open at once
#pragma unroll
            for (int n0 = 0; n0 < NB; n0 += NG) {
                float a[NG][4];
#pragma unroll
                for (int i = 0; i < NG; i++) a[i][0] = a[i][1] = a[i][2] = a[i][3] = 0.0f;
                // A column t is key 2t and column t + 4 key 2t + 1 of the 8: the scores' own layout
#pragma unroll
                for (int j = 0; j < KN; j++) {
                    uint32_t ah[4], al[4];
                    split_tf32(sc[j][0], ah[0], al[0]);
                    split_tf32(sc[j][2], ah[1], al[1]);
                    split_tf32(sc[j][1], ah[2], al[2]);
                    split_tf32(sc[j][3], ah[3], al[3]);
                    const T* v0 = vs + (j * 8 + 2 * t) * P + g + n0 * 8;
#pragma unroll
                    for (int i = 0; i < NG; i++) {
                        uint32_t bh[2], bl[2];
                        split_tf32(v0[i * 8], bh[0], bl[0]);
                        split_tf32(v0[i * 8 + P], bh[1], bl[1]);
                        mma8(a[i], al, bh[0], bh[1]);
                        mma8(a[i], ah, bl[0], bl[1]);
                        mma8(a[i], ah, bh[0], bh[1]);
                    }
                }
#pragma unroll
                for (int i = 0; i < NG; i++)
#pragma unroll
                    for (int c = 0; c < 4; c++) o[n0 + i][c] = fmaf(o[n0 + i][c], f[c >> 1], a[i][c]);
            }
        }
    }
    cp_async_wait<0>();
#pragma unroll
    for (int e = 0; e < 2; e++) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    }

    // A row's result goes to out, or, when its keys fill more than one split, to this split's record.
    auto whole = [&](int r) { return visible(p, len, n, r / G) <= p.split_len; };
    auto head_row = [&](int r) { return (int64_t)(first + r / G) * d.heads + kh * G + r % G; };
    auto out_at = [&](int r) { return (first + r / G) * d.o_stride + (kh * G + r % G) * d.o_head_stride; };
    if constexpr (WK == 1) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int r = row[e];
            if (r >= n * G) continue;
            if (whole(r)) {
                if (blockIdx.z > 0) continue;
                const float inv = vis[e] > 0 ? 1.0f / l[e] : 0.0f;
                const int64_t at = out_at(r);
#pragma unroll
                for (int j = 0; j < NB; j++)
                    if (j * 8 < d.head_dim) store_pair<T>(p, at + j * 8 + 2 * t, o[j][2 * e] * inv, o[j][2 * e + 1] * inv);
            } else if (k_beg < visible(p, len, n, r / G)) {
                const int64_t rec = head_row(r) * p.splits + blockIdx.z;
                if (t == 0) p.ml[rec] = make_float2(m[e], l[e]);
#pragma unroll
                for (int j = 0; j < NB; j++)
                    if (j * 8 < d.head_dim)
                        *reinterpret_cast<float2*>(p.acc + rec * d.head_dim + j * 8 + 2 * t) = make_float2(o[j][2 * e], o[j][2 * e + 1]);
            }
        }
    } else {
        // join the warps' sums over their shares of the keys
        constexpr int MP = HD + 4;
        __shared__ float2 wml[WK][16];
        float* mo = reinterpret_cast<float*>(kv);
        __syncthreads();  // every stage is read
#pragma unroll
        for (int e = 0; e < 2; e++) {
            if (t == 0) wml[wk][g + 8 * e] = make_float2(m[e], l[e]);
#pragma unroll
            for (int j = 0; j < NB; j++)
                *reinterpret_cast<float2*>(mo + (wk * 16 + g + 8 * e) * MP + j * 8 + 2 * t) = make_float2(o[j][2 * e], o[j][2 * e + 1]);
        }
        __syncthreads();
        const int r = threadIdx.x >> 3, rr = r0 + r;  // 8 threads a row
        if (r >= rows) return;
        float mm = -INFINITY, ll = 0.0f, f[WK];
#pragma unroll
        for (int w = 0; w < WK; w++) mm = fmaxf(mm, wml[w][r].x);
#pragma unroll
        for (int w = 0; w < WK; w++) {
            f[w] = wml[w][r].x == -INFINITY ? 0.0f : ex2(wml[w][r].x - mm);
            ll = fmaf(wml[w][r].y, f[w], ll);
        }
        const int seen = visible(p, len, n, rr / G);
        const bool all = seen <= p.split_len;
        if (all ? blockIdx.z > 0 : k_beg >= seen) return;
        const float inv = !all ? 1.0f : seen > 0 ? 1.0f / ll : 0.0f;
        const int64_t rec = head_row(rr) * p.splits + blockIdx.z, at = out_at(rr);
        if (!all && (threadIdx.x & 7) == 0) p.ml[rec] = make_float2(mm, ll);
        for (int c = (threadIdx.x & 7) * 2; c < d.head_dim; c += 16) {
            float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < WK; w++) {
                const float2 x = *reinterpret_cast<const float2*>(mo + (w * 16 + r) * MP + c);
                v.x = fmaf(x.x, f[w], v.x);
                v.y = fmaf(x.y, f[w], v.y);
            }
            if (all) store_pair<T>(p, at + c, v.x * inv, v.y * inv);
            else *reinterpret_cast<float2*>(p.acc + rec * d.head_dim + c) = v;
        }
    }
}

// Joins a row's splits in their order: M = max m_z, out = sum_z acc_z 2^(m_z - M)
// / sum_z l_z 2^(m_z - M).  One CTA per token, a thread per two dims.
template <typename T>
__global__ void __launch_bounds__(kPagedThreads) paged_combine_kernel(const __grid_constant__ PagedArgs p) {
    const voxq_paged_attn& d = p.d;
    pdl_wait();
    pdl_launch_dependents();
    const int tok = blockIdx.x;
    int s = -1;
    for (int i0 = 0; i0 < d.batch; i0 += kPagedThreads)
        s += __syncthreads_count(i0 + threadIdx.x < d.batch && __ldg(d.cu_q + i0 + threadIdx.x) <= tok);
    s = max(s, 0);
    const int first = __ldg(d.cu_q + s), n = min(__ldg(d.cu_q + s + 1), d.total_q) - first;
    const int len = min(max(__ldg(d.kv_len + s), 0), d.max_kv);
    const int seen = tok >= first && tok < first + n ? visible(p, len, n, tok - first) : 0;
    if (seen <= p.split_len) return;
    const int z = (seen + p.split_len - 1) / p.split_len, half = d.head_dim / 2;
    for (int i = blockIdx.y * kPagedThreads + threadIdx.x; i < d.heads * half; i += gridDim.y * kPagedThreads) {
        const int h = i / half, c = i % half * 2;
        const int64_t rec = ((int64_t)tok * d.heads + h) * p.splits;
        float mm = -INFINITY;
        for (int j = 0; j < z; j++) mm = fmaxf(mm, p.ml[rec + j].x);
        float l = 0.0f, x = 0.0f, y = 0.0f;
        for (int j = 0; j < z; j++) {
            const float2 ml = p.ml[rec + j];
            const float f = ml.x == -INFINITY ? 0.0f : ex2(ml.x - mm);
            const float2 a = *reinterpret_cast<const float2*>(p.acc + (rec + j) * d.head_dim + c);
            l = fmaf(ml.y, f, l);
            x = fmaf(a.x, f, x);
            y = fmaf(a.y, f, y);
        }
        store_pair<T>(p, tok * d.o_stride + h * d.o_head_stride + c, x / l, y / l);
    }
}

// What a call runs: rows per tile, and the keys per split.  A pure function of
// the descriptor's integers, so that the workspace is known beforehand.
struct PagedPlan {
    bool tc;        // tcgen05 kernel
    int wm;         // warps along the rows of the other
    int split_len, splits;
    size_t bytes;   // workspace
};

static PagedPlan paged_plan(const voxq_paged_attn& d) {
    PagedPlan r;
    const int G = d.heads / d.kv_heads;
    // 16-row tiles while a sequence's rows fit in one
    r.wm = (int64_t)d.max_q * G <= 16 ? 1 : 4;
    r.tc = (int64_t)d.max_q * G > kTcMinRows && paged_tc_takes(d);
    const int tr = r.tc ? kTcRows : 16 * r.wm, ctas = r.tc ? kTcSplitCtas : kSplitCtas;
    // CTAs without splitting, and the splits that bring them to kSplitCtas per SM
    const int64_t per_seq = std::max<int64_t>(1, std::min<int64_t>(d.batch, d.total_q));
    const int64_t tiles = std::max<int64_t>(per_seq, (int64_t)d.total_q * G / tr) * d.kv_heads;
    const int64_t want = (ctas * device_sm_count() + tiles - 1) / tiles;
    const int64_t most = std::max<int64_t>(1, (d.max_kv + kMinSplit - 1) / kMinSplit);
    const int64_t z = std::min(std::min(want, most), (int64_t)kMaxSplits);
    r.split_len = (int)(((d.max_kv + z - 1) / z + 127) / 128 * 128);  // whole tiles of either kernel
    r.splits = r.split_len ? (d.max_kv + r.split_len - 1) / r.split_len : 1;
    if (r.splits <= 1) {
        r.splits = 1;
        r.split_len = INT32_MAX;
    }
    r.bytes = r.splits > 1 ? (size_t)d.total_q * d.heads * r.splits * (8 + 4 * (size_t)d.head_dim) : 0;
    return r;
}

template <typename T, int HD, int WM>
static VoxCPMError paged_mma_launch(const PagedArgs& a, cudaStream_t st) {
    using S = PagedShape<T, HD, WM>;
    auto kern = paged_mma_kernel<T, HD, WM>;
    static std::once_flag once;
    static cudaError_t attr = cudaSuccess;
    std::call_once(once, [&] { attr = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::bytes); });
    VOXQ_CUDA_TRY(attr);
    const dim3 grid((int)((int64_t)a.d.total_q * a.group / S::TR) + a.d.batch, a.d.kv_heads, a.splits);
    VOXQ_CUDA_TRY(launch_pdl(kern, grid, dim3(kPagedThreads), S::bytes, st, a));
    return VOXCPM_SUCCESS;
}

template <typename T>
static VoxCPMError paged_run(const PagedArgs& a, const PagedPlan& plan, cudaStream_t st) {
    const int hd = a.d.head_dim;
    // (a cache layout that a tensor map cannot describe goes to the other kernel)
    VoxCPMError e = plan.tc ? paged_tc_launch(a, st) : VOXCPM_ERR_UNSUPPORTED;
    if (e == VOXCPM_ERR_UNSUPPORTED && plan.wm == 1)
        e = hd <= 64 ? paged_mma_launch<T, 64, 1>(a, st) : hd <= 128 ? paged_mma_launch<T, 128, 1>(a, st) : paged_mma_launch<T, 256, 1>(a, st);
    else if (e == VOXCPM_ERR_UNSUPPORTED)
        e = hd <= 64 ? paged_mma_launch<T, 64, 4>(a, st) : hd <= 128 ? paged_mma_launch<T, 128, 4>(a, st) : paged_mma_launch<T, 256, 4>(a, st);
    if (e != VOXCPM_SUCCESS || a.splits == 1) return e;
    const int per = a.d.heads * hd / 2, y = std::min(8, (per + kPagedThreads - 1) / kPagedThreads);
    VOXQ_CUDA_TRY(launch_pdl(paged_combine_kernel<T>, dim3(a.d.total_q, y), dim3(kPagedThreads), 0, st, a));
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
    if ((int64_t)d->total_q * d->heads + d->batch > INT32_MAX || d->kv_heads > 65535 || d->max_kv > 1 << 30)
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
    a.split_len = plan.split_len;
    a.splits = plan.splits;
    a.scale2 = (d->scale != 0.0f ? d->scale : 1.0f / sqrtf((float)d->head_dim)) * kLog2e;
    a.acc = (float*)d->workspace;
    a.ml = (float2*)(a.acc + (size_t)d->total_q * d->heads * plan.splits * d->head_dim);
    return with_elem(d->dtype, [&](auto x) { return paged_run<decltype(x)>(a, plan, (cudaStream_t)stream); });
}
