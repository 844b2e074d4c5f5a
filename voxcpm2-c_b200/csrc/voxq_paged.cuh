// voxq_paged.cuh -- what the paged-attention kernels share: the call's sizes,
// the walk through the block table, the causal limit and the output types.
#pragma once

#include <cuda.h>

#include "voxq_batch.cuh"

namespace voxq {

constexpr float kLog2e = 1.4426950408889634f;

// voxq_paged_step.cu: what a block leaves for the join of the row tile whose last piece it has.
struct StepCut {
    int pieces;           // its pieces, this block's and the ones before it; fewer than 2: nothing to join
    int later;            // the first piece's block came to it after another part
    int first, n, len;    // the sequence: first row in the batch, rows, positions
    int row, kh;          // the tile's first row among n * group, kv head
};

// The call's sizes as the kernels take them.
struct PagedArgs {
    voxq_paged_attn d;
    int group;        // query heads per kv head
    int page_shift;   // log2(page_size), or -1
    int split_len;    // keys per split (a multiple of the key tile)
    int splits;       // most splits a row can have; 1: none
    float scale2;     // scale * log2(e): the softmax runs in base 2
    float2* ml;       // [total_q][heads][splits] running maximum and sum
    float* acc;       // [total_q][heads][splits][head_dim] unnormalised sums
    int* err;         // device error word of the bounded waits
    StepCut* cut;     // voxq_paged_step.cu: [blocks]
    int step_blocks, step_whole;  // voxq_paged_step.cu: blocks at most; no row's keys are cut
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Offset of cache position j of a sequence (its block-table row `table`) at
// kv head kh, in elements.
__device__ __forceinline__ int64_t cache_row(const PagedArgs& p, const int32_t* table, int j, int kh) {
    const int e = p.page_shift >= 0 ? j >> p.page_shift : (int)((uint32_t)j / (uint32_t)p.d.page_size);
    const int page = __ldg(table + e);
    return (int64_t)((uint32_t)page < (uint32_t)p.d.pages ? page : 0) * p.d.page_stride +
           (int64_t)(j - e * p.d.page_size) * p.d.row_stride + (int64_t)kh * p.d.head_stride;
}

// Positions that row i of a sequence's n sees.
__device__ __forceinline__ int visible(const PagedArgs& p, int len, int n, int i) {
    return p.d.causal ? max(min(len, len - n + i + 1), 0) : len;
}

template <typename T>
__device__ __forceinline__ void store_pair(const PagedArgs& p, int64_t at, float x, float y) {
    if (is_f32<T> || p.d.out_dtype == VOXQ_F32) {
        *reinterpret_cast<float2*>((float*)p.d.out + at) = make_float2(x, y);
    } else {
        T e[2] = {from_f<T>(x), from_f<T>(y)};
        uint32_t v;
        memcpy(&v, e, 4);
        *reinterpret_cast<uint32_t*>((T*)p.d.out + at) = v;
    }
}

__device__ __forceinline__ float lds_f32(uint32_t a) { return __uint_as_float(lds32(a)); }

// Rows of P elements at a shared address.
template <typename T, int P>
struct PaddedRows {
    uint32_t base;
    __device__ __forceinline__ uint32_t operator()(int row, int dim) const { return base + (row * P + dim) * (int)sizeof(T); }
};

// One step of a warp: its 16 rows against 8 KN keys.  16-bit types: m16n8k16 with fp32 accumulation; the weights p
// enter the second product as two 16-bit parts, since one would cost as much accuracy as the output's own rounding.
// fp32: three TF32 products per operand pair (high and low parts).  MMA accumulation truncates, so no sum is left in it for
// long: the scores' go over in fp32 every 64 dims, the low parts' stay apart, the second product's start afresh each step
// (with one chain of three MMAs a step the error at 256 dims was 2e-6, three to seven times a plain fp32 product's).  qs: the rows' queries in shared memory (16-bit types with
// HD <= 128 take them from the registers qf instead), pitch HD + 16 bytes; ks(row, dim), vs(row, dim): shared addresses
// of the keys and values; base: the position
// of this lane's first score column (2 t into the keys); vis: what rows g and g + 8 see; m, l, o: running maxima, this
// lane's share of the sums, and outputs.
template <typename T, int HD, int KN, int QN, typename A>
__device__ __forceinline__ void attend_keys(const PagedArgs& p, const T* qs, const uint32_t (&qf)[QN][4], const A& ks, const A& vs, int base,
                                            const int (&vis)[2], float (&m)[2], float (&l)[2], float (&o)[HD / 8][4]) {
    constexpr int NB = HD / 8, P = HD + 16 / (int)sizeof(T);
    constexpr bool QREG = QN > 1;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
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
                ldsm4(a, smem_u32(qs + (lane & 15) * P + k * 16 + (lane >> 4) * 8));
            }
#pragma unroll
            for (int j = 0; j < KN; j += 2) {
                uint32_t b[4];
                ldsm4(b, ks(j * 8 + (lane & 7) + (lane >> 4) * 8, k * 16 + ((lane >> 3) & 1) * 8));
                mma16<T>(sc[j], a, b[0], b[1]);
                mma16<T>(sc[j + 1], a, b[2], b[3]);
            }
        }
    } else {
        float low[KN][4];
#pragma unroll
        for (int j = 0; j < KN; j++) low[j][0] = low[j][1] = low[j][2] = low[j][3] = 0.0f;
#pragma unroll 1
        for (int k0 = 0; k0 < HD; k0 += 64) {
            float a[KN][4];
#pragma unroll
            for (int j = 0; j < KN; j++) a[j][0] = a[j][1] = a[j][2] = a[j][3] = 0.0f;
#pragma unroll 4
            for (int k = k0; k < k0 + 64; k += 8) {
                uint32_t ah[4], al[4];
                split_tf32(qs[g * P + k + t], ah[0], al[0]);
                split_tf32(qs[(g + 8) * P + k + t], ah[1], al[1]);
                split_tf32(qs[g * P + k + t + 4], ah[2], al[2]);
                split_tf32(qs[(g + 8) * P + k + t + 4], ah[3], al[3]);
#pragma unroll
                for (int j = 0; j < KN; j++) {
                    uint32_t bh[2], bl[2];
                    split_tf32(lds_f32(ks(j * 8 + g, k + t)), bh[0], bl[0]);
                    split_tf32(lds_f32(ks(j * 8 + g, k + t + 4)), bh[1], bl[1]);
                    mma8(low[j], al, bh[0], bh[1]);
                    mma8(low[j], ah, bl[0], bl[1]);
                    mma8(a[j], ah, bh[0], bh[1]);
                }
            }
#pragma unroll
            for (int j = 0; j < KN; j++)
#pragma unroll
                for (int c = 0; c < 4; c++) sc[j][c] += a[j][c];
        }
#pragma unroll
        for (int j = 0; j < KN; j++)
#pragma unroll
            for (int c = 0; c < 4; c++) sc[j][c] += low[j][c];
    }

    // masks, the rows' maxima over the quad, weights
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
                const uint32_t at = vs(k * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, j * 8 + (lane >> 4) * 8);
                asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                             : "=r"(b[0]), "=r"(b[1]), "=r"(b[2]), "=r"(b[3]) : "r"(at) : "memory");
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
#pragma unroll
                for (int i = 0; i < NG; i++) {
                    uint32_t bh[2], bl[2];
                    split_tf32(lds_f32(vs(j * 8 + 2 * t, g + (n0 + i) * 8)), bh[0], bl[0]);
                    split_tf32(lds_f32(vs(j * 8 + 2 * t + 1, g + (n0 + i) * 8)), bh[1], bl[1]);
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

// What the matrix instructions get wrong where something is not finite, put right by a warp.  Operands and weights in two
// parts turn an infinity (and an fp32 value that rounds to one) into a NaN, inf - inf or 0 * inf, and a key that only some of
// a tile's rows see has the weight 0 in the others, where 0 * NaN and 0 * inf are NaN.  So the rows whose sums came out that
// way are looked at again, over the keys that each of them sees: an element that meets values which are not finite is the sum
// of those (a weight is not 0), and a row with any other element that is not finite is taken again in plain fp32.  What is
// still not finite then is so by the formula.  Rows with finite sums pay for a test of them.  us, next
// to the same call without them, with an infinite or a NaN value at every sequence's first position: a step of 64 sequences 405 : 39,
// 6 causal prompts in bf16 5400 : 286, fp32 prompts 1070 : 540.  (A NaN in a query or a key makes its weights NaN: nothing to do in
// 16 bits; 1780 in those fp32 prompts.)

// A row (among the sequence's n * group, its first at `first` of the batch) in plain fp32: a key a lane for the scores, four
// head dims a lane, twice, for the sums.  rec < 0: the result goes to out, else maximum, sum and sums to that record.
template <typename T>
__device__ __forceinline__ void plain_row(const PagedArgs& p, int s, int first, int row, int kh, int k_beg, int k_stop, int64_t rec) {
    const voxq_paged_attn& d = p.d;
    const int lane = threadIdx.x & 31, h = kh * p.group + row % p.group;
    const int64_t tok = first + row / p.group;
    const int32_t* table = d.block_table + s * d.table_stride;
    const T* q = (const T*)d.q + tok * d.q_stride + h * d.q_head_stride;
    float m = -INFINITY, l = 0.0f, o[2][4] = {};
    bool lost = false;  // every element is a NaN for good
#pragma unroll 1
    for (int k0 = k_beg; k0 < k_stop && !lost; k0 += 32) {
        const int64_t at = k0 + lane < k_stop ? cache_row(p, table, k0 + lane, kh) : 0;
        float w = -INFINITY;
        if (k0 + lane < k_stop) {
            w = 0.0f;
#pragma unroll 4
            for (int c = 0; c < d.head_dim; c += 4) {
                float x[4], y[4];
                load4(x, q + c);
                load4(y, (const T*)d.k + at + c);
#pragma unroll
                for (int e = 0; e < 4; e++) w = fmaf(x[e], y[e], w);
            }
            w *= p.scale2;
        }
        float top = fmaxf(w, m);
#pragma unroll
        for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float base = top == -INFINITY ? 0.0f : top, f = ex2(m - base);
        m = top;
        w = ex2(w - base);
        float sum = w;
#pragma unroll
        for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        l = fmaf(l, f, sum);
#pragma unroll
        for (int i = 0; i < 8; i++) o[i / 4][i % 4] *= f;
        const int keys = min(k_stop - k0, 32);
#pragma unroll 4
        for (int j = 0; j < keys; j++) {
            const float wj = __shfl_sync(0xffffffffu, w, j);
            const T* v = (const T*)d.v + __shfl_sync(0xffffffffu, at, j);
#pragma unroll
            for (int i = 0; i < 2; i++)
                if (lane * 4 + i * 128 < d.head_dim) {
                    float x[4];
                    load4(x, v + lane * 4 + i * 128);
#pragma unroll
                    for (int e = 0; e < 4; e++) o[i][e] = fmaf(wj, x[e], o[i][e]);
                }
        }
        lost = true;
#pragma unroll
        for (int i = 0; i < 8; i++) lost = lost && (o[i / 4][i % 4] != o[i / 4][i % 4] || lane * 4 + i / 4 * 128 >= d.head_dim);
        lost = __all_sync(0xffffffffu, lost) || l != l;  // (a NaN in a weight is one in every element)
    }
    if (rec >= 0 && lane == 0) p.ml[rec] = make_float2(m, l);
    const float inv = rec >= 0 ? 1.0f : k_stop > k_beg ? 1.0f / l : 0.0f;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int c = lane * 4 + i * 128;
        if (c >= d.head_dim) break;
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
            const float x = l == l ? o[i][e] * inv : l, y = l == l ? o[i][e + 1] * inv : l;
            if (rec >= 0) *reinterpret_cast<float2*>(p.acc + rec * d.head_dim + c + e) = make_float2(x, y);
            else store_pair<T>(p, tok * d.o_stride + h * d.o_head_stride + c + e, x, y);
        }
    }
}

// Four elements of the output as fp32.
template <typename T>
__device__ __forceinline__ void load_out(const PagedArgs& p, float (&x)[4], int64_t at) {
    if (is_f32<T> || p.d.out_dtype == VOXQ_F32) load4(x, (const float*)p.d.out + at);
    else load4(x, (const T*)p.d.out + at);
}

// The rows of one sequence and kv head that a warp puts right, in rising order: `sum` are the values that are not finite
// among the keys from k_beg to upto, by this lane's head dims.
template <typename T>
struct RowsAgain {
    float sum[2][4];
    int upto;
    __device__ __forceinline__ explicit RowsAgain(int k_beg) : sum{}, upto(k_beg) {}
    // weights: the row's weights are finite.  k_stop: the end of the keys that it sees here.
    __device__ __forceinline__ void row(const PagedArgs& p, int s, int first, int r, int kh, int k_beg, int k_stop, int64_t rec, bool weights) {
        const voxq_paged_attn& d = p.d;
        const int lane = threadIdx.x & 31;
        const int32_t* table = d.block_table + s * d.table_stride;
#pragma unroll 1
        for (; upto < k_stop; upto += 32) {
            const int64_t at = upto + lane < k_stop ? cache_row(p, table, upto + lane, kh) : 0;
            const int keys = min(k_stop - upto, 32);
#pragma unroll 8
            for (int j = 0; j < keys; j++) {
                const T* v = (const T*)d.v + __shfl_sync(0xffffffffu, at, j);
#pragma unroll
                for (int i = 0; i < 2; i++)
                    if (lane * 4 + i * 128 < d.head_dim) {
                        float x[4];
                        load4(x, v + lane * 4 + i * 128);
#pragma unroll
                        for (int e = 0; e < 4; e++) sum[i][e] += x[e] - x[e] == 0.0f ? 0.0f : x[e];
                    }
            }
        }
        // (A row that ends before k_beg sets upto back; the next then counts what is not finite in the keys before k_beg as
        // well, which it sees and which the piece that has them counts too.  Kept from falling, the step kernel's code came
        // out such that one sequence of 517 keys took 8.8 us for 8.1.)
        upto = min(upto, k_stop);
        const int64_t to = rec >= 0 ? rec * d.head_dim : (first + r / p.group) * d.o_stride + (kh * p.group + r % p.group) * d.o_head_stride;
        bool plain = !weights;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int c = lane * 4 + i * 128;
            if (c >= d.head_dim) break;
            float x[4];
            if (rec >= 0) load4(x, p.acc + to + c);
            else load_out<T>(p, x, to + c);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (sum[i][e] != 0.0f) x[e] = sum[i][e];
                else plain = plain || x[e] - x[e] != 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                if (rec >= 0) *reinterpret_cast<float2*>(p.acc + to + c + e) = make_float2(x[e], x[e + 1]);
                else store_pair<T>(p, to + c + e, x[e], x[e + 1]);
            }
        }
        __syncwarp();
        if (__any_sync(0xffffffffu, plain)) plain_row<T>(p, s, first, r, kh, k_beg, k_stop, rec);
    }
};

// A row's sums that have to be looked at again: chk is a sum of 0 * each of them, so a NaN where one is not finite.  In 16 bits the
// scores are single products, so a NaN in l is the formula's, and reaches every element by itself.
template <typename T>
__device__ __forceinline__ bool not_finite(float chk, float l) { return is_f32<T> ? chk != chk || l != l : chk != chk && l == l; }

// Tensor maps of a call's caches: boxes of 128 bytes of one head x box_rows rows of a page, 128-byte-swizzled.
struct PagedMaps {
    CUtensorMap k, v;
    int box_rows;    // a power of two that divides page_size, at least 8, at most max_rows
    int head_first;  // the map's order: dims, heads, rows, pages (else dims, rows, heads, pages), by their strides
};
// page_size a multiple of 8 and positive strides.
bool paged_maps_take(const voxq_paged_attn& d);
VoxCPMError paged_maps(const voxq_paged_attn& d, int max_rows, PagedMaps* m);
// One box: dims x.., rows of a page from `row` on.
__device__ __forceinline__ void tma_page(uint32_t dst, const PagedMaps& m, const CUtensorMap* map, int x, int row, int head, int page, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(m.head_first ? head : row), "r"(m.head_first ? row : head), "r"(page), "r"(smem_u32(bar))
                 : "memory");
}

// Tiles of tr rows, pairs (token, head of the group), that a call can have for all its kv heads: at most one more than full
// tiles for every sequence, and as many a sequence as the longest has.
inline int64_t paged_tiles(const voxq_paged_attn& d, int tr) {
    const int64_t group = d.heads / d.kv_heads, every = d.total_q * group / tr + (d.batch < d.total_q ? d.batch : d.total_q),
                  longest = d.max_q < d.total_q ? d.max_q : d.total_q, most = (longest * group + tr - 1) / tr * d.batch;
    const int64_t tiles = every < most ? every : most;
    return (tiles > 1 ? tiles : 1) * d.kv_heads;
}

constexpr int kPagedThreads = 128;
constexpr int kPagedMaxHeadDim = 256;
// At most 16 rows a sequence (voxq_paged_step.cu), caches that paged_maps_take: everything that the call needs, and the
// workspace that it takes.  VOXCPM_ERR_UNSUPPORTED, like paged_tc_launch, for a layout that a tensor map cannot describe.
size_t paged_step_bytes(const voxq_paged_attn& d);
VoxCPMError paged_step_launch(const PagedArgs& a, cudaStream_t st);
// Attention on the tcgen05 tensor cores (voxq_paged_tc.cu): 16-bit types, scale >= 0, caches that
// paged_maps_take.  Launches the main kernel only.
int paged_tc_rows(const voxq_paged_attn& d);  // rows of a CTA
bool paged_tc_takes(const voxq_paged_attn& d);
VoxCPMError paged_tc_launch(const PagedArgs& a, cudaStream_t st);

}  // namespace voxq
