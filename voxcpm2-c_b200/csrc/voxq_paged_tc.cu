// voxq_paged_tc.cu -- paged attention of many rows on the tcgen05 tensor cores.
#include <cuda.h>

#include <mutex>

#include "voxq_internal.h"
#include "voxq_paged.cuh"

namespace voxq {

constexpr int kTcTile = 128;                 // rows of a query tile, keys of a key tile
constexpr int kTcThreads = 384;              // two softmax warpgroups; the loader warp, the MMA warp and two idle ones
constexpr int kTcRegsSoftmax = 208, kTcRegsOther = 80;  // 256 * 208 + 128 * 80 <= the 384 * 168 of the launch
constexpr int kTcStages = 5;                 // ring of key and value tiles
constexpr int kTcHalf = kTcTile * 128;       // bytes of 128 rows x 64 dims, 128-byte-swizzled rows
constexpr float kTcSlack = 8.0f;             // how far a row's maximum may grow (log2) before its sums are rescaled
template <int HD>
constexpr int kTcTileBytes = kTcHalf * (HD / 64);
template <int HD>
constexpr int kTcSmem = (2 + kTcStages) * kTcTileBytes<HD> + 1024;

// Operand descriptors, 128-byte swizzle, 8-row groups 1024 bytes apart.
// K-major (queries, keys): a row holds 64 of the inner dimension.
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}
// MN-major (values): a row holds 64 head dims of one key; the next 64 dims lie kTcHalf bytes further.
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(kTcHalf >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// kind::f16, fp32 accumulators, M = 128; b_mn: B is MN-major.
template <typename T>
constexpr uint32_t tc_idesc(int n, bool b_mn) {
    const uint32_t type = std::is_same<T, bf16>::value ? 1 : 0;
    return (1u << 4) | (type << 7) | (type << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
                 : "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

#define VOXQ_R8(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
#define VOXQ_S8(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])
// 32 columns of this thread's tensor-memory lane; the caller waits.
__device__ __forceinline__ void tm_ld32(uint32_t addr, uint32_t* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
                 "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : VOXQ_R8(v, 0), VOXQ_R8(v, 8), VOXQ_R8(v, 16), VOXQ_R8(v, 24)
                 : "r"(addr));
}
__device__ __forceinline__ void tm_st32(uint32_t addr, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
                 "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
                 VOXQ_S8(v, 0), VOXQ_S8(v, 8), VOXQ_S8(v, 16), VOXQ_S8(v, 24)
                 : "memory");
}
__device__ __forceinline__ void tm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tma_page(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int page, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(page), "r"(smem_u32(bar))
                 : "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    if constexpr (std::is_same<T, bf16>::value) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __half2 v = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

// A bounded wait whose answer is the same for the whole warp.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int site, int* err) {
    return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, site, err));
}

struct TcMaps {
    CUtensorMap k, v;
    int box_rows;  // rows of a page that one copy takes: gcd(page_size, 128)
    int head_first;  // the map's order: dims, heads, rows, pages (else dims, rows, heads, pages), by their strides
    int* err;
};

// 256 rows -- pairs (token, query head of the group) -- of one sequence and kv
// head against its keys, 128 at a time, as two query tiles of 128 whose steps
// alternate on the tensor cores: while a tile's softmax runs, the other's
// products do.
//   warps 0-3, 4-7  softmax of tile 0, 1: a thread owns one row; scores from
//                   tensor memory, weights back to it over them as the A
//                   operand of the second product, and the output at the end
//   warp 8          loader: the block table's pages by TMA, one box per lane
//   warp 9          issues S = Q K^T and O += P V (one thread)
// Tensor memory: S0, S1 (128 columns each, P over their first 64), O0, O1.
// The tensor pipe runs one thread's MMAs in order, so the S of the next key
// tile may follow the PV that still reads P, and a thread that has seen S
// complete knows that every earlier PV is complete too: it may rescale O
// without a barrier of its own.  Rescaling is rare: sums stay relative to a
// maximum that may be up to 2^8 behind (exact: p, l and O share it).
// p is rounded to the operand type, l sums the fp32 values.  Bound by the
// tensor pipe and, equally at head_dim 128, by the exponentials (16 a clock
// and SM).  Every wait is bounded and records the device error word.
template <typename T, int HD>
__global__ void __launch_bounds__(kTcThreads, 1) paged_tc_kernel(const __grid_constant__ PagedArgs p, const __grid_constant__ TcMaps maps) {
    constexpr int TILE = kTcTileBytes<HD>, ST = kTcStages;
    extern __shared__ uint8_t tc_raw[];
    __shared__ uint64_t bar[2 * ST + 7];
    __shared__ uint32_t tmem_slot;
    uint64_t *full = bar, *empty = bar + ST, *s_full = bar + 2 * ST, *p_full = s_full + 2, *o_done = p_full + 2, *q_full = o_done + 2;
    const voxq_paged_attn& d = p.d;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, G = p.group, kh = blockIdx.y;
    const uint32_t qsm = (smem_u32(tc_raw) + 1023) & ~1023u, ring = qsm + 2 * TILE;
    pdl_wait();
    pdl_launch_dependents();

    // the last rows of a sequence see most keys: start with those
    const int tile = gridDim.x - 1 - blockIdx.x;
    const int s = tile_owner<kTcRows>(d.cu_q, d.batch, G, tile);
    const int first = __ldg(d.cu_q + s), n = min(__ldg(d.cu_q + s + 1), d.total_q) - first;
    const int r0 = (tile - (first * G / kTcRows + s)) * kTcRows, rows = min(n * G - r0, kTcRows);
    if (first < 0 || n <= 0 || r0 < 0 || rows <= 0) return;
    const int len = min(max(__ldg(d.kv_len + s), 0), d.max_kv);
    const int k_end = visible(p, len, n, (r0 + rows - 1) / G);
    const int k_beg = blockIdx.z * p.split_len, k_stop = min(k_end, k_beg + p.split_len);
    if (k_beg >= k_end && blockIdx.z > 0) return;
    const int tiles = k_stop > k_beg ? (k_stop - k_beg + kTcTile - 1) / kTcTile : 0;
    const bool two = rows > kTcTile;

    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; i++) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(s_full + i, 1);
            mbar_init(p_full + i, 4);
            mbar_init(o_done + i, 1);
        }
        mbar_init(q_full, 8);
        mbar_fence_init();
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);

    if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTcRegsOther));
    if (warp == 8) {
        // ---------------- loader: K0, V0, K1, V1, ... ----------------
        const int32_t* table = d.block_table + s * d.table_stride;
        const int R = maps.box_rows, boxes = kTcTile / R * (HD / 64);
        bool ok = true;
        int c = 0;
        for (; c < 2 * tiles && ok; c++) {
            const int slot = c % ST, t0 = k_beg + c / 2 * kTcTile;
            if (c >= ST) ok = warp_wait(empty + slot, (c / ST - 1) & 1, VOXQ_DEVERR_WAIT_EMPTY, maps.err);
            if (!ok) break;
            // boxes that start before k_stop; the rest of the tile is masked
            const int live = (min(k_stop - t0, kTcTile) + R - 1) / R * (HD / 64);
            if (lane == 0) mbar_arrive_expect_tx(full + slot, live * R * 128);
            __syncwarp();
            for (int b = lane; b < boxes; b += 32) {
                const int half = b % (HD / 64), row = b / (HD / 64) * R, key = t0 + row;
                if (key >= k_stop) continue;
                const int e = p.page_shift >= 0 ? key >> p.page_shift : (int)((uint32_t)key / (uint32_t)d.page_size);
                int page = __ldg(table + e);
                if ((uint32_t)page >= (uint32_t)d.pages) page = 0;
                tma_page(ring + slot * TILE + half * kTcHalf + row * 128, c & 1 ? &maps.v : &maps.k, half * 64,
                         maps.head_first ? kh : key - e * d.page_size, maps.head_first ? key - e * d.page_size : kh, page, full + slot);
            }
        }
        if (!ok)  // nothing of this CTA may still be writing its shared memory when it ends
            for (int i = max(0, c - ST); i < c; i++) warp_wait(full + i % ST, (i / ST) & 1, VOXQ_DEVERR_NONE, maps.err);
    } else if (warp == 9) {
        // ---------------- MMA issue ----------------
        constexpr uint32_t id_s = tc_idesc<T>(kTcTile, false), id_o = tc_idesc<T>(HD, true);
        bool ok = tiles == 0 || warp_wait(q_full, 0, VOXQ_DEVERR_WAIT_FULL, maps.err);
        // One lane issues; the operands are the same in every lane, so that they stay in uniform registers.
        const bool one = elect_one();
        auto scores = [&](int t, int slot) {
            const uint64_t qd = desc_k(qsm + t * TILE), kd = desc_k(ring + slot * TILE);
            if (one) {
#pragma unroll
                for (int k = 0; k < HD / 16; k++) {
                    const uint32_t off = ((k / 4) * kTcHalf + (k % 4) * 32) >> 4;
                    mma_ss(tmem + t * kTcTile, qd + off, kd + off, id_s, k > 0);
                }
                tc_commit(s_full + t);
            }
        };
        if (ok && tiles > 0) {
            ok = warp_wait(full + 0, 0, VOXQ_DEVERR_WAIT_FULL, maps.err);
            tc_after();
            if (ok) {
                scores(0, 0);
                if (two) scores(1, 0);
                if (one) tc_commit(empty + 0);
            }
        }
        for (int i = 0; i < tiles && ok; i++) {
            const int cv = 2 * i + 1, sv = cv % ST, ck = 2 * i + 2, sk = ck % ST;
            const int valid = min(k_stop - (k_beg + i * kTcTile), kTcTile), steps = (valid + 15) / 16;
            ok = warp_wait(full + sv, (cv / ST) & 1, VOXQ_DEVERR_WAIT_FULL, maps.err);
            if (!ok) break;
            if (valid % 16) {
                // The last 16 keys that enter the product: values past the end may be anything, and 0 * NaN is
                // NaN, so those rows become zeros.
                const int bad = steps * 16 - valid;
                for (int j = lane; j < bad * (HD / 8); j += 32) {
                    const int row = valid + j / (HD / 8), ch = j % (HD / 8);
                    sts128(ring + sv * TILE + (ch / 8) * kTcHalf + row * 128 + (ch % 8) * 16, make_uint4(0, 0, 0, 0));
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
            for (int t = 0; t < (two ? 2 : 1) && ok; t++) {
                ok = warp_wait(p_full + t, i & 1, VOXQ_DEVERR_WAIT_MMA, maps.err);
                if (!ok) break;
                tc_after();
                const uint64_t vd = desc_mn(ring + sv * TILE);
                if (one) {
#pragma unroll
                    for (int k = 0; k < kTcTile / 16; k++)
                        if (k < steps) mma_ts(tmem + 256 + t * HD, tmem + t * kTcTile + k * 8, vd + (k * 2048 >> 4), id_o, i > 0 || k > 0);
                }
                if (i + 1 < tiles) {
                    if (t == 0) ok = warp_wait(full + sk, (ck / ST) & 1, VOXQ_DEVERR_WAIT_FULL, maps.err);
                    if (ok) scores(t, sk);
                } else if (one) {
                    tc_commit(o_done + t);
                }
            }
            if (one && i + 1 < tiles) {  // (after the last tile nothing waits for them)
                tc_commit(empty + sv);
                tc_commit(empty + sk);
            }
        }
        __syncwarp();
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTcRegsSoftmax));
        // ---------------- softmax and output: one row a thread ----------------
        const int t = warp >> 2, lr = threadIdx.x & 127, r = r0 + t * kTcTile + lr;  // row of the sequence
        const bool mine = t * kTcTile + lr < rows;
        const int tok = r / G, h = kh * G + r % G;
        {
            // the row's queries to shared memory, 16-byte chunk j of a 128-byte row at chunk j ^ (row & 7)
            const uint4* src = reinterpret_cast<const uint4*>((const T*)d.q + (mine ? (first + tok) * d.q_stride + h * d.q_head_stride : 0));
            uint4 v[HD / 8];
#pragma unroll
            for (int j = 0; j < HD / 8; j++) v[j] = mine ? src[j] : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int j = 0; j < HD / 8; j++) sts128(qsm + t * TILE + (j / 8) * kTcHalf + lr * 128 + (((j % 8) ^ (lr & 7)) << 4), v[j]);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        const int seen = mine ? visible(p, len, n, tok) : 0, vis = min(seen, k_stop);
        // keys that every row of the tile sees need no mask
        const int all_see = visible(p, len, n, (r0 + t * kTcTile) / G);
        const uint32_t ts = tmem + ((uint32_t)((warp & 3) * 32) << 16) + t * kTcTile, to = tmem + ((uint32_t)((warp & 3) * 32) << 16) + 256 + t * HD;
        const bool active = t == 0 || two;
        float m = -INFINITY, l = 0.0f;  // m in base-2 units
        bool ok = true;
        for (int i = 0; i < tiles && active; i++) {
            const int t0 = k_beg + i * kTcTile;
            ok = warp_wait(s_full + t, i & 1, VOXQ_DEVERR_WAIT_MMA, maps.err);
            if (!ok) break;
            tc_after();
            uint32_t sv[kTcTile];
#pragma unroll
            for (int c = 0; c < kTcTile; c += 32) tm_ld32(ts + c, sv + c);
            tm_wait_ld();
            if (t0 + kTcTile > min(all_see, k_stop)) {
#pragma unroll
                for (int c = 0; c < kTcTile; c++)
                    if (t0 + c >= vis) sv[c] = __float_as_uint(-INFINITY);
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < kTcTile; c += 8)
#pragma unroll
                for (int e = 0; e < 4; e++) mx[e] = fmaxf(fmaxf(mx[e], __uint_as_float(sv[c + e])), __uint_as_float(sv[c + e + 4]));
            const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale2;
            if (i == 0) {
                m = mt;
            } else {
                const bool grow = mt > m + kTcSlack;
                if (__any_sync(0xffffffffu, grow)) {
                    const float f = grow ? ex2(m - mt) : 1.0f;
                    if (grow) m = mt;
                    l *= f;
#pragma unroll
                    for (int c = 0; c < HD; c += 32) {
                        uint32_t o[32];
                        tm_ld32(to + c, o);
                        tm_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tm_st32(to + c, o);
                    }
                }
            }
            const float neg = m == -INFINITY ? 0.0f : -m;  // no key so far: every weight is ex2(-inf) = 0
            const uint64_t sc2 = pk(p.scale2, p.scale2), ng2 = pk(neg, neg);
            uint64_t sum[2] = {pk(0.0f, 0.0f), pk(0.0f, 0.0f)};
#pragma unroll
            for (int c0 = 0; c0 < kTcTile; c0 += 64) {
                uint32_t w[32];
#pragma unroll
                for (int c = 0; c < 64; c += 2) {
                    float x, y;
                    upk(fma2(pk(__uint_as_float(sv[c0 + c]), __uint_as_float(sv[c0 + c + 1])), sc2, ng2), x, y);
                    x = ex2(x);
                    y = ex2(y);
                    sum[(c >> 1) & 1] = add2(sum[(c >> 1) & 1], pk(x, y));
                    w[c >> 1] = pack2<T>(x, y);
                }
                tm_st32(ts + c0 / 2, w);
            }
            float a, b, e, f;
            upk(sum[0], a, b);
            upk(sum[1], e, f);
            l += (a + b) + (e + f);
            tm_wait_st();
            tc_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + t);
        }
        if (ok && tiles > 0 && active) {
            ok = warp_wait(o_done + t, 0, VOXQ_DEVERR_WAIT_MMA, maps.err);
            tc_after();
        }
        const bool whole = seen <= p.split_len;
        // a row with more keys than a split holds leaves a record, one with fewer is split 0's
        const bool put = ok && mine && (whole ? blockIdx.z == 0 : k_beg < seen);
        const float inv = !whole ? 1.0f : seen > 0 ? 1.0f / l : 0.0f;
        const int64_t rec = ((int64_t)(first + tok) * d.heads + h) * p.splits + blockIdx.z;
        const int64_t at = (first + tok) * d.o_stride + h * d.o_head_stride;
        if (put && !whole) p.ml[rec] = make_float2(m, l);
        if (active)
#pragma unroll
            for (int c = 0; c < HD; c += 32) {
                uint32_t o[32];
                if (tiles > 0) {
                    tm_ld32(to + c, o);
                    tm_wait_ld();
                }
                if (!put) continue;
#pragma unroll
                for (int e = 0; e < 32; e++) o[e] = seen > 0 ? __float_as_uint(__uint_as_float(o[e]) * inv) : 0u;
                if (!whole || d.out_dtype == VOXQ_F32) {
                    uint4* dst = reinterpret_cast<uint4*>((whole ? (float*)d.out + at : p.acc + rec * HD) + c);
#pragma unroll
                    for (int e = 0; e < 8; e++) dst[e] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                } else {
                    uint4* dst = reinterpret_cast<uint4*>((T*)d.out + at + c);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        uint32_t w[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) w[j] = pack2<T>(__uint_as_float(o[8 * e + 2 * j]), __uint_as_float(o[8 * e + 2 * j + 1]));
                        dst[e] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
    }
    tc_before();
    __syncthreads();
    if (warp == 9) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
    static std::once_flag once;
    static EncodeTiled fn = nullptr;
    std::call_once(once, [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiled>(f);
    });
    return fn;
}

bool paged_tc_takes(const voxq_paged_attn& d) {
    const int64_t lim = (int64_t)1 << 39;  // elements: a tensor map's strides are below 2^40 bytes
    return d.dtype != VOXQ_F32 && (d.head_dim == 64 || d.head_dim == 128) && d.page_size > 0 && d.page_size % 8 == 0 && d.scale >= 0.0f &&
           d.pages > 0 && d.page_stride > 0 && d.row_stride > 0 && d.head_stride > 0 && d.page_stride < lim && d.row_stride < lim &&
           d.head_stride < lim;
}

template <typename T, int HD>
static VoxCPMError tc_launch(const PagedArgs& a, cudaStream_t st) {
    auto kern = paged_tc_kernel<T, HD>;
    static std::once_flag once;
    static cudaError_t attr = cudaSuccess;
    std::call_once(once, [&] { attr = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kTcSmem<HD>); });
    VOXQ_CUDA_TRY(attr);
    const voxq_paged_attn& d = a.d;
    EncodeTiled enc = encode_tiled();
    TcMaps m;
    m.err = device_error_word();
    if (!enc || !m.err) return VOXCPM_ERR_INTERNAL;
    m.box_rows = d.page_size & -d.page_size;
    if (m.box_rows > kTcTile) m.box_rows = kTcTile;
    m.head_first = d.head_stride <= d.row_stride;
    const int hi = m.head_first ? 1 : 2, ri = 3 - hi;
    cuuint64_t dims[4] = {(cuuint64_t)HD, 0, 0, (cuuint64_t)d.pages}, strides[3] = {0, 0, (cuuint64_t)d.page_stride * 2};
    cuuint32_t box[4] = {64, 1, 1, 1}, one[4] = {1, 1, 1, 1};
    dims[hi] = (cuuint64_t)d.kv_heads;
    dims[ri] = (cuuint64_t)d.page_size;
    strides[hi - 1] = (cuuint64_t)d.head_stride * 2;
    strides[ri - 1] = (cuuint64_t)d.row_stride * 2;
    box[ri] = (cuuint32_t)m.box_rows;
    const CUtensorMapDataType dt = std::is_same<T, bf16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    for (int i = 0; i < 2; i++)
        if (enc(i ? &m.v : &m.k, dt, 4, const_cast<void*>(i ? d.v : d.k), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return VOXCPM_ERR_UNSUPPORTED;  // a layout that a tensor map cannot describe
    const dim3 grid((int)((int64_t)d.total_q * a.group / kTcRows) + d.batch, d.kv_heads, a.splits);
    VOXQ_CUDA_TRY(launch_pdl(kern, grid, dim3(kTcThreads), kTcSmem<HD>, st, a, m));
    return VOXCPM_SUCCESS;
}

VoxCPMError paged_tc_launch(const PagedArgs& a, cudaStream_t st) {
    if (a.d.dtype == VOXQ_F16) return a.d.head_dim == 64 ? tc_launch<__half, 64>(a, st) : tc_launch<__half, 128>(a, st);
    return a.d.head_dim == 64 ? tc_launch<bf16, 64>(a, st) : tc_launch<bf16, 128>(a, st);
}

}  // namespace voxq
