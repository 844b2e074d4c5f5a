// voxq_paged_tc.cu -- paged attention of many rows on the tcgen05 tensor cores.
#include <cuda.h>

#include <mutex>

#include "voxq_internal.h"
#include "voxq_paged.cuh"

namespace voxq {

constexpr int kTcTile = 128;                 // rows of a query tile, keys of a key tile
constexpr int kTcThreads = 384;              // two softmax warpgroups; loader, MMA and unit warps, one for rows to put right
constexpr int kTcRegsSoftmax = 208, kTcRegsOther = 80;  // 256 * 208 + 128 * 80 <= the 384 * 168 of the launch
template <int HD>
constexpr int kTcTiles = HD > 128 ? 1 : 2;   // query tiles of a unit: tensor memory holds the output of 256 columns once
template <int HD>
constexpr int kTcStages = HD > 128 ? 2 : 5;  // ring of key and value tiles
constexpr int kTcHalf = kTcTile * 128;       // bytes of 128 rows x 64 dims, 128-byte-swizzled rows
// Barriers of the mended ends of units, in turn.  Before the MMA warp waits for a unit's it has freed that unit's last key tile but
// not its last value tile, so of a ring of five the loader can have mended that unit's end and two more (units of one tile
// each: V K V K V), never a fourth, and a barrier's phase is seen before its next one begins.
constexpr int kTcTails = 3;
constexpr int kTcItems = 4;                  // units in flight between the warps of a block
constexpr int kTcSeqs = 4;                   // of 32 sequences: up to how many the units are taken in order of their keys
constexpr float kTcSlack = 8.0f;             // how far a row's maximum may grow (log2) before its sums are rescaled
template <int HD>
constexpr int kTcTileBytes = kTcHalf * (HD / 64);
template <int HD>
constexpr int kTcSmem = (kTcTiles<HD> + kTcStages<HD>) * kTcTileBytes<HD> + 1024;

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

// The softmax's arithmetic in an order that stays as it is written.
__device__ __forceinline__ float ex2v(float x) {
    float y;
    asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint64_t fma2v(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm volatile("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2v(uint64_t a, uint64_t b) {
    uint64_t d;
    asm volatile("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3v(float a, float b, float c) {
    float d;
    asm volatile("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2v(float x, float y) {  // x in the low half
    uint32_t r;
    if constexpr (std::is_same<T, bf16>::value)
        asm volatile("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    else
        asm volatile("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    return r;
}

// pack2v's r as fp32 again, and what it leaves of x and y, in the same type.
template <typename T>
__device__ __forceinline__ uint64_t both_f(uint32_t r) {
    if constexpr (std::is_same<T, bf16>::value) return pk(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
    T e[2];
    memcpy(e, &r, 4);
    return pk(to_f(e[0]), to_f(e[1]));
}
template <typename T>
__device__ __forceinline__ uint32_t rest2v(uint32_t r, float x, float y) {
    float a, b;
    upk(fma2v(both_f<T>(r), pk(-1.0f, -1.0f), pk(x, y)), a, b);
    return pack2v<T>(a, b);
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

// The waits that span a whole unit of work, which lasts as long as its keys are many: bounded by the clock, 20 seconds.  (A poll
// of mbar_wait_bounded takes some 4 us: 20 000 of them end after 80 ms, the time of some 4 million keys.)
__device__ __forceinline__ bool wait_unit(uint64_t* bar, uint32_t parity, int site, int* err) {
    uint64_t from = 0, now;
#pragma unroll 1
    while (!mbar_try_wait_suspend(bar, parity, 1000000u)) {
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
        if (from == 0) from = now;
        const bool late = now - from > 20000000000ull;
        if (late) atomicCAS(err, 0, site);
        // this wait or another gave up (an error of an earlier call stops no wait that goes on as it should)
        if (late || (now - from > 20000 && *reinterpret_cast<volatile int*>(err) != 0)) return false;
    }
    return true;
}

// A bounded wait whose answer is the same for the whole warp.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int site, int* err) {
    return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, site, err));
}

// One unit of work: up to 256 rows of a sequence and kv head against one split of its keys.
struct TcItem {
    int first, n;       // the sequence's first row in the batch and its rows (tokens)
    int r0, rows;       // the unit's rows among the sequence's n * group
    int len, table;     // the sequence's length, its block-table row
    int k_beg, k_stop;  // its keys
    int kh, z;          // kv head, split
    __device__ int tiles() const { return k_stop > k_beg ? (k_stop - k_beg + kTcTile - 1) / kTcTile : 0; }
    __device__ bool has(int t) const { return rows > t * kTcTile; }
};

// Cluster launch control: asks the hardware for a block of this grid that has not started yet, so that this one can
// do its work; the 16-byte answer completes on `bar`.
__device__ __forceinline__ void ask_next_block(uint4* answer, uint64_t* bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(smem_u32(answer)),
                 "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ bool next_block(const uint4* answer, int& x, int& y, int& z) {
    uint32_t got;
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b128 h;\n\tld.shared.b128 h, [%4];\n\t"
                 "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\tselp.u32 %0, 1, 0, p;\n\t"
                 "mov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t"
                 "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, %2, %3, _}, h;\n\t}"
                 : "=&r"(got), "=&r"(x), "=&r"(y), "=&r"(z)
                 : "r"(smem_u32(answer))
                 : "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // read before the next answer may be written
    return got != 0;
}

// Units of 256 rows -- pairs (token, query head of the group) -- of one sequence and kv head against its keys, 128 at
// a time, as two query tiles of 128 whose steps alternate on the tensor cores: while a tile's softmax runs, the
// other's products do.
//   warps 0-3, 4-7  softmax of tile 0, 1: a thread owns one row; scores from tensor memory, weights back to it over
//                   them as the A operand of the second product, and the output at the end
//   warp 8          loader: the block table's pages by TMA, one box per lane, into a ring of 128-key tiles;
//                   zeroes the values past a unit's last key
//   warp 9          issues S = Q K^T and O += P V
//   warp 10         finds the units: this block's own, then those of blocks that have not started
//   warp 11         puts rows right that met something not finite, behind their output: on the softmax warps the same code,
//                   though never run, cost their loop the registers for a tenth of the prompts' time
// Tensor memory: S0, S1 (128 columns each, P over their first 64, its low part over the rest), O0, O1.  The tensor pipe runs one thread's MMAs in
// order, so the S of the next key tile may follow the PV that still reads P, and a thread that has seen S complete
// knows that every earlier PV is complete too: it may rescale O without a barrier of its own.  Rescaling is rare: sums
// stay relative to a maximum that may be up to 2^8 behind (exact: p, l and O share it).  l sums the fp32 values of
// p.  For a 16-bit output p is rounded once to the operand type: that moves the output by 0.0006 of its norm in bf16, where its
// own rounding moves it by 0.0017, and a second part takes a quarter more time (the prompts below 356 us for 285).  An fp32
// output has no rounding to hide behind: there p enters the second product as two 16-bit parts (LOW; 305 us with one part and
// an error of 2^-9.6 of the norm, 356 with two and under 2^-13).
// Head dims below HD are zeros in shared memory: the tensor maps end there, and the queries are written so.  HD 256: one
// query tile a unit and a ring of two, so that a tile's softmax waits for its products and they for it; 4 prompts of 300
// tokens on 1000 keys 111 us, 0.2 PFLOP/s, where the MMA kernel takes 252.
// A block stays for many units (the grid is one block per unit; the running ones take over the rest): the loader and
// the first scores of a unit run ahead of the previous one's output, and tensor memory, barriers and shared memory are
// set up once.  Every wait is bounded and records the device error word.
// 6 causal prompts of 1500..4096 tokens, 16 query heads over 2 kv heads x 128, bf16 (279 GFLOP): 322 us over and over, 0.87
// PFLOP/s, when the power limit lowers the clocks; 289 us where a few calls follow one another.  (One block a unit, in the order of the batch,
// with a maximum before the weights: 380 us.)  Bound by the chain of a key tile: the softmax warps wait 1300 clocks for the
// scores, read them in 70, take 1450 for maximum, exponentials (at 16 a clock an SM alone 1024 for both tiles) and
// rounding, 220 to write the weights; a unit's output and next queries add 8500.  One or two tiles that fill the machine
// once (3 sequences of 40..64 tokens on 12 000 keys: 38 us) pay that start and end and the join for one short run.
template <typename T, int HD, bool LOW>
__global__ void __launch_bounds__(kTcThreads, 1) paged_tc_kernel(const __grid_constant__ PagedArgs p, const __grid_constant__ PagedMaps maps) {
    constexpr int TILE = kTcTileBytes<HD>, ST = kTcStages<HD>, TW = kTcTiles<HD>, ROWS = TW * kTcTile;
    static_assert(ST < 2 * kTcTails, "as many mended ends as the ring can hold");
    extern __shared__ uint8_t tc_raw[];
    __shared__ uint64_t bar[2 * ST + 3 * kTcItems + 10 + kTcTails];
    __shared__ uint4 answer;
    __shared__ TcItem items[kTcItems];
    __shared__ uint32_t again[kTcItems][8];  // by softmax warp: rows of a unit whose sums are not finite
    __shared__ uint32_t tmem_slot;
    uint64_t *full = bar, *empty = full + ST;                                // ring
    uint64_t *s_full = empty + ST, *p_full = s_full + 2;  // per query tile
    uint64_t *o_done = p_full + 2, *q_full = o_done + 2;
    uint64_t *item_full = q_full + 2, *item_empty = item_full + kTcItems, *tail = item_empty + kTcItems, *asked = tail + kTcTails, *begun = asked + 1, *written = begun + 1;
    const voxq_paged_attn& d = p.d;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, G = p.group;
    const uint32_t qsm = (smem_u32(tc_raw) + 1023) & ~1023u, ring = qsm + TW * TILE;

    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; i++) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(s_full + i, 1);
            mbar_init(p_full + i, 4);
            mbar_init(o_done + i, 1);
            mbar_init(q_full + i, 4);
        }
        for (int i = 0; i < kTcTails; i++) mbar_init(tail + i, 1);
        for (int i = 0; i < kTcItems; i++) {
            mbar_init(item_full + i, 1);
            mbar_init(item_empty + i, 11);  // every warp that works on units
            mbar_init(written + i, 8);
        }
        mbar_init(asked, 1);
        mbar_init(begun, 1);
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
    pdl_wait();
    pdl_launch_dependents();

    // The k-th unit; rows 0: no more.  done(k) frees its slot.
    auto unit_ready = [&](int k) {
        return __all_sync(0xffffffffu, wait_unit(item_full + k % kTcItems, (k / kTcItems) & 1, VOXQ_DEVERR_WAIT_FULL, p.err));
    };
    auto done = [&](int k) {
        __syncwarp();
        if (lane == 0) mbar_arrive(item_empty + k % kTcItems);
    };
    auto take = [&](int k, TcItem& it) {  // copied out, the slot freed at once
        const bool ok = unit_ready(k);
        it = items[k % kTcItems];
        done(k);
        if (!ok) it.rows = 0;
        return ok;
    };

    if (warp < 8) {
        // ---------------- softmax and output: one row a thread ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTcRegsSoftmax));
        const int t = warp >> 2, lr = threadIdx.x & 127;
        const uint32_t ts = tmem + ((uint32_t)((warp & 3) * 32) << 16) + t * kTcTile, to = tmem + ((uint32_t)((warp & 3) * 32) << 16) + 256 + t * HD;
        // The warp's 32 rows of queries, HD / 8 lanes a row so that every load covers whole lines, and their place in
        // shared memory: 16-byte chunk j of a 128-byte row at chunk j ^ (row & 7).
        constexpr int CPR = HD / 8, STEP = 32 / CPR;  // chunks of a row, rows of an access
        const int cj = lane % CPR, crow = lane / CPR;
        auto place = [&](int row, int j) {
            return qsm + t * TILE + (j / 8) * kTcHalf + ((warp & 3) * 32 + row) * 128 + (((j % 8) ^ (row & 7)) << 4);
        };
        auto load_q = [&](const TcItem& u) {
            const int row0 = t * kTcTile + (warp & 3) * 32 + crow, r = u.r0 + row0;
            int tok = r / G, h = r % G;
            constexpr int BATCH = CPR < 16 ? CPR : 16;
            uint4 v[BATCH];
#pragma unroll
            for (int i0 = 0; i0 < CPR; i0 += BATCH) {
#pragma unroll
                for (int i = 0; i < BATCH; i++) {
                    v[i] = make_uint4(0, 0, 0, 0);
                    if (row0 + (i0 + i) * STEP < u.rows && cj * 8 < d.head_dim)
                        v[i] = *reinterpret_cast<const uint4*>((const T*)d.q + (u.first + tok) * d.q_stride + (u.kh * G + h) * d.q_head_stride + cj * 8);
                    for (h += STEP; h >= G; h -= G) tok++;
                }
#pragma unroll
                for (int i = 0; i < BATCH; i++) sts128(place(crow + (i0 + i) * STEP, cj), v[i]);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full + t);
        };
        // (a unit's fields are read from shared memory where they are needed: the loop over its keys wants the registers)
        bool ok = unit_ready(0);
        uint32_t step = 0, unit = 0;
        if (ok && items[0].has(t) && items[0].tiles() > 0) load_q(items[0]);
        for (int k = 0; ok && items[k % kTcItems].rows > 0; k++) {
            const TcItem& it = items[k % kTcItems];
            const int tiles = it.has(t) ? it.tiles() : 0;
            const bool mine = t * kTcTile + lr < it.rows;
            const int vis = mine ? min(visible(p, it.len, it.n, (it.r0 + t * kTcTile + lr) / G), it.k_stop) : 0;
            // keys that every row of the tile sees need no mask
            const int all_see = min(visible(p, it.len, it.n, (it.r0 + t * kTcTile) / G), it.k_stop);
            int t0 = it.k_beg;
            float m = -INFINITY, l = 0.0f;  // m in base-2 units
            for (int i = 0; i < tiles; i++, t0 += kTcTile) {
                ok = warp_wait(s_full + t, step++ & 1, VOXQ_DEVERR_WAIT_MMA, p.err);
                if (!ok) break;
                tc_after();
                uint32_t sv[kTcTile], low[LOW ? kTcTile / 2 : 1];
                uint64_t sum[2];
                // The weights are taken relative to the maximum so far, while this tile's maximum is found beside them:
                // only if a row has outgrown its own by 2^8 are sums rescaled and the tile's weights computed again.
                while (true) {
#pragma unroll
                    for (int c = 0; c < kTcTile; c += 32) tm_ld32(ts + c, sv + c);
                    tm_wait_ld();
                    if (t0 + kTcTile > all_see) {
#pragma unroll
                        for (int c = 0; c < kTcTile; c++)
                            if (t0 + c >= vis) sv[c] = __float_as_uint(-INFINITY);
                    }
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    auto row_max = [&](int c) {  // of 16 scores
#pragma unroll
                        for (int e = 0; e < 16; e += 8)
#pragma unroll
                            for (int j = 0; j < 4; j++) mx[j] = fmaxf(fmaxf(mx[j], __uint_as_float(sv[c + e + j])), __uint_as_float(sv[c + e + j + 4]));
                    };
                    auto top = [&] { return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale2; };
                    if (i == 0) {
#pragma unroll
                        for (int c = 0; c < kTcTile; c += 16) row_max(c);
                        m = top();
                    }
                    const float neg = m == -INFINITY ? 0.0f : -m;  // no key so far: every weight is ex2(-inf) = 0
                    const uint64_t sc2 = pk(p.scale2, p.scale2), ng2 = pk(neg, neg);
                    sum[0] = sum[1] = pk(0.0f, 0.0f);
                    // One pair of exponentials after the other, the scaling of a later pair and the sums and rounding of an
                    // earlier one between them: a lone warp keeps its special-function unit busy only if nothing else
                    // is issued in a bunch.
                    constexpr int AHEAD = 3, BEHIND = 3;
                    uint64_t x[kTcTile / 2];
                    float y[kTcTile];
                    auto scaled = [&](int c) { x[c] = fma2v(pk(__uint_as_float(sv[2 * c]), __uint_as_float(sv[2 * c + 1])), sc2, ng2); };
#pragma unroll
                    for (int c = 0; c < AHEAD; c++) scaled(c);
#pragma unroll
                    for (int c = 0; c < kTcTile / 2 + BEHIND; c++) {
                        if (c < kTcTile / 2) {
                            upk(x[c], y[2 * c], y[2 * c + 1]);
                            y[2 * c] = ex2v(y[2 * c]);
                        }
                        if (c + AHEAD < kTcTile / 2) scaled(c + AHEAD);
                        if (c < kTcTile / 2) {
                            mx[c & 3] = max3v(mx[c & 3], __uint_as_float(sv[2 * c]), __uint_as_float(sv[2 * c + 1]));
                            y[2 * c + 1] = ex2v(y[2 * c + 1]);
                        }
                        if (c >= BEHIND) {
                            const int o = c - BEHIND;
                            if (!LOW) sum[o & 1] = add2v(sum[o & 1], pk(y[2 * o], y[2 * o + 1]));
                            sv[o] = pack2v<T>(y[2 * o], y[2 * o + 1]);  // (over scores that are done with)
                            if (LOW) {
                                low[o] = rest2v<T>(sv[o], y[2 * o], y[2 * o + 1]);
                                sum[o & 1] = add2v(sum[o & 1], pk(y[2 * o], y[2 * o + 1]));
                            }
                        }
                    }
                    const float mt = top();
                    const bool grow = mt > m + kTcSlack;
                    if (!__any_sync(0xffffffffu, grow)) break;
                    const float f = grow ? ex2(m - mt) : 1.0f;
                    if (grow) m = mt;
                    l *= f;
#pragma unroll
                    for (int c = 0; c < HD; c += 32) {  // (i > 0: the first tile's weights are relative to its own maximum)
                        uint32_t o[32];
                        tm_ld32(to + c, o);
                        tm_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tm_st32(to + c, o);
                    }
                }
                tm_st32(ts, sv);
                tm_st32(ts + 32, sv + 32);
                if (LOW) {
                    tm_st32(ts + 64, low);
                    tm_st32(ts + 96, low + 32);
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
            // The next unit's queries start their way (into L2) while the last product runs.  Their buffer is free (this
            // unit's last scores are complete): it first takes the output, so that rows leave in whole lines, then them.
            ok = ok && unit_ready(k + 1);
            const TcItem& next = items[(k + 1) % kTcItems];
            const bool more = ok && next.has(t) && next.tiles() > 0;
            if (more && t * kTcTile + lr < next.rows) {
                const int r = next.r0 + t * kTcTile + lr;
                const T* src = (const T*)d.q + (next.first + r / G) * d.q_stride + (next.kh * G + r % G) * d.q_head_stride;
#pragma unroll
                for (int c = 0; c < HD; c += 64)
                    if (c < d.head_dim) asm volatile("prefetch.global.L2 [%0];" ::"l"(src + c));
            }
            if (ok && tiles > 0) {
                ok = warp_wait(o_done + t, unit++ & 1, VOXQ_DEVERR_WAIT_MMA, p.err);
                tc_after();
            }
            uint32_t rows_again = 0;
            if (it.has(t)) {
                const int r = it.r0 + t * kTcTile + lr, tok = r / G, h = it.kh * G + r % G;
                const int seen = mine ? visible(p, it.len, it.n, tok) : 0;
                const bool whole = seen <= p.split_len;
                // a row with more keys than a split holds leaves a record, one with fewer is split 0's
                const bool put = ok && mine && (whole ? it.z == 0 : it.k_beg < seen);
                const float inv = !whole ? 1.0f : seen > 0 ? 1.0f / l : 0.0f;
                const int64_t rec = ((int64_t)(it.first + tok) * d.heads + h) * p.splits + it.z;
                if (put && !whole) p.ml[rec] = make_float2(m, l);
                const int64_t dst = whole ? (it.first + tok) * d.o_stride + h * d.o_head_stride : rec * d.head_dim;
                const int kind = !put ? 0 : whole ? 1 : 2;
                // 16-bit rows of the output at once, fp32 ones (records, or an fp32 output) in two halves of the head
                const bool fast = d.out_dtype != VOXQ_F32 && __all_sync(0xffffffffu, kind < 2);
                float chk[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
                for (int part = 0; part < (fast ? 1 : 2); part++) {
#pragma unroll 1
                    for (int c = 0; c < (fast ? HD : HD / 2); c += 32) {
                        uint32_t o[32];
                        if (tiles > 0) {
                            tm_ld32(to + part * (HD / 2) + c, o);
                            tm_wait_ld();
                        }
                        if (seen > 0 && tiles > 0)
#pragma unroll
                            for (int e = 0; e < 32; e++) chk[e & 3] = fmaf(__uint_as_float(o[e]), 0.0f, chk[e & 3]);
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = seen > 0 ? __float_as_uint(__uint_as_float(o[e]) * inv) : 0u;
                        if (fast) {
#pragma unroll
                            for (int e = 0; e < 16; e++) o[e] = pack2<T>(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]));
                        }
                        const int chunk = fast ? c / 8 : c / 4;
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            if (e < 4 || !fast)
                                sts128(place(lane, chunk + e), make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]));
                    }
                    __syncwarp();
#pragma unroll 4
                    for (int i = 0; i < CPR; i++) {
                        const int row = crow + i * STEP, what = __shfl_sync(0xffffffffu, kind, row);
                        const int64_t at = __shfl_sync(0xffffffffu, dst, row);
                        const uint4 v = lds128(place(row, cj));
                        if (what == 0 || part * (HD / 2) + cj * (fast ? 8 : 4) >= d.head_dim) continue;
                        if (fast) {
                            *reinterpret_cast<uint4*>((T*)d.out + at + cj * 8) = v;
                        } else {
                            const int64_t x = at + part * (HD / 2) + cj * 4;
                            if (what == 2) *reinterpret_cast<uint4*>(p.acc + x) = v;
                            else if (d.out_dtype == VOXQ_F32) *reinterpret_cast<uint4*>((float*)d.out + x) = v;
                            else *reinterpret_cast<uint2*>((T*)d.out + x) = make_uint2(pack2<T>(__uint_as_float(v.x), __uint_as_float(v.y)), pack2<T>(__uint_as_float(v.z), __uint_as_float(v.w)));
                        }
                    }
                    __syncwarp();
                }
                rows_again = __ballot_sync(0xffffffffu, put && not_finite<T>((chk[0] + chk[1]) + (chk[2] + chk[3]), l));
            }
            if (lane == 0) again[k % kTcItems][warp] = rows_again;
            __syncwarp();
            if (lane == 0) mbar_arrive(written + k % kTcItems);
            if (more) load_q(next);
            tc_before();  // the output is read before the next unit's first product may overwrite it (p_full)
            done(k);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTcRegsOther));
        if (warp == 8) {
            // ---------------- loader: K0, V0, K1, V1, ... of every unit ----------------
            const int R = maps.box_rows, boxes = kTcTile / R * (HD / 64);
            TcItem it;
            bool ok = true;
            uint32_t c = 0, tails = 0;  // tiles loaded; units whose last tile was mended
            for (int k = 0; ok; k++) {
                ok = take(k, it);
                if (lane == 0) mbar_arrive(begun);
                if (it.rows == 0) break;
                const int32_t* table = d.block_table + (int64_t)it.table * d.table_stride;
                const int loads = 2 * it.tiles();
                for (int i = 0; i < loads; i++, c++) {
                    const int slot = c % ST, t0 = it.k_beg + i / 2 * kTcTile;
                    if (c >= ST) ok = warp_wait(empty + slot, (c / ST - 1) & 1, VOXQ_DEVERR_WAIT_EMPTY, p.err);
                    if (!ok) break;
                    // boxes that start before k_stop; the rest of the tile is masked
                    const int live = (min(it.k_stop - t0, kTcTile) + R - 1) / R * (HD / 64);
                    if (lane == 0) mbar_arrive_expect_tx(full + slot, live * R * 128);
                    __syncwarp();
                    for (int b = lane; b < boxes; b += 32) {
                        const int half = b % (HD / 64), row = b / (HD / 64) * R, key = t0 + row;
                        if (key >= it.k_stop) continue;
                        const int e = p.page_shift >= 0 ? key >> p.page_shift : (int)((uint32_t)key / (uint32_t)d.page_size);
                        int page = __ldg(table + e);
                        if ((uint32_t)page >= (uint32_t)d.pages) page = 0;
                        const int off = key - e * d.page_size;
                        tma_page(ring + slot * TILE + half * kTcHalf + row * 128, maps, i & 1 ? &maps.v : &maps.k, half * 64, off, it.kh, page, full + slot);
                    }
                }
                const int odd = (it.k_stop - it.k_beg) % 16;
                if (ok && loads > 0 && odd) {
                    // The last 16 keys that enter the second product: what lies past the end may be anything, and
                    // 0 * NaN is NaN, so those rows become zeros.
                    const int slot = (c - 1) % ST, valid = (it.k_stop - it.k_beg) % kTcTile;
                    ok = warp_wait(full + slot, ((c - 1) / ST) & 1, VOXQ_DEVERR_WAIT_FULL, p.err);
                    for (int j = lane; ok && j < (16 - odd) * (HD / 8); j += 32) {
                        const int row = valid + j / (HD / 8), ch = j % (HD / 8);
                        sts128(ring + slot * TILE + (ch / 8) * kTcHalf + row * 128 + (ch % 8) * 16, make_uint4(0, 0, 0, 0));
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(tail + tails % kTcTails);
                    tails++;
                }
            }
            if (!ok)  // nothing of this block may still be writing its shared memory when it ends
                for (uint32_t i = c > ST ? c - ST : 0; i < c; i++) mbar_wait_bounded(full + i % ST, (i / ST) & 1, VOXQ_DEVERR_NONE, p.err);
        } else if (warp == 9) {
            // ---------------- MMA issue ----------------
            // One thread, operands in uniform registers, few instructions between a barrier and the MMAs that wait for
            // it: they are on the chain of both tiles.  The strict order tile 0, tile 1 keeps the tiles' softmaxes half
            // a period apart: with an issuing warp for each they fell into step, computed their exponentials at the
            // same time and left the tensor pipe idle meanwhile (403 us where this order took 305).
            constexpr uint32_t id_s = tc_idesc<T>(kTcTile, false), id_o = tc_idesc<T>(HD, true);
            const bool one = elect_one();
            TcItem it;
            bool ok = true;
            uint32_t slot = 0, phase = 0, steps_done[2] = {0, 0}, units[2] = {0, 0}, tails = 0;
            auto ready = [&] { return mbar_wait_bounded(full + slot, phase, VOXQ_DEVERR_WAIT_FULL, p.err); };
            auto advance = [&] {
                slot = slot + 1 == ST ? 0 : slot + 1;
                phase ^= slot == 0;
            };
            auto scores = [&](int t, uint32_t sl) {
                const uint64_t qd = desc_k(qsm + t * TILE), kd = desc_k(ring + sl * TILE);
#pragma unroll
                for (int k = 0; k < HD / 16; k++) {
                    const uint32_t off = ((k / 4) * kTcHalf + (k % 4) * 32) >> 4;
                    mma_ss(tmem + t * kTcTile, qd + off, kd + off, id_s, k > 0);
                }
                tc_commit(s_full + t);
            };
            for (int k = 0; ok; k++) {
                ok = take(k, it);
                if (it.rows == 0) break;
                const int tiles = it.tiles();
                if (tiles == 0) continue;
                const bool two = it.has(1);
                if (one) {
                    const int keys = it.k_stop - it.k_beg, odd = keys % 16;
                    // K(0), then what the first step needs
                    ok = ready();
                    uint32_t sk = slot;
                    advance();
#pragma unroll
                    for (int t = 0; t < TW; t++) {
                        if (t && !two) break;
                        ok = ok && wait_unit(q_full + t, units[t]++ & 1, VOXQ_DEVERR_WAIT_FULL, p.err);
                        tc_after();
                        if (ok) scores(t, sk);
                    }
                    if (ok) tc_commit(empty + sk);
                    uint32_t sv = 0;
                    // V(i) and, before the last, K(i + 1)
                    auto fetch = [&](bool more) {
                        ok = ok && ready();
                        sv = slot;
                        advance();
                        if (more) {
                            ok = ok && ready();
                            sk = slot;
                            advance();
                        } else if (odd) {
                            ok = ok && mbar_wait_bounded(tail + tails % kTcTails, (tails / kTcTails) & 1, VOXQ_DEVERR_WAIT_FULL, p.err);
                            tails++;
                        }
                    };
                    fetch(tiles > 1);
                    for (int i = 0; i < tiles && ok; i++) {
                        const bool more = i + 1 < tiles;
                        const int steps = more ? kTcTile / 16 : (keys - i * kTcTile + 15) / 16;
                        const uint64_t vd = desc_mn(ring + sv * TILE);
                        const uint32_t now_v = sv, now_k = sk;
#pragma unroll
                        for (int t = 0; t < TW; t++) {
                            if (t && !two) break;
                            ok = ok && mbar_wait_bounded(p_full + t, steps_done[t]++ & 1, VOXQ_DEVERR_WAIT_MMA, p.err);
                            tc_after();
                            if (!ok) break;
#pragma unroll
                            for (int j = 0; j < kTcTile / 16; j++)
                                if (j < steps) {
                                    const uint32_t pt = tmem + t * kTcTile + j * 8;
                                    if (LOW) mma_ts(tmem + 256 + t * HD, pt + kTcTile / 2, vd + (j * 2048 >> 4), id_o, i > 0 || j > 0);
                                    mma_ts(tmem + 256 + t * HD, pt, vd + (j * 2048 >> 4), id_o, LOW || i > 0 || j > 0);
                                }
                            if (more) {
                                scores(t, now_k);
                            } else {
                                if (t == (two ? 1 : 0)) tc_commit(empty + now_v);
                                tc_commit(o_done + t);
                            }
                            if (TW > 1 && t == 0 && more) fetch(i + 2 < tiles);  // the next step's tiles, while tile 1's softmax works
                        }
                        if (!ok || !more) break;
                        tc_commit(empty + now_v);
                        tc_commit(empty + now_k);
                        if (TW == 1) fetch(i + 2 < tiles);  // (into the slots that are being freed)
                    }
                }
                ok = __all_sync(0xffffffffu, ok);
            }
        } else if (warp == 10) {
            // ---------------- units ----------------
            int x = blockIdx.x, y, z = blockIdx.z, k = 0;
            bool ok = true;
            auto put = [&](const TcItem& it) {
                if (k >= kTcItems) ok = __all_sync(0xffffffffu, wait_unit(item_empty + k % kTcItems, (k / kTcItems - 1) & 1, VOXQ_DEVERR_WAIT_EMPTY, p.err));
                if (lane == 0 && ok) {
                    items[k % kTcItems] = it;
                    mbar_arrive(item_full + k % kTcItems);
                }
                __syncwarp();
                k++;
            };
            // Sequences j * 32 + lane: units, length, rows (kept for the search below).
            const bool sorted = d.batch <= 32 * kTcSeqs;
            int seq_units[kTcSeqs], seq_len[kTcSeqs], seq_past[kTcSeqs];
#pragma unroll
            for (int j = 0; j < kTcSeqs; j++) {
                const int i = j * 32 + lane;
                const bool in = sorted && i < d.batch;
                const int first = in ? __ldg(d.cu_q + i) : 0, n = in ? min(__ldg(d.cu_q + i + 1), d.total_q) - first : 0;
                seq_units[j] = first >= 0 && n > 0 ? (n * G + ROWS - 1) / ROWS : 0;
                seq_len[j] = in ? min(max(__ldg(d.kv_len + i), 0), d.max_kv) : 0;
                seq_past[j] = seq_len[j] - n;
            }
            // Units of this lane's j-th sequence, and of all, whose last visible key is past the v-th.
            auto above_of = [&](int j, int v) {
                if (v < 0) return seq_units[j];
                if (seq_len[j] <= v || seq_units[j] == 0) return 0;
                if (!d.causal) return seq_units[j];
                // all but the last unit end on a multiple of ROWS rows: unit r is past v from (v - past) * G / ROWS on
                return 1 + min(max(seq_units[j] - 1 - (int)((int64_t)max(v - seq_past[j], 0) * G / ROWS), 0), max(seq_units[j] - 1, 0));
            };
            auto above = [&](int v) {
                int c = 0;
#pragma unroll
                for (int j = 0; j < kTcSeqs; j++) c += above_of(j, v);
                return __reduce_add_sync(0xffffffffu, c);
            };
            TcItem it;
            for (uint32_t a = 0; ok; a++) {
                const int kh = x % d.kv_heads, nth = x / d.kv_heads;
                int s = -1, r = 0;
                if (sorted) {
                    // The nth unit in falling order of the last key it sees, without sorting: the value v with (units
                    // above v) <= nth < (units from v on), then the sequence among those that have units at v.
                    int lo = 0, hi = d.max_kv;
                    while (lo < hi) {
                        const int mid = (lo + hi) / 2;
                        if (above(mid) <= nth) hi = mid;
                        else lo = mid + 1;
                    }
                    int left = nth - above(lo);
#pragma unroll
                    for (int j = 0; j < kTcSeqs; j++) {
                        const int more = above_of(j, lo), at = above_of(j, lo - 1) - more;
                        int sum = at;  // inclusive prefix sum over the lanes
#pragma unroll
                        for (int o = 1; o < 32; o *= 2) {
                            const int v = __shfl_up_sync(0xffffffffu, sum, o);
                            if (lane >= o) sum += v;
                        }
                        const uint32_t hit = __ballot_sync(0xffffffffu, left < sum && left >= sum - at);
                        if (s < 0 && hit) {
                            const int from = __ffs(hit) - 1;
                            s = j * 32 + from;
                            r = __shfl_sync(0xffffffffu, seq_units[j] - 1 - more - (left - (sum - at)), from);
                        }
                        left -= __shfl_sync(0xffffffffu, sum, 31);
                    }
                } else {
                    // many sequences: in the order of the batch, the last rows of each first
                    const int tile = gridDim.x / d.kv_heads - 1 - nth;
                    for (int i0 = 0; i0 < d.batch; i0 += 32) {
                        const int i = i0 + lane;
                        s += __popc(__ballot_sync(0xffffffffu, i < d.batch && __ldg(d.cu_q + i) * G / ROWS + i <= tile));
                    }
                    s = max(s, 0);
                    r = tile - (__ldg(d.cu_q + s) * G / ROWS + s);
                }
                it.table = max(s, 0);
                it.first = __ldg(d.cu_q + it.table);
                it.n = s < 0 ? 0 : min(__ldg(d.cu_q + s + 1), d.total_q) - it.first;
                it.r0 = r * ROWS;
                it.rows = min(it.n * G - it.r0, ROWS);
                it.len = min(max(__ldg(d.kv_len + it.table), 0), d.max_kv);
                it.kh = kh;
                it.z = z;
                if (it.first >= 0 && it.n > 0 && it.r0 >= 0 && it.rows > 0) {
                    const int k_end = visible(p, it.len, it.n, (it.r0 + it.rows - 1) / G);
                    it.k_beg = z * p.split_len;
                    it.k_stop = min(k_end, it.k_beg + p.split_len);
                    if (it.k_beg < k_end || z == 0) {
                        put(it);
                        // No unit is taken before the loader has come to this one: a block that reserved more would sit on
                        // them while others run out of work.
                        ok = ok && __all_sync(0xffffffffu, wait_unit(begun, (k - 1) & 1, VOXQ_DEVERR_WAIT_EMPTY, p.err));
                        if (!ok) break;
                    }
                }
                if (lane == 0) {
                    mbar_arrive_expect_tx(asked, 16);
                    ask_next_block(&answer, asked);
                }
                const bool answered = warp_wait(asked, a & 1, VOXQ_DEVERR_WAIT_FULL, p.err);
                ok = ok && answered;
                if (!ok || !next_block(&answer, x, y, z)) break;
                __syncwarp();
            }
            it.rows = 0;
            if (ok) put(it);
        } else {
            // ---------------- rows to put right: none, as a rule ----------------
            // (the kernel's last code: between the others' it took 10 us more from cold caches)
            for (int k = 0; unit_ready(k) && items[k % kTcItems].rows > 0; k++) {
                const TcItem& it = items[k % kTcItems];
                if (!__all_sync(0xffffffffu, wait_unit(written + k % kTcItems, (k / kTcItems) & 1, VOXQ_DEVERR_WAIT_FULL, p.err))) break;
                RowsAgain<T> found(it.k_beg);
                for (int w = 0; w < 8; w++)
                    for (uint32_t rows = again[k % kTcItems][w]; rows; rows &= rows - 1) {
                        const int r = it.r0 + w * 32 + __ffs(rows) - 1, seen = visible(p, it.len, it.n, r / G);
                        const int64_t rec = ((int64_t)(it.first + r / G) * d.heads + it.kh * G + r % G) * p.splits + it.z;
                        found.row(p, it.table, it.first, r, it.kh, it.k_beg, min(seen, it.k_stop), seen <= p.split_len ? -1 : rec, true);
                    }
                done(k);
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

bool paged_maps_take(const voxq_paged_attn& d) {
    const int64_t lim = (int64_t)1 << 38;  // elements: a tensor map's strides are below 2^40 bytes
    return d.page_size > 0 && d.page_size % 8 == 0 && d.pages > 0 && d.page_stride > 0 && d.row_stride > 0 && d.head_stride > 0 &&
           d.page_stride < lim && d.row_stride < lim && d.head_stride < lim;
}

VoxCPMError paged_maps(const voxq_paged_attn& d, int max_rows, PagedMaps* m) {
    EncodeTiled enc = encode_tiled();
    if (!enc) return VOXCPM_ERR_INTERNAL;
    const int e = elem_bytes(d.dtype);
    m->box_rows = d.page_size & -d.page_size;
    if (m->box_rows > max_rows) m->box_rows = max_rows;
    m->head_first = d.head_stride <= d.row_stride;
    const int hi = m->head_first ? 1 : 2, ri = 3 - hi;
    cuuint64_t dims[4] = {(cuuint64_t)d.head_dim, 0, 0, (cuuint64_t)d.pages}, strides[3] = {0, 0, (cuuint64_t)d.page_stride * e};
    cuuint32_t box[4] = {(cuuint32_t)(128 / e), 1, 1, 1}, one[4] = {1, 1, 1, 1};
    dims[hi] = (cuuint64_t)d.kv_heads;
    dims[ri] = (cuuint64_t)d.page_size;
    strides[hi - 1] = (cuuint64_t)d.head_stride * e;
    strides[ri - 1] = (cuuint64_t)d.row_stride * e;
    box[ri] = (cuuint32_t)m->box_rows;
    const CUtensorMapDataType dt = d.dtype == VOXQ_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : d.dtype == VOXQ_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    for (int i = 0; i < 2; i++)
        if (enc(i ? &m->v : &m->k, dt, 4, const_cast<void*>(i ? d.v : d.k), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return VOXCPM_ERR_UNSUPPORTED;
    return VOXCPM_SUCCESS;
}

int paged_tc_rows(const voxq_paged_attn& d) { return kTcTile * (d.head_dim > 128 ? kTcTiles<256> : kTcTiles<128>); }

bool paged_tc_takes(const voxq_paged_attn& d) {
    return d.dtype != VOXQ_F32 && d.scale >= 0.0f && paged_maps_take(d);
}

template <typename T, int HD, bool LOW>
static VoxCPMError tc_launch(const PagedArgs& a, cudaStream_t st) {
    auto kern = paged_tc_kernel<T, HD, LOW>;
    static std::atomic<uint64_t> asked{0};
    VOXQ_CUDA_TRY(allow_shared((const void*)kern, kTcSmem<HD>, asked));
    const voxq_paged_attn& d = a.d;
    PagedMaps m;
    const VoxCPMError e = paged_maps(d, kTcTile, &m);
    if (e != VOXCPM_SUCCESS) return e;
    // a block for every unit there can be (the search of many sequences numbers one more a sequence)
    const int rows = paged_tc_rows(d);
    const dim3 grid(d.batch <= 32 * kTcSeqs ? (int)paged_tiles(d, rows) : ((int)((int64_t)d.total_q * a.group / rows) + d.batch) * d.kv_heads, 1, a.splits);
    VOXQ_CUDA_TRY(launch_pdl(kern, grid, dim3(kTcThreads), kTcSmem<HD>, st, a, m));
    return VOXCPM_SUCCESS;
}

template <typename T, int HD>
static VoxCPMError tc_launch(const PagedArgs& a, cudaStream_t st) {
    return a.d.out_dtype == VOXQ_F32 ? tc_launch<T, HD, true>(a, st) : tc_launch<T, HD, false>(a, st);
}

VoxCPMError paged_tc_launch(const PagedArgs& a, cudaStream_t st) {
    const int hd = a.d.head_dim;
    if (a.d.dtype == VOXQ_F16) return hd <= 64 ? tc_launch<__half, 64>(a, st) : hd <= 128 ? tc_launch<__half, 128>(a, st) : tc_launch<__half, 256>(a, st);
    return hd <= 64 ? tc_launch<bf16, 64>(a, st) : hd <= 128 ? tc_launch<bf16, 128>(a, st) : tc_launch<bf16, 256>(a, st);
}

}  // namespace voxq
