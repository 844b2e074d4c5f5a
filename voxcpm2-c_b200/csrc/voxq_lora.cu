// voxq_lora.cu -- low-rank adapters of many requests beside a shared projection.
#include <algorithm>
#include <type_traits>

#include "voxq_batch.cuh"
#include "voxq_internal.h"

namespace voxq {

constexpr int kLoraThreads = 128;
constexpr int kLoraWarps = kLoraThreads / 32;
constexpr int kLoraMaxRank = 128;

// Shape of the kernel for x of type T, weights of type W, TM rows a tile and NB output columns a step.
template <typename T, typename W, int TM, int COLS>
struct LoraShape {
    static constexpr int WM = TM / 16;                // warps along the rows
    static constexpr int WK = kLoraWarps / WM;        // warps along K (first product) or the columns (second)
    static constexpr int KB = is_f32<W> || TM == 64 ? 64 : 128;  // K per stage: four blocks of TM 64 share an SM
    static constexpr int NB = COLS;
    static constexpr int NW = NB / WK;                // of a warp
    static constexpr int XP = KB + 16 / sizeof(T);    // shared pitches: 16 bytes more than a row, so that the 8 rows
    static constexpr int AP = KB + 16 / sizeof(W);    // of a fragment load lie in different banks
    int Rp, stage, hp, bp;                            // rank in steps of 16; bytes of a stage; pitches of h and B
    int o_hpart, o_hs, o_b0, o_b1, bytes;      // byte offsets
    __host__ __device__ explicit LoraShape(int rank) {
        Rp = (rank + 15) / 16 * 16;
        stage = TM * XP * (int)sizeof(T) + Rp * AP * (int)sizeof(W);
        hp = Rp + 8;
        bp = Rp + 16 / (int)sizeof(W);
        // the stages are free once the first product is done: the second
        // buffer of B lives there
        const int bbytes = NB * bp * (int)sizeof(W);
        o_b1 = 0;
        const int low = 2 * stage > bbytes ? 2 * stage : bbytes;
        o_hpart = (low + 15) / 16 * 16;
        o_hs = o_hpart + WK * TM * hp * 4;
        o_b0 = o_hs + TM * hp * 4;  // fp32, or two 16-bit parts
        bytes = o_b0 + bbytes;
    }
};

// d[i] += a b[i]^T over 16 of the inner dimension, the 16 x 16 a at `as` and NBLK 8-row blocks of b at `bs`, both in
// shared memory with the inner dimension contiguous.  16-bit: one MMA per block (and one more for a's low part at
// as_lo).  fp32: TF32 MMAs on a's high and low parts and, for fp32 weights, on b's; a 16-bit weight is a TF32 value.
template <typename T, typename W, int NBLK, bool LOW>
__device__ __forceinline__ void mul_16(float (*d)[4], const T* as, const T* as_lo, int ap, const W* bs, int bp, int blocks) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if constexpr (!is_f32<T>) {
        uint32_t a[4], al[4];
        const int off = (lane & 15) * ap + (lane >> 4) * 8;
        ldsm4(a, smem_u32(as + off));
        if (LOW) ldsm4(al, smem_u32(as_lo + off));
        const int boff = ((lane & 7) + (lane >> 4) * 8) * bp + ((lane >> 3) & 1) * 8;
#pragma unroll
        for (int i = 0; i < NBLK; i += 2) {
            if (i >= blocks) break;
            uint32_t b[4];
            ldsm4(b, smem_u32(bs + i * 8 * bp + boff));
            if (LOW) {
                mma16<T>(d[i], al, b[0], b[1]);
                mma16<T>(d[i + 1], al, b[2], b[3]);
            }
            mma16<T>(d[i], a, b[0], b[1]);
            mma16<T>(d[i + 1], a, b[2], b[3]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 16; k += 8) {
            uint32_t ah[4], al[4];
            split_tf32(as[g * ap + k + t], ah[0], al[0]);
            split_tf32(as[(g + 8) * ap + k + t], ah[1], al[1]);
            split_tf32(as[g * ap + k + t + 4], ah[2], al[2]);
            split_tf32(as[(g + 8) * ap + k + t + 4], ah[3], al[3]);
#pragma unroll
            for (int i = 0; i < NBLK; i++) {
                if (i >= blocks) break;
                const W* br = bs + (i * 8 + g) * bp + k + t;
                uint32_t bh[2], bl[2];
                if constexpr (is_f32<W>) {
                    split_tf32(br[0], bh[0], bl[0]);
                    split_tf32(br[4], bh[1], bl[1]);
                } else {  // as it is: rounding would carry a NaN of nothing but ones over into a zero
                    bh[0] = __float_as_uint(to_f(br[0]));
                    bh[1] = __float_as_uint(to_f(br[4]));
                }
                mma8(d[i], al, bh[0], bh[1]);
                if (is_f32<W>) mma8(d[i], ah, bl[0], bl[1]);
                mma8(d[i], ah, bh[0], bh[1]);
            }
        }
    }
}

// NB columns of B[w] from n0 on, [column][rank], to shared memory; zeros past N and past the adapter's own rank r (what
// lies there may be anything).  Within a warp's NW columns, column c goes to row (c % CW / 2) * 8 + 2 (c / CW) + c % 2
// with CW = NW / 4: the columns that a thread gets from the MMAs -- 2 t and 2 t + 1 of every block of 8 rows -- are then
// CW neighbours of the output, and base and out move straight between memory and the accumulators.  per: 16-byte vectors
// of a column, inv: 2^20 / per rounded up.
template <typename W, int NB, int NW>
__device__ __forceinline__ void load_b(W* dst, int bp, const W* b, int n0, int N, int rank, int r, int per, uint32_t inv) {
    constexpr int E = 16 / sizeof(W);
    for (int i = threadIdx.x; i < NB * per; i += kLoraThreads) {
        constexpr int CW = NW / 4;
        const int row = (uint32_t)i * inv >> 20, c = (i - row * per) * E, in = row % NW;
        const int to = row - in + in % CW / 2 * 8 + in / CW * 2 + in % 2;
        const bool ok = n0 + row < N && c < r;
        const W* src = b + (ok ? (int64_t)(n0 + row) * rank + c : 0);
        if (ok && c + E > r) {  // the adapter's rank ends inside these 16 bytes
            uint4 v = *reinterpret_cast<const uint4*>(src);
            W e[E];
            memcpy(e, &v, 16);
#pragma unroll
            for (int j = 0; j < E; j++)
                if (c + j >= r) e[j] = from_f<W>(0.0f);
            memcpy(&v, e, 16);
            *reinterpret_cast<uint4*>(dst + to * bp + c) = v;
        } else {
            cp_async16_or_zero(dst + to * bp + c, src, ok);
        }
    }
}

// A sum that products in two TF32 parts did not leave finite, once more in plain fp32: the parts of an infinity, or of an fp32
// value that rounds to one, make a NaN (inf - inf, 0 * inf).  What is not finite here is so by the formula.  x and a are rows of
// whole fours, a's past K whatever they may be.  (An infinity in B meets h's parts in every column step; looking for it there
// took the prompts 13 % more time in bf16 and 7 % in fp32.)
template <typename W>
__device__ __forceinline__ float plain_sum(const float* x, const W* a, int K) {
    float v = 0.0f;
#pragma unroll 1
    for (int k = 0; k < K && v == v; k += 4) {
        float p[4], w[4];
        load4(p, x + k);
        load4(w, a + k);
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (k + e < K) v = fmaf(p[e], w[e], v);
    }
    return v;
}

// One cluster per tile of up to TM rows of one request, both products in one
// launch.  The CTAs of the cluster split K for h = x A^T (chunks of KB, two
// cp.async stages), add their partial sums of h through each other's shared
// memory in rank order, and split the columns for out = base + scale h B^T.
// The traffic is x, base, out and the weights once: bound by HBM for prompts
// and by the latency of one chain (tile, x and A, cluster barrier, store) for
// single tokens, so the first columns of B are already on their way during
// the first product.  TM 16 puts the four warps along K and the columns (a
// step's tile has one row), TM 64 along the rows.  Both sums are fp32; h
// enters the second product unrounded to 16 significant bits or more (two
// 16-bit parts, or TF32 parts), because a 16-bit h would cost as much accuracy
// as the output's own rounding.
// 40 single fp32 rows, K = N = 2048, rank 16: 8.2 us (19 with a block a row and no cluster).  9 bf16 prompts, 8000 rows, K
// 1024, N 4096, ranks up to 32: 42 us, 2.7 TB/s, against 17 at HBM's rate: 17 000 clocks to h, then 3500 a column
// step of a block (wait for B, the products, base, store), which four blocks an SM overlap only in part; a deeper
// prefetch of B or base gained nothing.
template <typename T, typename W, int TM, int RB, int COLS>
__global__ void __launch_bounds__(kLoraThreads) lora_kernel(const __grid_constant__ voxq_lora d) {
    using S = LoraShape<T, W, TM, COLS>;
    constexpr int WM = S::WM, WK = S::WK, KB = S::KB, NB = S::NB, NW = S::NW;
    extern __shared__ __align__(16) uint8_t lora_sh[];
    const S z(d.rank);
    uint32_t crank, csize;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(crank));
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(csize));
    const int tile = blockIdx.x / csize;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wm = warp % WM, wk = warp / WM;
    pdl_wait();
    pdl_launch_dependents();

    const int s = tile_owner<TM>(d.cu, d.batch, 1, tile);
    const int first = __ldg(d.cu + s), m0 = first + (tile - (first / TM + s)) * TM;
    const int rows = min(min(__ldg(d.cu + s + 1), d.rows) - m0, TM);
    if (rows <= 0 || m0 < 0) return;  // the whole cluster
    const int w = __ldg(d.adapter + s);
    const bool on = w >= 0 && w < d.adapters;
    const int r = !on ? 0 : d.ranks ? min(max(__ldg(d.ranks + w), 0), d.rank) : d.rank;
    const W* wa = (const W*)d.a + (int64_t)w * d.rank * d.K;
    const W* wb = (const W*)d.b + (int64_t)w * d.N * d.rank;
    const int blocks = (r + 7) / 8, inner = (r + 15) / 16;
    const int per = z.Rp / (16 / (int)sizeof(W));
    const uint32_t inv = (1u << 20) / per + 1;

    W* bs0 = reinterpret_cast<W*>(lora_sh + z.o_b0);
    T* hs = reinterpret_cast<T*>(lora_sh + z.o_hs);  // h as two 16-bit parts, or fp32
    T* hs_lo = hs + (is_f32<T> ? 0 : TM * z.hp);
    bool plain = false;  // h is not finite somewhere, which two parts of it would not survive
    if (r > 0) {
        load_b<W, NB, NW>(bs0, z.bp, wb, crank * NB, d.N, d.rank, r, per, inv);
        cp_async_commit();
        const int chunks = (d.K + KB - 1) / KB, mine = chunks > (int)crank ? (chunks - crank + csize - 1) / csize : 0;
        // A chunk of K to its stage.  Rows of x past the tile's and of A past the rank keep what was there: they only reach
        // sums that nobody reads.
        constexpr int EX = 16 / sizeof(T), EA = 16 / sizeof(W), VX = KB / EX, VA = KB / EA, RX = kLoraThreads / VX, RA = kLoraThreads / VA;
        const int rx = threadIdx.x / VX, kx = threadIdx.x % VX * EX, ra = threadIdx.x / VA, ka = threadIdx.x % VA * EA;
        const T* x0 = (const T*)d.x + (m0 + rx) * d.ldx + kx;
        const W* a0 = wa + (int64_t)ra * d.K + ka;
        auto fetch = [&](int c) {
            T* xs = reinterpret_cast<T*>(lora_sh + (c & 1) * z.stage);
            W* as = reinterpret_cast<W*>(xs + TM * S::XP);
            const int k0 = (crank + c * csize) * KB;
            const bool okx = k0 + kx < d.K, oka = k0 + ka < d.K;
            const T* xp = okx ? x0 + k0 : (const T*)d.x;
            const W* ap = oka ? a0 + k0 : wa;
#pragma unroll 2
            for (int row = rx; row < rows; row += RX) {
                cp_async16_or_zero(xs + row * S::XP + kx, xp, okx);
                xp += okx ? RX * d.ldx : 0;
            }
#pragma unroll 2
            for (int row = ra; row < r; row += RA) {
                cp_async16_or_zero(as + row * S::AP + ka, ap, oka);
                ap += oka ? (int64_t)RA * d.K : 0;
            }
        };
        float acc[RB][4];
#pragma unroll
        for (int i = 0; i < RB; i++) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
        if (mine > 0) fetch(0);
        cp_async_commit();
        for (int c = 0; c < mine; c++) {
            if (c + 1 < mine) fetch(c + 1);
            cp_async_commit();
            cp_async_wait<1>();
            __syncthreads();
            const T* xs = reinterpret_cast<const T*>(lora_sh + (c & 1) * z.stage) + wm * 16 * S::XP;
            const W* as = reinterpret_cast<const W*>(reinterpret_cast<const T*>(lora_sh + (c & 1) * z.stage) + TM * S::XP);
            if constexpr (is_f32<T>) {  // (MMA accumulation truncates: fp32 sums leave it after every stage)
                float part[RB][4];
#pragma unroll
                for (int i = 0; i < RB; i++) part[i][0] = part[i][1] = part[i][2] = part[i][3] = 0.0f;
                for (int k = wk * 16; k < KB; k += WK * 16)
                    mul_16<T, W, RB, false>(part, xs + k, nullptr, S::XP, as + k, S::AP, blocks);
#pragma unroll
                for (int i = 0; i < RB; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[i][e] += part[i][e];
            } else {
                for (int k = wk * 16; k < KB; k += WK * 16)
                    mul_16<T, W, RB, false>(acc, xs + k, nullptr, S::XP, as + k, S::AP, blocks);
            }
            __syncthreads();
        }
        // this CTA's part of h: [K part of a warp][row][rank]
        float* hp = reinterpret_cast<float*>(lora_sh + z.o_hpart);
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int i = 0; i < RB; i++) {
            if (i >= blocks) break;
            float* at = hp + (wk * TM + wm * 16 + g) * z.hp + i * 8 + 2 * t;
            *reinterpret_cast<float2*>(at) = make_float2(acc[i][0], acc[i][1]);
            *reinterpret_cast<float2*>(at + 8 * z.hp) = make_float2(acc[i][2], acc[i][3]);
        }
        if (WK > 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < rows * blocks * 8; i += kLoraThreads) {
                const int at = i / (blocks * 8) * z.hp + i % (blocks * 8);
                float v = hp[at];
#pragma unroll
                for (int j = 1; j < WK; j++) v += hp[j * TM * z.hp + at];
                hp[at] = v;
            }
        }
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        // every CTA takes the whole of h: the parts in rank order, four values a step
        const float scale = __ldg(d.scale + w);
        const uint32_t local = smem_u32(hp);
        for (int i = threadIdx.x; i < TM * (z.Rp / 4); i += kLoraThreads) {
            const int row = i / (z.Rp / 4), col = i % (z.Rp / 4) * 4;
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (row < rows && col < r) {
                for (uint32_t c = 0; c < csize; c++) {
                    uint32_t addr;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(local + (row * z.hp + col) * 4), "r"(c));
                    float p[4];
                    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                                 : "=f"(p[0]), "=f"(p[1]), "=f"(p[2]), "=f"(p[3]) : "r"(addr) : "memory");
#pragma unroll
                    for (int j = 0; j < 4; j++) v[j] += p[j];
                }
                if constexpr (is_f32<T>) {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (v[j] - v[j] != 0.0f && col + j < r)
                            v[j] = plain_sum((const T*)d.x + (m0 + row) * d.ldx, wa + (int64_t)(col + j) * d.K, d.K);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float h = col + j < r ? v[j] * scale : 0.0f;
                hs[row * z.hp + col + j] = from_f<T>(h);
                if (is_f32<T>) plain = plain || !(fabsf(h) < 3.4e38f);
                if constexpr (!is_f32<T>) {
                    const float hi = to_f(from_f<T>(h));
                    hs_lo[row * z.hp + col + j] = from_f<T>(hi - hi == 0.0f ? h - hi : 0.0f);  // (an infinity has no rest)
                }
            }
        }
        // peers may still read this CTA's part: no CTA leaves before all have arrived here
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        if constexpr (is_f32<T>) plain = __syncthreads_or(plain);
    }

    // Columns n0 .. n0 + NB - 1 at a time; a warp owns 16 rows x NW columns of them, a thread CW neighbours of rows g and
    // g + 8.  base comes a step ahead.
    constexpr int E = 16 / sizeof(T), CW = NW / 4, VC = CW / E;  // vectors of a row
    W* bs1 = reinterpret_cast<W*>(lora_sh + z.o_b1);
    const int step = csize * NB, g = lane >> 2, c0 = (WK > 1 ? wk * NW : 0) + (lane & 3) * CW, row0 = wm * 16 + g;
    const T* base0 = (const T*)d.base + (m0 + row0) * d.ldb + c0;
    T* out0 = (T*)d.out + (m0 + row0) * d.ldo + c0;
    auto fetch_base = [&](int n0, uint4 (&v)[2][VC]) {
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int j = 0; j < VC; j++) {
                v[e][j] = make_uint4(0, 0, 0, 0);
                if (d.base && row0 + 8 * e < rows && n0 + c0 + j * E < d.N)
                    v[e][j] = *reinterpret_cast<const uint4*>(base0 + 8 * e * d.ldb + n0 + j * E);
            }
    };
    uint4 old[2][VC], next[2][VC];
    fetch_base(crank * NB, old);
    int it = 0;
    for (int n0 = crank * NB; n0 < d.N && !plain; n0 += step, it++) {
        fetch_base(n0 + step, next);
        float o[NW / 8][4];
#pragma unroll
        for (int i = 0; i < NW / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        if (r > 0) {
            cp_async_wait<0>();
            __syncthreads();  // this step's B has landed (and h is written); the other buffer is free
            if (n0 + step < d.N) load_b<W, NB, NW>(it & 1 ? bs0 : bs1, z.bp, wb, n0 + step, d.N, d.rank, r, per, inv);
            cp_async_commit();
            const W* bs = (it & 1 ? bs1 : bs0) + (WK > 1 ? wk * NW * z.bp : 0);
            for (int k = 0; k < inner; k++)
                mul_16<T, W, NW / 8, !is_f32<T>>(o, hs + wm * 16 * z.hp + k * 16, hs_lo + wm * 16 * z.hp + k * 16, z.hp,
                                                 bs + k * 16, z.bp, NW / 8);
        }
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int j = 0; j < VC; j++) {
                if (row0 + 8 * e >= rows || n0 + c0 + j * E >= d.N) continue;
                if (r > 0) {
                    T x[E];
                    memcpy(x, &old[e][j], 16);
#pragma unroll
                    for (int v = 0; v < E; v++) x[v] = from_f<T>(to_f(x[v]) + o[(j * E + v) / 2][2 * e + v % 2]);
                    memcpy(&old[e][j], x, 16);
                }
                *reinterpret_cast<uint4*>(out0 + 8 * e * d.ldo + n0 + j * E) = old[e][j];
            }
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int j = 0; j < VC; j++) old[e][j] = next[e][j];
    }
    if constexpr (is_f32<T>)
        if (plain)
            for (int n0 = crank * NB; n0 < d.N; n0 += step)
                for (int i = threadIdx.x; i < rows * NB; i += kLoraThreads) {
                    const int row = i / NB, n = n0 + i % NB;
                    if (n >= d.N) continue;
                    const float base = d.base ? ((const float*)d.base)[(m0 + row) * d.ldb + n] : 0.0f;
                    ((float*)d.out)[(m0 + row) * d.ldo + n] = base + plain_sum((const T*)hs + row * z.hp, wb + (int64_t)n * d.rank, r);
                }
    cp_async_wait<0>();
    if (r > 0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// As many tiles as the requests can need.
static int lora_tiles(const voxq_lora& d, int rows) { return d.rows / rows + d.batch; }

// As many CTAs to a tile as keep the grid within 4 an SM, up to 8.  Where 4 fit an SM any number, else a power of two, which
// leaves no holes in a second round.  bf16 prompts (8000 rows, K 1024, N 4096, rank 32): 42 us, 47 with powers of two, 71
// with a bound of 2 an SM and 50 with 8; 9 of 1000 rows, rank 64, K 2960, N 1032: 59 us, 78 with any number.
static int lora_cluster(int tiles, int bytes) {
    int cl = std::min(8, std::max(1, 4 * device_sm_count() / tiles));
    if (bytes + 1024 > 227 * 1024 / 4)
        while (cl & (cl - 1)) cl--;
    return cl;
}

template <typename T, typename W, int TM, int RB, int COLS>
static VoxCPMError lora_launch(const voxq_lora& d, cudaStream_t st) {
    using S = LoraShape<T, W, TM, COLS>;
    const S z(d.rank);
    auto kern = lora_kernel<T, W, TM, RB, COLS>;
    static std::atomic<uint64_t> asked{0};
    VOXQ_CUDA_TRY(allow_shared((const void*)kern, S(RB * 8).bytes, asked));
    const int tiles = lora_tiles(d, TM), cl = lora_cluster(tiles, z.bytes);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles * cl);
    cfg.blockDim = dim3(kLoraThreads);
    cfg.dynamicSmemBytes = z.bytes;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cl;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    VOXQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, d));
    return VOXCPM_SUCCESS;
}

// Tiles of 64 rows read the weights less often and pay where there are enough of them and few are part empty; fp32 rows split
// their operands for every MMA and want the more warps a row unless the rank is high.  us, 64 against 16 rows.  bf16, rank 32,
// K 1024, N 4096: 40 requests of 64 rows 31 : 29, of 128 43 : 53, of 300 81 : 91, 2 of 4096 50 : 58; rank 64, K 2960, N 1032: 30 of
// 96 32 : 45, 40 of 64 32 : 44, 4 of 40 17 : 13; rank 128, K 1024, N 2048: 9 of 1000 115 : 196.  fp32 x, K 1024, N 2048, bf16 weights, rank
// 64: 9 of 1000 91 : 109, 40 of 300 169 : 160, of 128 85 : 106; rank 128: 9 of 1000 237 : 326.  fp32 weights: rank 48 106 : 127, rank 64
// 182 : 155 (the one class whose tall tiles lose), rank 128 302 : 445.
// Steps of 256 columns pay each step's wait less often, but their registers leave an SM three blocks: taken where all blocks then
// run at once (a request that is shorter than a tile has one tile all the same) and have a step each.  us, 256 against 128 columns, fp32 x, bf16 weights, rank 16, K 2048, N 2048: 40 single rows 8.2 : 9.5, 40
// requests of 8 9.7 : 11.1, of 64 26 : 30; not all at once: 100 single rows 18.8 : 15.2, 3 of 300 19 : 14, 9 of 1000 90 : 69.  Rank
// 32, where clusters are powers of two: 100 single rows 15.3 : 18.5.  bf16 x: 40 of 8 7.7 : 8.6, 3 of 300 13.8 : 9.6.  N 1024: 20 single rows,
// rank 32, 8.5 : 7.3.
template <typename T, typename W>
static VoxCPMError lora_dispatch(const voxq_lora& d, cudaStream_t st) {
    const bool tall = d.rows >= 24 * (int64_t)d.batch && d.rows >= (d.rank > 32 && !is_f32<T> ? 16 : 32) * device_sm_count();
    if (d.rank > 64) return tall ? lora_launch<T, W, 64, 16, 64>(d, st) : lora_launch<T, W, 16, 16, 128>(d, st);
    if (d.rank > 32) return tall ? lora_launch<T, W, 64, 8, 64>(d, st) : lora_launch<T, W, 16, 8, 128>(d, st);
    if constexpr (!is_f32<T>)
        if (tall) return lora_launch<T, W, 64, 4, 64>(d, st);
    const int64_t blocks = (int64_t)std::max(d.batch, d.rows / 16) * lora_cluster(lora_tiles(d, 16), LoraShape<T, W, 16, 256>(d.rank).bytes);
    return d.N >= 8 * 256 && blocks <= 3 * device_sm_count() ? lora_launch<T, W, 16, 4, 256>(d, st) : lora_launch<T, W, 16, 4, 128>(d, st);
}

}  // namespace voxq

using namespace voxq;

extern "C" VoxCPMError voxq_lora_forward(const voxq_lora* d, void* stream) {
    if (!d) return VOXCPM_ERR_INTERNAL;
    if (d->rows < 0 || d->batch < 0 || d->K < 0 || d->N < 0 || d->rank < 0 || d->adapters < 0 || (d->rows && !d->batch))
        return VOXCPM_ERR_SHAPE_MISMATCH;
    if (!elem_ok(d->dtype) || !elem_ok(d->w_dtype) || (d->dtype != VOXQ_F32 && d->dtype != d->w_dtype) || d->K % 8 ||
        d->N % 8 || d->rank % 8 || d->rank > kLoraMaxRank)
        return VOXCPM_ERR_UNSUPPORTED;
    if (d->rows == 0 || d->N == 0) return VOXCPM_SUCCESS;
    const bool weights = d->adapters && d->rank && d->K;
    if (!d->out || !d->cu || !d->adapter || (weights && (!d->x || !d->a || !d->b || !d->scale))) return VOXCPM_ERR_INTERNAL;
    if (!rows16(d->out, d->ldo, d->dtype) || (d->base && !rows16(d->base, d->ldb, d->dtype)) ||
        (weights && (!rows16(d->x, d->ldx, d->dtype) || !rows16(d->a, 0, d->w_dtype) || !rows16(d->b, 0, d->w_dtype))))
        return VOXCPM_ERR_UNSUPPORTED;
    voxq_lora p = *d;
    if (!weights) p.adapters = 0;
    cudaStream_t st = (cudaStream_t)stream;
    return with_elem(p.dtype, [&](auto x) {
        return with_elem(p.w_dtype, [&](auto w) {
            using T = decltype(x);
            using W = decltype(w);
            if constexpr (is_f32<T> || std::is_same<T, W>::value) return lora_dispatch<T, W>(p, st);
            else return VOXCPM_ERR_UNSUPPORTED;
        });
    });
}
