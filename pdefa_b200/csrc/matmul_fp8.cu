// Matrix product of 8-bit floating-point operands (e4m3) with block scales:
//
//   out[m, n] = sum over kb of sa[m, kb] * sb[n / 128, kb] *
//               (sum over the 128 k of block kb of a[m, k] * b[n, k])
//
// a is [M, K] (rows are tokens), b is [N, K] (a weight as it is stored), or
// [experts, N, K] with `offsets` giving each expert's range of rows of a.
//
// Two warp-specialised tcgen05 kernels. The narrow one's tile is 128 rows of the weight
// (the M side of the instruction, its 128 TMEM lanes) times 16 to 128 tokens (its N side,
// TMEM columns), so a handful of tokens costs a narrow tile and not 128 padded rows; the
// wide one's is 128 or 256 tokens (lanes) times 256 weight rows (columns).
//
// Scales change with every 128 k, so an accumulator cannot run through K on the tensor
// core: each k-block (one 128-byte swizzled row per operand row, four instructions of
// K = 32) goes into a fresh TMEM accumulator, and the epilogue warps add accumulator *
// scale to 32-bit sums in registers while the tensor core fills the next. A weight tile of
// 128 rows shares one scale per k-block (tiles start at multiples of 128), tokens have one
// each. Narrow: the products of both scales come from shared memory as one broadcast load per
// four columns. Wide: a lane is a token, so it has one scale per k-block. Either way the sum is
// one packed fp32x2 multiply-add per two columns.
//
// What bounds them (B200). Few tokens: reading the weights, 64 rows over 64 experts of 2048 x
// 2048 in 31 us, 5.4 TB/s; for one weight of 16 MB a launch and the pipeline's ends are most of
// 6.2 us. Many tokens: TMEM, which the epilogue reads (128 KB per k-block and SM) beside the
// tensor core; 8192 x 8192 x 4096 takes 268 us from a graph, 2050 TFLOP/s (278 on a slower card;
// 310 in a loop of calls, where the power limit rules), at 990 cycles per k-block, where products
// alone, without loads and epilogue, need 640 and the epilogue's reads 350.
#include <algorithm>
#include <atomic>
#include <cuda.h>
#include <cuda_fp16.h>

#include "common.h"
#include "device_common.cuh"
#include "tc_common.cuh"

namespace pb {

namespace {

constexpr int kBlock = 128;             // k per scale, and bytes of an operand row per stage
constexpr int kTileN = 128;             // weight rows of a tile
constexpr int kScaleChunk = 8;          // k-blocks of scales staged at a time (one 32-byte sector per token)
constexpr uint32_t kABytes = 2 * kTileN * kBlock;   // weights of a stage
constexpr uint32_t kBarrierBytes = 512;

struct TcArgs {
    const int32_t* offsets;             // null: one weight
    int experts, m, n, nkb;             // nkb: k-blocks
    int n_tiles, m_tiles;               // m_tiles: token tiles (one weight)
    int stages, split;
    const float* sa; int64_t lda_scales;
    const float* sb; int64_t ldb_scales, sb_expert;
    void* out; int64_t ldo; int out_dtype;
    uint32_t table_bytes;               // the experts' tile table in shared memory (12 KB for the most experts)
    int wide_out;                       // output rows start at multiples of 16 bytes
    int tma_end;                        // TMA may store columns that end here at most
    int* err;
    long long wait_limit;
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster(uint32_t addr, uint32_t rank) {
    float4 v;
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\tld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr), "r"(rank) : "memory");
    return v;
}

// A bounded wait of a whole warp, with one answer for all lanes.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, long long limit) {
    return __all_sync(~0u, mbar_wait_bounded(bar, parity, limit));
}

// One k-block: four K = 32 products into a fresh accumulator.
__device__ __forceinline__ void mma_kblock(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred pf, pt;\n\t.reg .b64 a1, b1, a2, b2, a3, b3;\n\t"
        "setp.ne.u32 pf, 0, 0;\n\tsetp.eq.u32 pt, 0, 0;\n\t"
        "add.s64 a1, %1, 2;\n\tadd.s64 b1, %2, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 b2, %2, 4;\n\t"
        "add.s64 a3, %1, 6;\n\tadd.s64 b3, %2, 6;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, pf;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a1, b1, %3, pt;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a2, b2, %3, pt;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a3, b3, %3, pt;\n\t}"
        ::"r"(d), "l"(da), "l"(db), "r"(idesc)
        : "memory");
}

template <int BT>
struct Shape {
    static constexpr int kEpi = BT >= 128 ? 8 : 4;                  // epilogue warps
    static constexpr int kThreads = 128 + 32 * kEpi;
    static constexpr int kCols = BT * 4 / kEpi;                     // columns of an epilogue thread
    static constexpr int kBufs = 2;                                 // TMEM buffers, of two accumulators each
    static constexpr int kTmemCols = kBufs * 2 * BT;                // 64 .. 512
    static constexpr uint32_t kBBytes = 2 * BT * kBlock;            // tokens of a stage
    static constexpr uint32_t kScaleBytes = kScaleChunk * BT * 4;   // of one of two chunks
};

struct Tile {
    int expert, row0, rows, n0;         // first token, tokens that belong to the tile, first weight row
};

// The experts' rows: [first row | end | token tiles before it] for each, in shared memory;
// returns the number of token tiles. An offset outside 0 .. m or below one before it
// counts as the nearest value that is not, so every row has one expert at most. One warp.
template <int BT>
__device__ __forceinline__ int build_table(const TcArgs& p, int* table) {
    const int lane = threadIdx.x & 31;
    int before = 0, least = 0;
    for (int e0 = 0; e0 < p.experts; e0 += 32) {
        const int e = e0 + lane;
        int lo = 0, hi = 0;
        if (e < p.experts) {
            lo = min(max(p.offsets[e], 0), p.m);
            hi = min(max(p.offsets[e + 1], 0), p.m);
        }
        lo = max(lo, least);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) lo = max(lo, __shfl_up_sync(~0u, lo, o));
        hi = max(hi, lo);
        least = __shfl_sync(~0u, hi, 31);
        const int rows = hi - lo, tiles = e < p.experts ? rows / BT + (rows % BT != 0) : 0;
        int sum = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(~0u, sum, o);
            if (lane >= o) sum += v;
        }
        if (e < p.experts) {
            table[e] = lo;
            table[p.experts + e] = hi;
            table[2 * p.experts + e] = before + sum - tiles;
        }
        before += __shfl_sync(~0u, sum, 31);
    }
    return before;
}

// Tiles are numbered with the token tiles of an expert innermost, so that CTAs that run
// together read the same weight rows.
template <int BT, int TN>
__device__ __forceinline__ Tile tile_of(const TcArgs& p, const int* table, int token_tiles, int64_t t) {
    Tile r;
    if (!p.offsets) {
        const int nt = (int)(t / p.m_tiles);
        r.expert = 0;
        r.row0 = (int)(t - (int64_t)nt * p.m_tiles) * BT;
        r.rows = min(BT, p.m - r.row0);
        r.n0 = nt * TN;
        return r;
    }
    const int* before = table + 2 * p.experts;
    const int u = (int)(t / p.n_tiles);             // lies in the expert's range of token tiles
    int lo = 0, hi = p.experts - 1;                 // last expert with before <= u
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (before[mid] <= u) lo = mid;
        else hi = mid - 1;
    }
    const int mine = (lo + 1 < p.experts ? before[lo + 1] : token_tiles) - before[lo];
    const int64_t local = t - (int64_t)before[lo] * p.n_tiles;
    const int nt = (int)(local / mine);
    r.expert = lo;
    r.row0 = table[lo] + (int)(local - (int64_t)nt * mine) * BT;
    r.rows = min(BT, table[p.experts + lo] - r.row0);
    r.n0 = nt * TN;
    return r;
}

__device__ __forceinline__ void store_out(void* out, int dtype, int64_t i, float v) {
    if (dtype == ENGINE_F32) static_cast<float*>(out)[i] = v;
    else if (dtype == ENGINE_F16) static_cast<__half*>(out)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
}

// Four columns of a row, n a multiple of 4.
__device__ __forceinline__ void convert(float* d, float v) { *d = v; }
__device__ __forceinline__ void convert(__half* d, float v) { *d = __float2half_rn(v); }
__device__ __forceinline__ void convert(__nv_bfloat16* d, float v) { *d = __float2bfloat16_rn(v); }
// One weight row's values of up to N tokens; the lanes of a warp hold neighbouring ones.
template <int N, typename T>
__device__ __forceinline__ void store_column(T* d, int64_t ldo, int most, const float* v) {
#pragma unroll
    for (int i = 0; i < N; ++i, d += ldo)
        if (i < most) convert(d, v[i]);
}
__device__ __forceinline__ void store_out4(const TcArgs& p, int row, int n, float4 v) {
    const int64_t at = (int64_t)row * p.ldo + n;
    if (p.wide_out && n + 4 <= p.n) {
        if (p.out_dtype == ENGINE_F32) {
            *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = v;
        } else {
            uint2 q;
            if (p.out_dtype == ENGINE_F16) {
                const __half2 lo = __floats2half2_rn(v.x, v.y), hi = __floats2half2_rn(v.z, v.w);
                q = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
            } else {
                const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
                q = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
            }
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) = q;
        }
        return;
    }
    const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n + i < p.n) store_out(p.out, p.out_dtype, at + i, e[i]);
}

// Roles: warps 0 and 3 bring operands (TMA), warp 1 issues the products and owns TMEM, warp 2
// brings scales, warps 4 and up are the epilogue. Every wait is bounded; one that runs
// out records a code in the device's error word and ends its role, after which the
// others' waits run out too; loads and products in flight are waited for before exit.
// SPLIT: the CTAs of a cluster take the k-blocks of one tile in equal parts and join
// their sums through distributed shared memory in rank order.
template <int BT, bool SPLIT>
__global__ void __launch_bounds__(Shape<BT>::kThreads, 1)
matmul_fp8_kernel(const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmA, const TcArgs p) {
    using S = Shape<BT>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* const smem = smem_raw + (base - raw);
    const int stages = p.stages;
    // [weight slots | token slots | scales | barriers | table], slots 1024-aligned
    const uint32_t ring_b = base + (uint32_t)stages * kABytes;
    float* const scales = reinterpret_cast<float*>(smem + (size_t)stages * (kABytes + S::kBBytes));
    uint64_t* const full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(scales) + 2 * S::kScaleBytes);
    uint64_t* const done = full + stages;
    uint64_t* const tempty = done + stages;
    uint64_t* const sfull = tempty + S::kBufs;
    uint64_t* const sempty = sfull + 2;
    uint64_t* const mma_done = sempty + 2;
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
    int* const tile_count = reinterpret_cast<int*>(tmem_slot + 1);
    int* const table = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(full) + kBarrierBytes);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; ++i) { mbar_init(&full[i], 2); mbar_init(&done[i], 1); }
        for (int i = 0; i < S::kBufs; ++i) mbar_init(&tempty[i], S::kEpi);
        for (int i = 0; i < 2; ++i) { mbar_init(&sfull[i], 1); mbar_init(&sempty[i], S::kEpi); }
        mbar_init(mma_done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)S::kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    grid_trigger();
    grid_wait();                                             // what the stream wrote before is there
    if (warp == 2) {
        const int n = p.offsets ? build_table<BT>(p, table) : p.m_tiles;
        if (lane == 0) *tile_count = n;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    const int token_tiles = *tile_count;
    const int64_t total = (int64_t)token_tiles * p.n_tiles;

    // this CTA's tiles and, of each, its pairs of k-blocks (the last one's second may be past the end: zeros)
    const uint32_t rank = SPLIT ? cluster_rank() : 0;
    const int64_t t0 = SPLIT ? blockIdx.x / p.split : blockIdx.x;
    const int64_t tstep = SPLIT ? total : gridDim.x;        // SPLIT: one tile per cluster
    const int pairs = (p.nkb + 1) / 2;
    const int pr0 = SPLIT ? (int)((int64_t)pairs * rank / p.split) : 0;
    const int pr1 = SPLIT ? (int)((int64_t)pairs * (rank + 1) / p.split) : pairs;

    float acc[S::kCols];
    Tile mine{0, 0, 0, 0};
    bool failed = false;

    if (warp == 0 || warp == 3) {
        // Weights from one warp, tokens from another: issuing a load takes a thread some 150
        // cycles, and both from one held up the narrow tiles.
        if (lane == 0) {
            const bool weights = warp == 0;
            RingPos rp;
            int64_t it = 0;
            for (int64_t t = t0; t < total && !failed; t += tstep) {
                const Tile tl = tile_of<BT, kTileN>(p, table, token_tiles, t);
                for (int pr = pr0; pr < pr1; ++pr) {
                    const int st = rp.slot;
                    if (rp.wrapped && !mbar_wait_bounded(&done[st], rp.phase ^ 1u, p.wait_limit)) {
                        atomicExch(p.err, 21);
                        failed = true;
                        break;
                    }
                    rp.next(stages);
                    ++it;
                    mbar_expect_tx(&full[st], weights ? kABytes : S::kBBytes);
                    for (int h = 0; h < 2; ++h) {
                        const int k = (2 * pr + h) * kBlock;
                        if (weights) tma_load_3d(base + (uint32_t)st * kABytes + h * (kABytes / 2), &tmB, &full[st], k, tl.n0, tl.expert);
                        else tma_load_2d(ring_b + (uint32_t)st * S::kBBytes + h * (S::kBBytes / 2), &tmA, &full[st], k, tl.row0);
                    }
                }
            }
            // the last load of every slot has landed before the CTA may exit
            for (int64_t k = it > stages ? it - stages : 0; k < it; ++k)
                if (!mbar_wait_bounded(&full[k % stages], (uint32_t)((k / stages) & 1))) atomicExch(p.err, 22);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            // f32 accumulator, e4m3 operands, N = BT, M = 128
            const uint32_t idesc = (1u << 4) | ((uint32_t)(BT >> 3) << 17) | ((uint32_t)(kTileN >> 4) << 24);
            RingPos rp, ap;
            for (int64_t t = t0; t < total && !failed; t += tstep) {
                for (int pr = pr0; pr < pr1; ++pr) {
                    const int st = rp.slot, buf = ap.slot;
                    if ((ap.wrapped && !mbar_wait_bounded(&tempty[buf], ap.phase ^ 1u, p.wait_limit)) ||
                        !mbar_wait_bounded(&full[st], rp.phase, p.wait_limit)) {
                        atomicExch(p.err, 23);
                        failed = true;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t da = make_smem_desc(base + (uint32_t)st * kABytes, 128);
                    const uint64_t db = make_smem_desc(ring_b + (uint32_t)st * S::kBBytes, 128);
                    const uint32_t d = tmem + (uint32_t)(buf * 2 * BT);
                    // the second halves, in the descriptors' units of 16 bytes
                    mma_kblock(d, da, db, idesc);
                    mma_kblock(d + BT, da + (kABytes / 2 >> 4), db + (S::kBBytes / 2 >> 4), idesc);
                    umma_commit(&done[st]);
                    rp.next(stages);
                    ap.next(S::kBufs);
                }
            }
            umma_commit(mma_done);
        }
        __syncwarp();
    } else if (warp == 2) {
        // scales: chunk c holds sa[token, kb] * sb[kb] for kScaleChunk k-blocks, [kb][token]
        RingPos cp;
        for (int64_t t = t0; t < total && !failed; t += tstep) {
            const Tile tl = tile_of<BT, kTileN>(p, table, token_tiles, t);
            const float* sa = p.sa + (int64_t)tl.row0 * p.lda_scales;
            const float* sb = p.sb + tl.expert * p.sb_expert + (tl.n0 / kTileN) * p.ldb_scales;
            for (int kc = 2 * pr0; kc < 2 * pr1 && !failed; kc += kScaleChunk) {
                const int kb1 = min(2 * pr1, p.nkb);
                float w[kScaleChunk];
#pragma unroll
                for (int j = 0; j < kScaleChunk; ++j) w[j] = kc + j < kb1 ? __ldg(sb + kc + j) : 0.0f;
                if (cp.wrapped && !warp_wait(&sempty[cp.slot], cp.phase ^ 1u, p.wait_limit)) {
                    if (lane == 0) atomicExch(p.err, 24);
                    failed = true;
                    break;
                }
                float* dst = scales + cp.slot * (kScaleChunk * BT);
#pragma unroll(BT >= 128 ? 4 : 1)
                for (int i = lane; i < BT; i += 32) {
                    float v[kScaleChunk];
#pragma unroll
                    for (int j = 0; j < kScaleChunk; ++j)
                        v[j] = i < tl.rows && kc + j < kb1 ? __ldg(sa + i * p.lda_scales + kc + j) : 0.0f;
#pragma unroll
                    for (int j = 0; j < kScaleChunk; ++j) dst[j * BT + i] = v[j] * w[j];
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sfull[cp.slot]);
                cp.next(2);
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        const int q = warp & 3;                           // TMEM lane quarter
        const int c0 = ((warp - 4) >> 2) * S::kCols;      // first column of this warp's group
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        RingPos rp, ap, cp;      // done, accumulators, scales
        for (int64_t t = t0; t < total && !failed; t += tstep) {
            mine = tile_of<BT, kTileN>(p, table, token_tiles, t);
#pragma unroll
            for (int i = 0; i < S::kCols; ++i) acc[i] = 0.0f;
            for (int pr = pr0; pr < pr1; ++pr) {
                const int in_chunk = 2 * (pr - pr0) % kScaleChunk;
                if ((in_chunk == 0 && !warp_wait(&sfull[cp.slot], cp.phase, p.wait_limit)) ||
                    !warp_wait(&done[rp.slot], rp.phase, p.wait_limit)) {
                    if (lane == 0) atomicExch(p.err, 25);
                    failed = true;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t src = tmem + lanes + (uint32_t)(ap.slot * 2 * BT + c0);
                const float* sc = scales + cp.slot * (kScaleChunk * BT) + in_chunk * BT + c0;
                constexpr int kChunks = S::kCols / 16;               // per k-block
                uint32_t r[2][16];
                tmem_ld16_async(src, r[0]);
#pragma unroll
                for (int c = 0; c < 2 * kChunks; ++c) {
                    tmem_wait_ld();
                    if (c + 1 < 2 * kChunks) tmem_ld16_async(src + (c + 1) / kChunks * BT + (c + 1) % kChunks * 16, r[(c + 1) & 1]);
                    else {
                        // everything is in registers: the tensor core may refill the buffer
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&tempty[ap.slot]);
                    }
                    const uint32_t(&v)[16] = r[c & 1];
                    const float4* s4p = reinterpret_cast<const float4*>(sc + c / kChunks * BT + c % kChunks * 16);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float4 s4 = s4p[j];
                        float* d = acc + c % kChunks * 16 + j * 4;
                        const float2 lo = __ffma2_rn(make_float2(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1])),
                                                     make_float2(s4.x, s4.y), make_float2(d[0], d[1]));
                        const float2 hi = __ffma2_rn(make_float2(__uint_as_float(v[4 * j + 2]), __uint_as_float(v[4 * j + 3])),
                                                     make_float2(s4.z, s4.w), make_float2(d[2], d[3]));
                        d[0] = lo.x; d[1] = lo.y; d[2] = hi.x; d[3] = hi.y;
                    }
                }
                rp.next(stages);
                ap.next(S::kBufs);
                if (in_chunk == kScaleChunk - 2 || pr == pr1 - 1) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sempty[cp.slot]);
                    cp.next(2);
                }
            }
            if (SPLIT || failed) continue;
            const int n = mine.n0 + q * 32 + lane;
            const int most = n < p.n ? mine.rows - c0 : 0;
            const int64_t at = (int64_t)(mine.row0 + c0) * p.ldo + n;
            if (p.out_dtype == ENGINE_BF16) store_column<S::kCols>(static_cast<__nv_bfloat16*>(p.out) + at, p.ldo, most, acc);
            else if (p.out_dtype == ENGINE_F16) store_column<S::kCols>(static_cast<__half*>(p.out) + at, p.ldo, most, acc);
            else store_column<S::kCols>(static_cast<float*>(p.out) + at, p.ldo, most, acc);
        }
        if (!SPLIT && p.offsets) {
            // rows before the first and after the last expert's
            const int lo = table[0], hi = table[2 * p.experts - 1];
            const int tid = threadIdx.x - 128;
            for (int64_t i = (int64_t)blockIdx.x; i < (int64_t)lo + (p.m - hi); i += gridDim.x) {
                const int64_t row = i < lo ? i : hi + (i - lo);
                for (int n = tid; n < p.n; n += 32 * S::kEpi) store_out(p.out, p.out_dtype, row * p.ldo + n, 0.0f);
            }
        }
    }

    if (SPLIT) {
        // Sums as [token][weight row] in the ring's memory: every load and product of
        // this CTA is behind the epilogue's last accumulator.
        float* const part = reinterpret_cast<float*>(smem);
        const int q = warp & 3, c0 = ((warp - 4) >> 2) * S::kCols;
        if (warp >= 4 && !failed) {
#pragma unroll
            for (int i = 0; i < S::kCols; ++i) part[(c0 + i) * kTileN + q * 32 + lane] = acc[i];
        }
        __syncwarp();
        cluster_sync();
        if (warp >= 4 && !failed) {
            // each CTA joins its share of the tokens, four weight rows per thread and load
            const int per = BT / p.split;
            for (int i = threadIdx.x - 128; i < per * (kTileN / 4); i += 32 * S::kEpi) {
                const int j = (int)rank * per + i / (kTileN / 4), n = mine.n0 + i % (kTileN / 4) * 4;
                if (j >= mine.rows || n >= p.n) continue;
                const uint32_t at = smem_u32(part + j * kTileN + i % (kTileN / 4) * 4);
                float4 v[8], sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    if (c < p.split) v[c] = ld_cluster(at, c);
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    if (c < p.split) { sum.x += v[c].x; sum.y += v[c].y; sum.z += v[c].z; sum.w += v[c].w; }
                store_out4(p, mine.row0 + j, n, sum);
            }
        }
        __syncwarp();
        cluster_sync();
    }

    // TMEM is freed once every issued product has completed.
    __syncthreads();
    if (warp == 1) {
        if (!mbar_wait_bounded(mma_done, 0) && lane == 0) atomicExch(p.err, 26);
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)S::kTmemCols) : "memory");
    }
}

// ---------------------------------------------------------------------------
// Many tokens: tiles of 128 * CG tokens (TMEM lanes, 128 per CTA) times 256 weight rows (TMEM
// columns). CG = 2 is a pair of CTAs on one tile: each brings its own tokens and half of the
// weight rows, and the tensor cores of both read both halves, so that a CTA moves 32 KB per
// k-block instead of 48. (A product of 128 columns takes the tensor core as long as one of
// 256, so finer accumulators that change hands earlier lose: 353 us against 277.)
// ---------------------------------------------------------------------------
constexpr int kWideN = 256;
constexpr int kWideEpi = 8;
constexpr int kWideThreads = 128 + 32 * kWideEpi;
constexpr int kWideCols = kWideN * 4 / kWideEpi;    // columns of an epilogue thread
constexpr uint32_t kWideScales = kScaleChunk * (128 + 2) * 4;

__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}

template <int CG>
__device__ __forceinline__ void wide_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
    if (CG == 1)
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                     ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                     ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
template <int CG>
__device__ __forceinline__ void wide_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
    if (CG == 1)
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                     ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                     ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
// Arrival on the barrier at this address in every CTA of the group once the products
// issued so far have completed.
template <int CG>
__device__ __forceinline__ void wide_commit(uint64_t* bar) {
    if (CG == 1) umma_commit(bar);
    else
        asm volatile("{\n\t.reg .b16 m;\n\tmov.b16 m, 3;\n\t"
                     "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}"
                     ::"r"(smem_u32(bar)) : "memory");
}
template <int CG>
__device__ __forceinline__ void wide_mma(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc) {
    if (CG == 1)
        asm volatile(
            "{\n\t.reg .pred pf, pt;\n\t.reg .b64 a1, b1, a2, b2, a3, b3;\n\t"
            "setp.ne.u32 pf, 0, 0;\n\tsetp.eq.u32 pt, 0, 0;\n\t"
            "add.s64 a1, %1, 2;\n\tadd.s64 b1, %2, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 b2, %2, 4;\n\t"
            "add.s64 a3, %1, 6;\n\tadd.s64 b3, %2, 6;\n\t"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, pf;\n\t"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a1, b1, %3, pt;\n\t"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a2, b2, %3, pt;\n\t"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a3, b3, %3, pt;\n\t}"
            ::"r"(d), "l"(da), "l"(db), "r"(idesc) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred pf, pt;\n\t.reg .b64 a1, b1, a2, b2, a3, b3;\n\t"
            "setp.ne.u32 pf, 0, 0;\n\tsetp.eq.u32 pt, 0, 0;\n\t"
            "add.s64 a1, %1, 2;\n\tadd.s64 b1, %2, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 b2, %2, 4;\n\t"
            "add.s64 a3, %1, 6;\n\tadd.s64 b3, %2, 6;\n\t"
            "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, pf;\n\t"
            "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a1, b1, %3, pt;\n\t"
            "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a2, b2, %3, pt;\n\t"
            "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], a3, b3, %3, pt;\n\t}"
            ::"r"(d), "l"(da), "l"(db), "r"(idesc) : "memory");
}

// 32 consecutive fp32 columns of this thread's TMEM lane; no wait.
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}

// Registers: the launch gives every thread kWideRegs; the four warps of loads, products and
// scales hand most of theirs to the eight epilogue warps, whose 128 sums and 64 values in
// flight would not fit otherwise. The two sums are equal, as the instruction needs.
constexpr int kWideRegs = 168, kWideRegsLess = 72, kWideRegsMore = 216;
static_assert(128 * kWideRegsLess + 32 * kWideEpi * kWideRegsMore <= kWideThreads * kWideRegs, "register split");

// The warp's 32 rows (one per lane) of kWideCols sums to rows of the output, `rows` of which
// are this tile's: through the warp's own shared memory in chunks of 128 bytes per row, whose
// 16-byte pieces are swizzled against bank conflicts in the pattern of the output's tensor map.
// Full tiles leave by TMA while the warp goes on; rows that are not aligned for it, or belong to
// the next expert, and last columns that end inside 16 bytes are copied out by the warp. One fence and one pair of TMA
// stores per 256 bytes of a row: issuing them takes a warp some 400 cycles (a tile of 8192 x
// 8192 x 4096 has 32000).
constexpr int kWideChunk = 32 * 128, kWideChunks = 2, kWideStage = kWideChunks * kWideChunk;
template <typename T> __device__ __forceinline__ uint4 out_piece(const float* v);
template <> __device__ __forceinline__ uint4 out_piece<float>(const float* v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
template <> __device__ __forceinline__ uint4 out_piece<__half>(const float* v) {
    uint4 q;
    __half2* h = reinterpret_cast<__half2*>(&q);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    return q;
}
template <> __device__ __forceinline__ uint4 out_piece<__nv_bfloat16>(const float* v) {
    uint4 q;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&q);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    return q;
}
template <typename T>
__device__ __forceinline__ void wide_store(const TcArgs& p, const CUtensorMap* tmO, const float (&acc)[kWideCols], uint8_t* stage,
                                           int row0, int rows, int n0) {
    constexpr int kPer = 128 / sizeof(T), kPiece = 16 / sizeof(T);   // values of a chunk's row and of a piece
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int c = 0; c < kWideCols; c += kWideChunks * kPer) {
        const bool tma = rows >= 32 && n0 + c + kWideChunks * kPer <= p.tma_end;
        if (lane == 0) bulk_wait_read<0>();                          // what was here has left
        __syncwarp();
#pragma unroll
        for (int j = 0; j < kWideChunks * 8; ++j)
            *reinterpret_cast<uint4*>(stage + j / 8 * kWideChunk + lane * 128 + ((j ^ lane) & 7) * 16) = out_piece<T>(acc + c + j * kPiece);
        if (tma) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
#pragma unroll
                for (int h = 0; h < kWideChunks; ++h)
                    if (n0 + c + h * kPer < p.n)
                        tma_store_2d(tmO, smem_u32(stage + h * kWideChunk), (n0 + c + h * kPer) * (int)sizeof(T), row0);
                bulk_commit();
            }
            continue;
        }
        __syncwarp();
        if (p.wide_out && n0 + c + kWideChunks * kPer <= p.n) {
            // rows of a tile that the next expert shares: 16-byte pieces, two rows at a time
            const int j = lane & 15;
#pragma unroll
            for (int i0 = 0; i0 < 16; i0 += 4) {
                uint4 v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = (i0 + i) * 2 + (lane >> 4);
                    v[i] = *reinterpret_cast<const uint4*>(stage + (j >> 3) * kWideChunk + r * 128 + ((j ^ r) & 7) * 16);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = (i0 + i) * 2 + (lane >> 4);
                    if (r < rows) *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (int64_t)(row0 + r) * p.ldo + n0 + c + j * kPiece) = v[i];
                }
            }
        } else {
            // rows that do not start at multiples of 16 bytes, the last columns: a column per
            // lane, eight rows at a time (row by row a tile took 6 us and not 4.5)
#pragma unroll
            for (int i0 = 0; i0 < kWideChunks * kPer; i0 += 32) {
                const int i = i0 + lane;
                const uint8_t* src = stage + i / kPer * kWideChunk + i % kPiece * sizeof(T);
                T* dst = static_cast<T*>(p.out) + (int64_t)row0 * p.ldo + n0 + c + i;
                const int most = n0 + c + i < p.n ? rows : 0;
#pragma unroll
                for (int r0 = 0; r0 < 32; r0 += 8) {
                    T v[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] = *reinterpret_cast<const T*>(src + (r0 + k) * 128 + ((i % kPer / kPiece ^ k) & 7) * 16);
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (r0 + k < most) dst[(r0 + k) * p.ldo] = v[k];
                }
            }
        }
        __syncwarp();
    }
}

// Roles and bounded waits as above. Pairs: CTA 0 of the cluster issues the products for both;
// both CTAs' loads complete on its `full` barriers, its commits arrive in both CTAs, and both
// epilogues hand accumulators back to it.
template <int CG>
__global__ void __launch_bounds__(kWideThreads, 1)
matmul_fp8_wide_kernel(const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmA,
                       const __grid_constant__ CUtensorMap tmO, const TcArgs p) {
    constexpr int BT = 128 * CG;                             // tokens of a tile
    constexpr uint32_t kA = 128 * kBlock, kB = kWideN / CG * kBlock;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* const smem = smem_raw + (base - raw);
    const int stages = p.stages;
    // [token slots | weight slots | output staging | scales | barriers | table], slots 1024-aligned
    const uint32_t ring_b = base + (uint32_t)stages * kA;
    uint8_t* const staging = smem + (size_t)stages * (kA + kB);
    float* const scales = reinterpret_cast<float*>(staging + kWideEpi * kWideStage);
    uint64_t* const full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(scales) + 2 * kWideScales);
    uint64_t* const empty = full + stages;
    uint64_t* const tfull = empty + stages;
    uint64_t* const tempty = tfull + 2;
    uint64_t* const sfull = tempty + 2;
    uint64_t* const sempty = sfull + 2;
    uint64_t* const mma_done = sempty + 2;
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
    int* const tile_count = reinterpret_cast<int*>(tmem_slot + 1);
    int* const table = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(full) + kBarrierBytes);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0;
    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&tfull[i], 1); mbar_init(&tempty[i], kWideEpi * CG); }
        for (int i = 0; i < 2; ++i) { mbar_init(&sfull[i], 1); mbar_init(&sempty[i], kWideEpi); }
        mbar_init(mma_done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        if (CG == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
    }
    grid_trigger();
    grid_wait();                                             // what the stream wrote before is there
    if (warp == 2) {
        const int n = p.offsets ? build_table<BT>(p, table) : p.m_tiles;
        if (lane == 0) *tile_count = n;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (CG == 2) cluster_sync();                             // the other CTA's barriers and TMEM are ready too
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    const int token_tiles = *tile_count;
    const int64_t total = (int64_t)token_tiles * p.n_tiles;
    const int64_t t0 = blockIdx.x / CG, tstep = gridDim.x / CG;
    bool failed = false;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWideRegsLess));
        if (warp == 0) {
            if (lane == 0) {
                RingPos rp;
                int64_t it = 0;
                for (int64_t t = t0; t < total && !failed; t += tstep) {
                    const Tile tl = tile_of<BT, kWideN>(p, table, token_tiles, t);
                    for (int kb = 0; kb < p.nkb; ++kb) {
                        const int st = rp.slot;
                        if (rp.wrapped && !mbar_wait_bounded(&empty[st], rp.phase ^ 1u, p.wait_limit)) {
                            atomicExch(p.err, 31);
                            failed = true;
                            break;
                        }
                        rp.next(stages);
                        ++it;
                        if (rank == 0) mbar_expect_tx(&full[st], CG * (kA + kB));
                        const uint32_t bar = CG == 2 ? mapa(smem_u32(&full[st]), 0) : smem_u32(&full[st]);
                        wide_load_2d<CG>(base + (uint32_t)st * kA, &tmA, bar, kb * kBlock, tl.row0 + (int)rank * 128);
                        wide_load_3d<CG>(ring_b + (uint32_t)st * kB, &tmB, bar, kb * kBlock, tl.n0 + (int)rank * 128, tl.expert);
                    }
                }
                // the last load of every slot has landed before the CTA (or its pair) may exit
                if (rank == 0)
                    for (int64_t k = it > stages ? it - stages : 0; k < it; ++k)
                        if (!mbar_wait_bounded(&full[k % stages], (uint32_t)((k / stages) & 1))) atomicExch(p.err, 32);
            }
            __syncwarp();
        } else if (warp == 1) {
            if (lane == 0 && rank == 0) {
                const uint32_t idesc = (1u << 4) | ((uint32_t)(kWideN >> 3) << 17) | ((uint32_t)(BT >> 4) << 24);
                RingPos rp, ap;
                for (int64_t t = t0; t < total && !failed; t += tstep) {
                    for (int kb = 0; kb < p.nkb; ++kb) {
                        const int st = rp.slot, buf = ap.slot;
                        if ((ap.wrapped && !mbar_wait_bounded(&tempty[buf], ap.phase ^ 1u, p.wait_limit)) ||
                            !mbar_wait_bounded(&full[st], rp.phase, p.wait_limit)) {
                            atomicExch(p.err, 33);
                            failed = true;
                            break;
                        }
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        wide_mma<CG>(tmem + (uint32_t)(buf * kWideN), make_smem_desc(base + (uint32_t)st * kA, 128),
                                     make_smem_desc(ring_b + (uint32_t)st * kB, 128), idesc);
                        wide_commit<CG>(&empty[st]);
                        wide_commit<CG>(&tfull[buf]);
                        rp.next(stages);
                        ap.next(2);
                    }
                }
                wide_commit<CG>(mma_done);
            }
            __syncwarp();
        } else if (warp == 2) {
            // scales: chunk c holds sa[token] for kScaleChunk k-blocks, then sb of the two weight blocks
            RingPos cp;
            for (int64_t t = t0; t < total && !failed; t += tstep) {
                const Tile tl = tile_of<BT, kWideN>(p, table, token_tiles, t);
                const int rows = tl.rows - (int)rank * 128;
                const float* sa = p.sa + (int64_t)(tl.row0 + (int)rank * 128) * p.lda_scales;
                const float* sb = p.sb + tl.expert * p.sb_expert + (tl.n0 / kBlock) * p.ldb_scales;
                const bool second = tl.n0 + kBlock < p.n;
                for (int kc = 0; kc < p.nkb && !failed; kc += kScaleChunk) {
                    if (cp.wrapped && !warp_wait(&sempty[cp.slot], cp.phase ^ 1u, p.wait_limit)) {
                        if (lane == 0) atomicExch(p.err, 34);
                        failed = true;
                        break;
                    }
                    float* dst = scales + cp.slot * (kWideScales / 4);
                    float v[4][kScaleChunk];
    #pragma unroll
                    for (int i = 0; i < 4; ++i)
    #pragma unroll
                        for (int j = 0; j < kScaleChunk; ++j)
                            v[i][j] = i * 32 + lane < rows && kc + j < p.nkb ? __ldg(sa + (int64_t)(i * 32 + lane) * p.lda_scales + kc + j) : 0.0f;
                    if (lane < 2 * kScaleChunk) {
                        const int blk = lane / kScaleChunk, j = lane % kScaleChunk;
                        dst[kScaleChunk * 128 + lane] = (blk == 0 || second) && kc + j < p.nkb ? __ldg(sb + blk * p.ldb_scales + kc + j) : 0.0f;
                    }
    #pragma unroll
                    for (int i = 0; i < 4; ++i)
    #pragma unroll
                        for (int j = 0; j < kScaleChunk; ++j) dst[j * 128 + i * 32 + lane] = v[i][j];
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sfull[cp.slot]);
                    cp.next(2);
                }
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWideRegsMore));
        const int q = warp & 3, grp = (warp - 4) >> 2;       // TMEM lane quarter, group of columns
        const int half = grp * kWideCols / kBlock;           // their weight block
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        const int tok = q * 32 + lane;
        float acc[kWideCols];
        RingPos ap, cp;
        for (int64_t t = t0; t < total && !failed; t += tstep) {
            const Tile tl = tile_of<BT, kWideN>(p, table, token_tiles, t);
#pragma unroll
            for (int i = 0; i < kWideCols; ++i) acc[i] = 0.0f;
            for (int kb = 0; kb < p.nkb; ++kb) {
                const int in_chunk = kb % kScaleChunk;
                if ((in_chunk == 0 && !warp_wait(&sfull[cp.slot], cp.phase, p.wait_limit)) ||
                    !warp_wait(&tfull[ap.slot], ap.phase, p.wait_limit)) {
                    if (lane == 0) atomicExch(p.err, 35);
                    failed = true;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t src = tmem + lanes + (uint32_t)(ap.slot * kWideN + grp * kWideCols);
                const float* sc = scales + cp.slot * (kWideScales / 4);
                uint32_t r[2][32];
                tmem_ld32_async(src, r[0]);
                const float s1 = sc[in_chunk * 128 + tok] * sc[kScaleChunk * 128 + half * kScaleChunk + in_chunk];
                const float2 s2 = make_float2(s1, s1);
#pragma unroll
                for (int c = 0; c < kWideCols / 32; ++c) {
                    tmem_wait_ld();
                    if (c + 1 < kWideCols / 32) tmem_ld32_async(src + (c + 1) * 32, r[(c + 1) & 1]);
                    else {
                        // everything is in registers: the tensor core may refill the buffer
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) {
                            if (CG == 1) mbar_arrive(&tempty[ap.slot]);
                            else mbar_arrive_cluster(mapa(smem_u32(&tempty[ap.slot]), 0));
                        }
                    }
                    const uint32_t(&v)[32] = r[c & 1];
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        float* d = acc + c * 32 + j;
                        const float2 o = __ffma2_rn(make_float2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), s2, make_float2(d[0], d[1]));
                        d[0] = o.x;
                        d[1] = o.y;
                    }
                }
                ap.next(2);
                if (in_chunk == kScaleChunk - 1 || kb == p.nkb - 1) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sempty[cp.slot]);
                    cp.next(2);
                }
            }
            if (failed) continue;
            uint8_t* const mine = staging + (warp - 4) * kWideStage;
            const int row0 = q * 32 + (int)rank * 128, n0 = tl.n0 + grp * kWideCols;
            if (p.out_dtype == ENGINE_BF16) wide_store<__nv_bfloat16>(p, &tmO, acc, mine, tl.row0 + row0, tl.rows - row0, n0);
            else if (p.out_dtype == ENGINE_F16) wide_store<__half>(p, &tmO, acc, mine, tl.row0 + row0, tl.rows - row0, n0);
            else wide_store<float>(p, &tmO, acc, mine, tl.row0 + row0, tl.rows - row0, n0);
        }
        if (lane == 0) bulk_wait0();                         // the last stores have left shared memory
        if (p.offsets) {
            // rows before the first and after the last expert's
            const int lo = table[0], hi = table[2 * p.experts - 1];
            const int tid = threadIdx.x - 128;
            for (int64_t i = (int64_t)blockIdx.x; i < (int64_t)lo + (p.m - hi); i += gridDim.x) {
                const int64_t row = i < lo ? i : hi + (i - lo);
                for (int n = tid; n < p.n; n += 32 * kWideEpi) store_out(p.out, p.out_dtype, row * p.ldo + n, 0.0f);
            }
        }
    }

    // TMEM is freed, and a pair left, once every issued product has completed.
    __syncthreads();
    if (warp == 1) {
        if (!mbar_wait_bounded(mma_done, 0) && lane == 0) atomicExch(p.err, 36);
        __syncwarp();
    }
    if (CG == 2) {
        __syncwarp();
        cluster_sync();
    }
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// Rows of bytes into rows of `ld` bytes (a multiple of 16), for operands that TMA cannot read.
__global__ void __launch_bounds__(256)
repack_rows_kernel(const uint8_t* src, int64_t ld_src, int64_t group_src, uint8_t* dst, int64_t ld, int64_t rows, int64_t cols,
                   int64_t groups) {
    for (int64_t r = blockIdx.x; r < rows * groups; r += gridDim.x) {
        const uint8_t* s = src + (r / rows) * group_src + (r % rows) * ld_src;
        for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) dst[r * ld + c] = s[c];
    }
}

// Memory of the stream-ordered pool for the length of a call's work.
struct PoolBuffer {
    void* p = nullptr;
    cudaStream_t s;
    explicit PoolBuffer(cudaStream_t st) : s(st) {}
    void* get(size_t n) { PB_CUDA(cudaMallocAsync(&p, n, s)); return p; }
    ~PoolBuffer() { if (p) cudaFreeAsync(p, s); }
};

// The kernel with its shared memory, launched on a grid of clusters of `split` CTAs, or asked how
// many of these clusters the device holds at once.
template <int BT, bool SPLIT>
int tc_kernel(const TcArgs& args, int64_t grid, int split, const CUtensorMap* tmB, const CUtensorMap* tmA, int device,
              cudaStream_t s) {
    using S = Shape<BT>;
    TcArgs p = args;
    const uint32_t fixed = 1024 + 2 * S::kScaleBytes + kBarrierBytes + p.table_bytes;
    p.stages = (int)((227u * 1024u - fixed) / (kABytes + S::kBBytes));       // 3 to 6
    p.split = split;
    static bool ready[64] = {};
    if (device >= 64 || !ready[device]) {
        PB_CUDA(cudaFuncSetAttribute(matmul_fp8_kernel<BT, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
        if (device < 64) ready[device] = true;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(S::kThreads);
    cfg.dynamicSmemBytes = fixed + (size_t)p.stages * (kABytes + S::kBBytes);
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0] = dependent_launch();
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)split;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = SPLIT ? 2 : 1;
    if (!tmB) {
        int n = 0;
        PB_CUDA(cudaOccupancyMaxActiveClusters(&n, matmul_fp8_kernel<BT, SPLIT>, &cfg));
        return n;
    }
    PB_CUDA(cudaLaunchKernelEx(&cfg, matmul_fp8_kernel<BT, SPLIT>, *tmB, *tmA, p));
    return 0;
}

// Clusters of `split` CTAs of the narrow kernels that run at once. (They stay within a GPC,
// so it is fewer than the SMs make: 16 clusters of 8 took two waves.)
int64_t clusters_at_once(int split, int device) {
    static std::atomic<int> known[64][4] = {};
    const int i = split == 2 ? 0 : split == 4 ? 1 : 2;
    int n = device < 64 ? known[device][i].load() : 0;
    if (!n) {
        n = tc_kernel<16, true>(TcArgs{}, split, split, nullptr, nullptr, device, nullptr);
        if (device < 64) known[device][i].store(n);
    }
    return n;
}

template <int CG>
void launch_wide(const TcArgs& args, int64_t tiles, int sms, const CUtensorMap& tmB, const CUtensorMap& tmA, const CUtensorMap& tmO, int device,
                 cudaStream_t s) {
    TcArgs p = args;
    constexpr uint32_t stage = 128 * kBlock + kWideN / CG * kBlock;
    const uint32_t fixed = 1024 + kWideEpi * kWideStage + 2 * kWideScales + kBarrierBytes + p.table_bytes;
    p.stages = (int)std::min<uint32_t>(8, (227u * 1024u - fixed) / stage);
    static bool ready[64] = {};
    if (device >= 64 || !ready[device]) {
        // a build with fewer registers per thread would leave the epilogue waiting for ones that are not there
        cudaFuncAttributes attr;
        PB_CUDA(cudaFuncGetAttributes(&attr, matmul_fp8_wide_kernel<CG>));
        if (attr.numRegs != kWideRegs) fail(ENGINE_ERR_RUNTIME, "matmul_fp8: built with an unexpected number of registers");
        PB_CUDA(cudaFuncSetAttribute(matmul_fp8_wide_kernel<CG>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
        if (device < 64) ready[device] = true;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(std::min<int64_t>(tiles, sms / CG) * CG));
    cfg.blockDim = dim3(kWideThreads);
    cfg.dynamicSmemBytes = fixed + (size_t)p.stages * stage;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0] = dependent_launch();
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = CG;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    PB_CUDA(cudaLaunchKernelEx(&cfg, matmul_fp8_wide_kernel<CG>, tmB, tmA, tmO, p));
}

}  // namespace

namespace {

// Which kernel and tile. wide: 0, or the CTAs per wide tile; else tiles of bt tokens with the
// k-blocks of a tile split over `split` CTAs.
struct Plan { int wide, bt, split; };

// A k-block takes a CTA nearly as long whatever its tile holds, so what counts is how many of
// them the busiest CTA gets. With one weight all shapes are known: of every tile the time of
// the busiest CTA is waves * (k-blocks * time of one + time to store the tile), or with a split
// the k-blocks' and the joining's, and the least wins. The times (us) are fits to a sweep on
// a B200, which they meet within 10% or so; the plan's time is within 9% of the best one's for 469
// shapes of a sweep up to 8192 x 8192 x 8192 (mean 0.5%). Measured, m x n x k, bf16 out: 16 x 4096 x 4096: 16 tokens over 4 CTAs
// 7.5, over 2 9.1, over 1 12.3; 333 x 2048 x 272: 64: 5.3, 32: 5.8, 128: 6.3, wide 6.9; 2000 x 4096 x 1024:
// wide 15.3, 128: 20.9, 64: 23.3. Rows that do not start at multiples of 16 bytes: 2000 x 4097 x 1024: wide
// 19.2, 128: 22.0; f32 4000 x 4097 x 1024: 128: 43.6, 64: 46.4, wide 51.4. Pairs where wide tiles are
// more than one wave: 8192 x 8192 x 4096 267 against 277; 129 x 128256 x 4096 139 against 151. But where an
// odd number of 128-token tiles leaves half of the last pairs empty, single CTAs make fewer waves: 100 x
// 128256 x 4096 103, pairs 138, 128: 107; 300 x 50264 x 4096 86, pairs 115; 640 x 28672 x 8192 159, pairs 180. Over 75
// shapes of 48 to 1000 tokens with 28672 to 151936 weight rows the plan is within 7% of the best (mean 1%), but for
// 100 x 50264 x 4096 with f32 out (56, 128: 50).
// at_once(split): the clusters of `split` CTAs that run at once.
template <typename F>
Plan plan_matmul(const MatmulFp8Args& g, int64_t experts, int sms, bool wide_out, F at_once) {
    if (g.offsets) {
        // The experts' shares are on the GPU; what is known is the average. Measured, as the mean over
        // 15 shapes of the time over the best tile's (8 to 64 experts, even and uneven, 1024 to 2048 wide,
        // 512 to 2048 long, 16-bit output): 8 rows each: 16 tokens 1.00, 32: 1.04; 16 rows: 32: 1.01,
        // 64: 1.14, 16: 1.15; 32 rows: 64: 1.01, 32: 1.09, wide 1.22; 48 rows: 64: 1.02, wide 1.17; 64 rows:
        // wide 1.08, 64: 1.13, 128: 1.15; 256 rows: wide 1.00, 128: 1.24. Output rows that do not start at
        // multiples of 16 bytes cost a wide tile 2.3 more, and 6.5 in 32 bits: 64 rows: 64: 1.04, 128: 1.09,
        // wide 1.18; 96 rows: 128: 1.08, wide 1.14; 128 rows: wide 1.05, 128: 1.08; 512 rows: wide 1.01,
        // 128: 1.09; in 32 bits 512 rows: 128: 1.00, wide 1.26.
        const int64_t r = g.m / experts;
        if (r <= 48) return Plan{0, r <= 8 ? 16 : r <= 20 ? 32 : 64, 1};
        if (wide_out || (r >= 112 && g.out_dtype != ENGINE_F32)) return Plan{1, 128, 1};
        return Plan{0, r <= 80 ? 64 : 128, 1};
    }
    const int64_t nkb = (g.k + kBlock - 1) / kBlock, n_tiles = (g.n + kTileN - 1) / kTileN;
    auto waves = [&](int64_t tiles, int ctas = 1) { return (tiles + sms / ctas - 1) / (sms / ctas); };
    auto wide_tiles = [&](int ctas) { return (g.m + 128 * ctas - 1) / (128 * ctas) * ((g.n + kWideN - 1) / kWideN); };
    // a pair's tile takes as long as a single CTA's, but it has the tokens of two
    const int wide = wide_tiles(1) > sms && waves(wide_tiles(2), 2) <= waves(wide_tiles(1)) ? 2 : 1;
    Plan best{wide, 128, 1};
    double least = (double)waves(wide_tiles(wide), wide) * (nkb * 0.505 + (wide_out ? 2.2 : g.out_dtype == ENGINE_F32 ? 8.7 : 4.5));
    static const struct { int bt; double block, store, join; } kTiles[] = {
        {128, 0.345, 2.3, 5.7}, {64, 0.264, 1.05, 3.1}, {32, 0.24, 0.65, 2.2}, {16, 0.237, 0.55, 1.7}};
    for (const auto& c : kTiles) {
        const int64_t tiles = (g.m + c.bt - 1) / c.bt * n_tiles;
        for (int split = 1; split <= 8; split *= 2) {
            if (split > 1 && (nkb < 2 * split || tiles * split > sms || tiles > at_once(split))) break;
            const double t = split == 1 ? (double)waves(tiles) * (nkb * c.block + c.store) : (double)((nkb + split - 1) / split) * c.block + c.join;
            if (t < least) { least = t; best = Plan{0, c.bt, split}; }
        }
    }
    return best;
}

}  // namespace

void matmul_fp8_plan(const MatmulFp8Args& g, bool aligned_out, int sms, const int32_t (&clusters)[3], int32_t (&plan)[3]) {
    const Plan p = plan_matmul(g, g.offsets ? g.experts : 1, sms, aligned_out, [&](int split) { return clusters[split == 2 ? 0 : split == 4 ? 1 : 2]; });
    plan[0] = p.wide; plan[1] = p.wide ? 128 * p.wide : p.bt; plan[2] = p.split;
}

void launch_matmul_fp8(const MatmulFp8Args& g, cudaStream_t s) {
    if (g.m == 0 || g.n == 0) return;
    if (g.k == 0) {
        const size_t e = g.out_dtype == ENGINE_F32 ? 4 : 2;
        PB_CUDA(cudaMemset2DAsync(g.out, (size_t)(g.m > 1 ? g.ldo : g.n) * e, 0, (size_t)g.n * e, (size_t)g.m, s));
        return;
    }
    int device = 0;
    PB_CUDA(cudaGetDevice(&device));
    static int sm_count[64] = {};
    int sms = device < 64 ? sm_count[device] : 0;
    if (!sms) {
        PB_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
        if (device < 64) sm_count[device] = sms;
    }

    // TMA reads rows that start at multiples of 16 bytes and do not overlap; others are
    // copied into such rows first.
    const int64_t experts = g.offsets ? g.experts : 1;
    const int64_t k16 = (g.k + 15) & ~int64_t(15);
    auto plain = [&](const void* p, int64_t ld, int64_t rows) {
        return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows <= 1 || (ld % 16 == 0 && ld >= g.k));
    };
    PoolBuffer mem_a(s), mem_b(s);
    const void* a = g.a;
    const void* b = g.b;
    int64_t lda = g.m > 1 ? g.lda : k16, ldb = g.n > 1 ? g.ldb : k16, b_expert = experts > 1 ? g.b_expert : ldb * g.n;
    if (!plain(g.a, g.lda, g.m)) {
        a = mem_a.get((size_t)(g.m * k16));
        repack_rows_kernel<<<(unsigned)std::min<int64_t>(g.m, 16 * sms), 256, 0, s>>>(
            static_cast<const uint8_t*>(g.a), g.lda, 0, static_cast<uint8_t*>(mem_a.p), k16, g.m, g.k, 1);
        PB_CUDA(cudaGetLastError());
        lda = k16;
    }
    if (!plain(g.b, g.ldb, g.n) || (experts > 1 && (g.b_expert % 16 || g.b_expert < (g.n - 1) * ldb + g.k))) {
        b = mem_b.get((size_t)(experts * g.n * k16));
        repack_rows_kernel<<<(unsigned)std::min<int64_t>(experts * g.n, 16 * sms), 256, 0, s>>>(
            static_cast<const uint8_t*>(g.b), g.ldb, g.b_expert, static_cast<uint8_t*>(mem_b.p), k16, g.n, g.k, experts);
        PB_CUDA(cudaGetLastError());
        ldb = k16;
        b_expert = g.n * k16;
    }

    TcArgs p{};
    p.offsets = g.offsets;
    p.experts = (int)experts;
    p.m = (int)g.m;
    p.n = (int)g.n;
    p.nkb = (int)((g.k + kBlock - 1) / kBlock);
    p.n_tiles = (int)((g.n + kTileN - 1) / kTileN);
    p.sa = g.a_scales; p.lda_scales = g.lda_scales;
    p.sb = g.b_scales; p.ldb_scales = g.ldb_scales; p.sb_expert = g.offsets ? g.b_scales_expert : 0;
    p.out = g.out; p.ldo = g.ldo; p.out_dtype = g.out_dtype;
    p.table_bytes = g.offsets ? (uint32_t)(12 * experts + 15) & ~15u : 0;
    p.err = device_error_word(device);
    p.wait_limit = 1000000000LL;

    p.wide_out = reinterpret_cast<uintptr_t>(g.out) % 16 == 0 && (g.m <= 1 || g.ldo * (g.out_dtype == ENGINE_F32 ? 4 : 2) % 16 == 0);
    // TMA cuts the end of a row to whole 16 bytes: it would reach beyond rows that end inside them
    p.tma_end = !p.wide_out ? 0 : g.n * (g.out_dtype == ENGINE_F32 ? 4 : 2) % 16 ? p.n : 0x7FFFFFFF;
    const Plan plan = plan_matmul(g, experts, sms, p.wide_out, [&](int split) { return clusters_at_once(split, device); });
    const int wide = plan.wide, bt = wide ? 128 : plan.bt;
    const int tokens = wide ? 128 * wide : bt;
    p.m_tiles = (int)((g.m + tokens - 1) / tokens);

    CUtensorMap tmA, tmB;
    {
        const uint64_t dims[2] = {(uint64_t)g.k, (uint64_t)g.m}, st[1] = {(uint64_t)lda};
        const uint32_t box[2] = {kBlock, (uint32_t)bt};
        if (!encode_box_map(&tmA, 1, 2, a, dims, st, box, 128)) fail(ENGINE_ERR_INVALID_ARG, "matmul_fp8: tensor map of a refused");
    }
    {
        const uint64_t dims[3] = {(uint64_t)g.k, (uint64_t)g.n, (uint64_t)experts}, st[2] = {(uint64_t)ldb, (uint64_t)b_expert};
        const uint32_t box[3] = {kBlock, (uint32_t)(wide == 1 ? kWideN : kTileN), 1};
        if (!encode_box_map(&tmB, 1, 3, b, dims, st, box, 128)) fail(ENGINE_ERR_INVALID_ARG, "matmul_fp8: tensor map of b refused");
    }

    if (wide) {
        p.n_tiles = (int)((g.n + kWideN - 1) / kWideN);
        const int64_t tiles = (g.offsets ? std::min<int64_t>(g.m, experts + g.m / tokens) : p.m_tiles) * p.n_tiles;
        CUtensorMap tmO = tmA;
        if (p.wide_out) {
            const uint64_t e = g.out_dtype == ENGINE_F32 ? 4 : 2;
            const uint64_t dims[2] = {(uint64_t)g.n * e, (uint64_t)g.m}, st[1] = {(uint64_t)(g.m > 1 ? g.ldo : (g.n + 15) / 16 * 16) * e};
            const uint32_t box[2] = {128, 32};
            if (!encode_box_map(&tmO, 1, 2, g.out, dims, st, box, 128)) fail(ENGINE_ERR_INVALID_ARG, "matmul_fp8: tensor map of the output refused");
        }
        if (wide == 1) launch_wide<1>(p, tiles, sms, tmB, tmA, tmO, device, s);
        else launch_wide<2>(p, tiles, sms, tmB, tmA, tmO, device, s);
        return;
    }
    // Token tiles there can be at most: one per expert with rows, and one per full tile.
    const int64_t tiles = (g.offsets ? std::min<int64_t>(g.m, experts + g.m / bt) : p.m_tiles) * p.n_tiles;
    const int split = plan.split;
    const int64_t grid = split > 1 ? tiles * split : std::min<int64_t>(tiles, sms);
    switch (bt) {
        case 16: split > 1 ? tc_kernel<16, true>(p, grid, split, &tmB, &tmA, device, s) : tc_kernel<16, false>(p, grid, 1, &tmB, &tmA, device, s); break;
        case 32: split > 1 ? tc_kernel<32, true>(p, grid, split, &tmB, &tmA, device, s) : tc_kernel<32, false>(p, grid, 1, &tmB, &tmA, device, s); break;
        case 64: split > 1 ? tc_kernel<64, true>(p, grid, split, &tmB, &tmA, device, s) : tc_kernel<64, false>(p, grid, 1, &tmB, &tmA, device, s); break;
        default: split > 1 ? tc_kernel<128, true>(p, grid, split, &tmB, &tmA, device, s) : tc_kernel<128, false>(p, grid, 1, &tmB, &tmA, device, s); break;
    }
}

}  // namespace pb
