// One token per row of logits: temperature, top-k, top-p and min-p, with the randomness
// given as exponential variates.
//
// With x the row (NaN counts as -inf), M its maximum and T the temperature,
//   w_i = exp((x_i - M) / T),  Z = sum of w over the whole row,
// and tokens ordered by falling x, equal ones by rising index, a token is kept if
//   * fewer than top_k tokens come before it,
//   * the mass before it is less than top_p * Z,
//   * w >= min_p (the largest w is 1), and w > 0;
// each test looks at the whole row, so the order of the filters does not matter, and
// the first token is always kept. The kept tokens race: the token with the largest
// w_i / e_i wins (lowest index among equals). For e_i independent exponential variates
// that is token i with probability w_i / (sum of the kept w).
//
// The cut of the order is never searched for as such. What is kept is a prefix of the
// order, so the winner of a race over any longer prefix is the winner if it is itself
// kept, and if it is not, everything from it on is out. A round races the tokens before
// `hi`, counts the tokens and the mass before the winner, and ends or moves `hi` to the
// winner. The same counting pass also tests the midpoint between the last position
// known to be kept and `hi`, so rounds are bounded by the bits of a position whatever
// the variates are; with random ones there are one or two.
//
// A row is read once into the shared memory of a cluster. What bounds it is not that read but
// the phases after it, each a barrier and an exchange over the cluster's CTAs (1 to 1.3 us):
// 256 x 131072 bf16 with top-k, top-p and min-p 51 us (1.3 TB/s; the read alone 10), one row of
// 32000 6.4 us. So rows are spread over CTAs to have all of them in flight at once, candidates are
// counted before they are listed, and what one CTA can finish alone is sent to one.
#include <algorithm>
#include <cuda_fp16.h>

#include "common.h"
#include "device_common.cuh"
#include "row_vec.cuh"

namespace pb {

namespace {

constexpr int kThreads = 1024;
constexpr float kLog2e = 1.4426950408889634f;

template <typename T> __device__ __forceinline__ float logit(T v);
template <> __device__ __forceinline__ float logit(float v) { return v; }
template <> __device__ __forceinline__ float logit(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float logit(__nv_bfloat16 v) { return __bfloat162float(v); }

// NaN -> -inf, -0 -> +0 (the two zeros are equal tokens)
__device__ __forceinline__ float clean(float v) { return v == v ? v + 0.0f : -INFINITY; }

// Position in the order: falling value, then rising index; unsigned, ascending.
__device__ __forceinline__ uint64_t position(float v, uint32_t idx, int shift) {
    const uint32_t b = __float_as_uint(v);
    const uint32_t up = b & 0x80000000u ? ~b : b | 0x80000000u;     // rises with v
    return ((uint64_t)(~up) << shift) | idx;
}

// The logit of a position (-inf where no number has it).
__device__ __forceinline__ float value_of(uint64_t at, int shift) {
    const uint32_t up = ~(uint32_t)(at >> shift);
    const float v = __uint_as_float(up & 0x80000000u ? up & 0x7FFFFFFFu : ~up);
    return v == v ? v : -INFINITY;
}

// log2(e) / T, within the numbers: neither 0 * inf from an infinite T nor inf * 0 from one below 2^-127
// may meet a difference of logits.
__device__ __forceinline__ float factor(float temp) { return fminf(fmaxf(kLog2e / temp, 1.17549435e-38f), 3.40282347e38f); }

// A variate that races: not NaN and without a sign. -0, which -log(1 - u) gives for u = 0, would make
// w / e negative.
__device__ __forceinline__ bool races(float e) { return __float_as_uint(e) <= 0x7F800000u; }

struct Race {
    float key = -1.0f;
    uint32_t idx = 0xFFFFFFFFu;
    float x = 0.0f;
    __device__ __forceinline__ void take(float k, uint32_t i, float v) {
        if (k > key || (k == key && i < idx)) { key = k; idx = i; x = v; }
    }
};

__device__ __forceinline__ float block_max(float v, float* buf) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    v = buf[threadIdx.x & 31];
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
    return v;
}

template <typename V>
__device__ __forceinline__ V block_sum(V v, V* buf) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    v = buf[threadIdx.x & 31];
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}

__device__ __forceinline__ Race warp_race(Race r) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float k = __shfl_xor_sync(~0u, r.key, o);
        const uint32_t i = __shfl_xor_sync(~0u, r.idx, o);
        const float x = __shfl_xor_sync(~0u, r.x, o);
        r.take(k, i, x);
    }
    return r;
}

// A CTA per row that reads the row again in every pass, for rows that a cluster's shared memory
// does not hold (8 slices of 200 KB; 16 x 409700 f32: 579 us, 16 x 409600 by clusters 31).
template <typename T>
__global__ void __launch_bounds__(kThreads)
sample_rows_kernel(SampleArgs a, int shift) {
    __shared__ float fbuf[32];
    __shared__ int ibuf[32];
    __shared__ float rkey[32], rx[32];
    __shared__ uint32_t ridx[32];
    const int64_t row = blockIdx.x;
    const T* lg = static_cast<const T*>(a.logits) + row * a.logits_stride;
    const float* noise = a.noise + row * a.noise_stride;
    const uint32_t V = (uint32_t)a.vocab;
    float temp = a.temperature ? a.temperature[row] : 1.0f;
    int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    const float floor_w = a.min_p ? a.min_p[row] : 0.0f;
    if (!(temp > 0.0f)) { temp = 1.0f; k = 1; }
    if (k <= 0) k = 0x7FFFFFFF;
    const bool by_mass = !(p >= 1.0f);

    float mx = -INFINITY;
    uint32_t first = 0xFFFFFFFFu;
    for (uint32_t i = threadIdx.x; i < V; i += kThreads) mx = fmaxf(mx, clean(logit<T>(lg[i])));
    mx = block_max(mx, fbuf);
    if (mx == -INFINITY) {                     // nothing to choose from
        if (threadIdx.x == 0) {
            a.tokens[row] = -1;
            if (a.probs) a.probs[row] = 0.0f;
        }
        return;
    }
    const float c = factor(temp);
    auto weight = [&](float x) {
        if (x == mx) return 1.0f;              // also inf - inf
        if (x == -INFINITY) return 0.0f;
        return exp2f((x - mx) * c);
    };
    float z = 0.0f;
    for (uint32_t i = threadIdx.x; i < V; i += kThreads) {
        const float x = clean(logit<T>(lg[i]));
        z += weight(x);
        if (x == mx && first == 0xFFFFFFFFu) first = i;
    }
    z = block_sum(z, fbuf);
    // lowest index of the maximum
    {
        Race r;
        if (first != 0xFFFFFFFFu) r.take(1.0f, first, mx);
        r = warp_race(r);
        if ((threadIdx.x & 31) == 0) ridx[threadIdx.x >> 5] = r.idx;
        __syncthreads();
        first = ridx[0];
        for (int i = 1; i < 32; ++i) first = min(first, ridx[i]);
        __syncthreads();
    }
    const float limit = p * z;
    uint64_t lo = position(mx, first, shift), hi = ~0ull;
    Race won;
    for (;;) {
        Race r;
        for (uint32_t i = threadIdx.x; i < V; i += kThreads) {
            const float x = clean(logit<T>(lg[i]));
            const uint64_t at = position(x, i, shift);
            if (at >= hi) continue;
            const float w = weight(x);
            if (!(w >= floor_w && w > 0.0f) && i != first) continue;
            const float e = noise[i];
            if (races(e)) r.take(w / e, i, x);
        }
        r = warp_race(r);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) {
            rkey[threadIdx.x >> 5] = r.key;
            ridx[threadIdx.x >> 5] = r.idx;
            rx[threadIdx.x >> 5] = r.x;
        }
        __syncthreads();
        r = Race();
        r.take(rkey[threadIdx.x & 31], ridx[threadIdx.x & 31], rx[threadIdx.x & 31]);
        won = warp_race(r);
        if (won.idx == 0xFFFFFFFFu) { won.idx = first; won.x = mx; }     // no usable variate
        const uint64_t at_won = position(won.x, won.idx, shift);
        if (at_won <= lo || (k == 0x7FFFFFFF && !by_mass)) break;
        const uint64_t mid = lo + (hi - lo) / 2;
        int n_won = 0, n_mid = 0;
        float m_won = 0.0f, m_mid = 0.0f;
        for (uint32_t i = threadIdx.x; i < V; i += kThreads) {
            const float x = clean(logit<T>(lg[i]));
            const uint64_t at = position(x, i, shift);
            if (at >= at_won && at >= mid) continue;
            const float w = weight(x);
            if (at < at_won) { ++n_won; m_won += w; }
            if (at < mid) { ++n_mid; m_mid += w; }
        }
        n_won = block_sum(n_won, ibuf);
        n_mid = block_sum(n_mid, ibuf);
        m_won = block_sum(m_won, fbuf);
        m_mid = block_sum(m_mid, fbuf);
        if (n_won < k && (!by_mass || m_won < limit)) break;
        hi = at_won;
        if (n_mid < k && (!by_mass || m_mid < limit)) lo = max(lo, mid);
        else hi = min(hi, mid);
    }
    if (threadIdx.x == 0) {
        a.tokens[row] = (int32_t)won.idx;
        if (a.probs) a.probs[row] = (won.x == mx ? 1.0f : expf((won.x - mx) / temp)) / z;
    }
}

// ---------------------------------------------------------------------------
// A cluster per row: the row is read once, kept in the CTAs' shared memory, and every
// further pass reads it there.
// ---------------------------------------------------------------------------
constexpr int kSlice = 512;             // threads of a CTA
constexpr int kResident = 2;            // CTAs an SM
constexpr int kWarps = kSlice / 32;
constexpr int kBins = 256;
constexpr int kList = 512;              // candidates that are listed at most (one thread each, at least)
constexpr int kMostCtas = 8;
constexpr float kBinsPerOctave = 16.0f; // the bins cover w from 1 down to 2^-16

template <typename T> constexpr int kVec = 16 / (int)sizeof(T);
template <typename T> constexpr bool kIsHalf = false;
template <> constexpr bool kIsHalf<__half> = true;

// A vector of -inf, and the larger of two vectors element by element (a NaN gives way).
template <typename T> __device__ __forceinline__ uint4 vec_none() {
    const uint32_t w = sizeof(T) == 4 ? 0xFF800000u : kIsHalf<T> ? 0xFC00FC00u : 0xFF80FF80u;
    return make_uint4(w, w, w, w);
}
template <typename T> __device__ __forceinline__ uint32_t word_max(uint32_t a, uint32_t b);
template <> __device__ __forceinline__ uint32_t word_max<float>(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
}
template <> __device__ __forceinline__ uint32_t word_max<__half>(uint32_t a, uint32_t b) {
    const __half2 m = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
}
template <> __device__ __forceinline__ uint32_t word_max<__nv_bfloat16>(uint32_t a, uint32_t b) {
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
}
template <typename T> __device__ __forceinline__ uint4 vec_max_of(const uint4& a, const uint4& b) {
    return make_uint4(word_max<T>(a.x, b.x), word_max<T>(a.y, b.y), word_max<T>(a.z, b.z), word_max<T>(a.w, b.w));
}
template <typename T> __device__ __forceinline__ void unpack(const uint4& v, float (&x)[kVec<T>]);
template <> __device__ __forceinline__ void unpack<float>(const uint4& v, float (&x)[4]) {
    x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
}
template <> __device__ __forceinline__ void unpack<__half>(const uint4& v, float (&x)[8]) {
    const __half2* w = reinterpret_cast<const __half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
template <> __device__ __forceinline__ void unpack<__nv_bfloat16>(const uint4& v, float (&x)[8]) {
    const uint32_t* w = &v.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
template <typename T> __device__ __forceinline__ float vec_max(const uint4& v) {
    const uint32_t m = word_max<T>(word_max<T>(v.x, v.y), word_max<T>(v.z, v.w));
    if (sizeof(T) == 4) return __uint_as_float(m);
    float x[kVec<T>];
    unpack<T>(make_uint4(m, m, m, m), x);
    return fmaxf(x[0], x[1]);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_barrier() {
    cluster_arrive();
    cluster_wait();
}
__device__ __forceinline__ uint32_t remote_u32(const void* p, uint32_t rank) {
    uint32_t v;
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.u32 %0, [a];\n\t}"
                 : "=r"(v) : "r"(smem_u32(p)), "r"(rank) : "memory");
    return v;
}
__device__ __forceinline__ void remote_store(void* p, uint32_t rank, uint4 v) {
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, %1;\n\tst.shared::cluster.v4.u32 [a], {%2, %3, %4, %5};\n\t}"
                 ::"r"(smem_u32(p)), "r"(rank), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void remote_store(void* p, uint32_t rank, uint2 v) {
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, %1;\n\tst.shared::cluster.v2.u32 [a], {%2, %3};\n\t}"
                 ::"r"(smem_u32(p)), "r"(rank), "r"(v.x), "r"(v.y) : "memory");
}

// The warp-wide joins, over the four words that CTAs tell each other. Whole numbers and
// the race go through the integer reduction instruction; the order of float sums is fixed.
struct JoinMax {                // x: a float's bits
    static __device__ __forceinline__ uint4 none() { return make_uint4(__float_as_uint(-INFINITY), 0, 0, 0); }
    static __device__ __forceinline__ uint4 warp(uint4 w) {
        int i = (int)w.x;
        i ^= (i >> 31) & 0x7FFFFFFF;            // orders as the float does
        i = __reduce_max_sync(~0u, i);
        i ^= (i >> 31) & 0x7FFFFFFF;
        w.x = (uint32_t)i;
        return w;
    }
};
__device__ __forceinline__ uint32_t warp_sum(uint32_t bits) {
    float v = __uint_as_float(bits);
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return __float_as_uint(v);
}
struct JoinRace {               // x: the race's key + 1 (0: nobody), y: token, z: its logit's bits, w: mass
    static __device__ __forceinline__ uint4 none() { return make_uint4(0, 0xFFFFFFFFu, 0, 0); }
    static __device__ __forceinline__ uint4 warp(uint4 w) {
        const uint32_t key = __reduce_max_sync(~0u, w.x);
        const uint32_t idx = w.x == key ? w.y : 0xFFFFFFFFu;
        const uint32_t best = __reduce_min_sync(~0u, idx);
        const int from = __ffs(__ballot_sync(~0u, idx == best)) - 1;
        return make_uint4(key, best, __shfl_sync(~0u, w.z, from), warp_sum(w.w));
    }
};
struct JoinCounts {             // x, y: tokens, z, w: masses
    static __device__ __forceinline__ uint4 none() { return make_uint4(0, 0, 0, 0); }
    static __device__ __forceinline__ uint4 warp(uint4 w) {
        return make_uint4(__reduce_add_sync(~0u, w.x), __reduce_add_sync(~0u, w.y), warp_sum(w.z), warp_sum(w.w));
    }
};
struct JoinLeast {              // x: a token
    static __device__ __forceinline__ uint4 none() { return make_uint4(0xFFFFFFFFu, 0, 0, 0); }
    static __device__ __forceinline__ uint4 warp(uint4 w) {
        w.x = __reduce_min_sync(~0u, w.x);
        return w;
    }
};
struct JoinList {               // x: candidates, y: most of a CTA, w: mass
    static __device__ __forceinline__ uint4 none() { return make_uint4(0, 0, 0, 0); }
    static __device__ __forceinline__ uint4 warp(uint4 w) {
        return make_uint4(__reduce_add_sync(~0u, w.x), __reduce_max_sync(~0u, w.y), 0, warp_sum(w.w));
    }
};

struct Shared {
    uint4 part[kWarps];
    uint4 told[2][kMostCtas];   // every CTA's word of the last two joins
    uint2 mine[kList];          // this CTA's candidates: logit, token
    union {
        uint32_t hist[kBins];   // tokens per bin of w
        uint2 list[kList];      // CTA 0: the row's candidates, kList / CTAs places for each
    };
    uint32_t count[kBins];      // tokens of bins <= b, over the row
    float most[kBins];          // upper bound of their mass
    float scan[3][kBins / 32];
    uint32_t listed;            // candidates of this CTA, kept or not
    uint32_t first;
    int cut;
};

// One join over the cluster: every CTA's word goes to every other, and every thread gets
// the result. Two slots suffice: a CTA writes a slot again only after the next join's
// barrier, which every CTA reaches after it has read this one.
template <typename J>
__device__ __forceinline__ uint4 cluster_join(uint4 w, Shared& sh, int& turn, int ctas, uint32_t rank) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    w = J::warp(w);
    if (lane == 0) sh.part[warp] = w;
    __syncthreads();
    if (warp == 0) {
        w = J::warp(lane < kWarps ? sh.part[lane] : J::none());
        if (lane < ctas) remote_store(&sh.told[turn][rank], (uint32_t)lane, w);
        __syncwarp();
    }
    cluster_barrier();
    w = lane < ctas ? sh.told[turn][lane] : J::none();
    turn ^= 1;
    return J::warp(w);
}

// The row's token from its candidates (all tokens that can be kept are among the n of
// them, and those before them in the order), by CTA 0 alone: each candidate counts the
// candidates and the mass before it. Masses are whole numbers, so that the order in
// which the list was filled does not matter. If no kept token has a usable variate the
// first one is the answer. The slice is not needed any more: positions and masses (w * 2^40)
// lie over it.
__device__ __forceinline__ uint4 choose(Shared& sh, uint64_t* at_of, int n, int turn, int ctas, int k, bool by_mass, float limit, float top,
                                        float c, const float* noise, int shift) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int room = kList / ctas;
    uint64_t* const mass_of = at_of + kList;
    if (tid < n) {
        int r = 0, slot = tid;
        while (slot >= (int)sh.told[turn][r].x) slot -= (int)sh.told[turn][r++].x;
        const uint2 e = sh.list[r * room + slot];
        const float x = __uint_as_float(e.x);
        sh.mine[tid] = e;
        at_of[tid] = position(x + 0.0f, e.y, shift);
        mass_of[tid] = (uint64_t)(ex2((x - top) * c) * 1099511627776.0f);
    }
    __syncthreads();
    int g = 1;                              // threads per candidate
    while (g < 32 && n * g * 2 <= kSlice) g *= 2;
    const int i = tid / g;
    uint4 race = JoinRace::none();
    float e = -1.0f;
    uint2 own = make_uint2(0, 0);
    if (i < n) {
        own = sh.mine[i];
        if (tid % g == 0) e = __ldg(noise + own.y);
    }
    const uint64_t at = i < n ? at_of[i] : 0;
    uint32_t before = 0;
    unsigned long long mass = 0;
    for (int j = tid % g; j < n; j += g)
        if (at_of[j] < at) { ++before; mass += mass_of[j]; }
    for (int o = g >> 1; o; o >>= 1) {
        before += __shfl_xor_sync(~0u, before, o);
        mass += __shfl_xor_sync(~0u, mass, o);
    }
    if (i < n && tid % g == 0) {
        if (before == 0) sh.first = own.y;
        const bool kept = before == 0 || ((int)before < k && (!by_mass || (double)mass < (double)limit * 1099511627776.0));
        if (kept && races(e))
            race = make_uint4(__float_as_uint(__fdividef(ex2((__uint_as_float(own.x) - top) * c), e)) + 1, own.y, own.x, 0);
    }
    race = JoinRace::warp(race);
    if (lane == 0) sh.part[warp] = race;
    __syncthreads();
    race = JoinRace::warp(lane < kWarps ? sh.part[lane] : JoinRace::none());
    if (!race.x) { race.y = sh.first; race.z = __float_as_uint(top); }
    return race;
}

template <typename T>
__global__ void __launch_bounds__(kSlice, kResident)
sample_cluster_kernel(SampleArgs a, int shift, int ctas) {
    constexpr int VEC = kVec<T>;
    extern __shared__ uint4 slice[];
    __shared__ Shared sh;
    const int tid = threadIdx.x;
    uint32_t rank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    grid_trigger();
    grid_wait();
    const int64_t row = blockIdx.x / ctas;
    const T* lg = static_cast<const T*>(a.logits) + row * a.logits_stride;
    const float* noise = a.noise + row * a.noise_stride;
    const uint32_t V = (uint32_t)a.vocab;
    float temp = a.temperature ? a.temperature[row] : 1.0f;
    int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    float floor_w = a.min_p ? a.min_p[row] : 0.0f;
    if (!(temp > 0.0f)) { temp = 1.0f; k = 1; }
    if (floor_w != floor_w) floor_w = INFINITY;         // no w reaches it
    const bool by_count = k > 0, by_mass = !(p >= 1.0f);
    if (!by_count) k = 0x7FFFFFFF;

    // Vector v holds the elements from v * VEC on (-inf past the end), wherever the row
    // starts in memory, so that sums do not depend on that.
    const uint32_t nv = (V + VEC - 1) / VEC;
    const uint32_t v0 = (uint32_t)((uint64_t)nv * rank / ctas), all = (uint32_t)((uint64_t)nv * (rank + 1) / ctas) - v0;
    const uint32_t i_own = v0 * VEC + tid * VEC;        // first element of this thread's first vector

    cluster_arrive();                   // answered below: before memory of another CTA is written, it has started
    const RowLoader<T> load(lg, V, vec_none<T>().x & (sizeof(T) == 4 ? ~0u : 0xFFFFu));
    float top;
    {
        uint4 m = vec_none<T>();
        const uint4* src = load.base + v0;
        auto put = [&](uint32_t v, uint4 q) {
            q = vec_max_of<T>(q, vec_none<T>());        // NaN -> -inf
            slice[v] = q;
            m = vec_max_of<T>(m, q);
        };
        // Several loads per thread are under way before the first is used: 8 vectors of an aligned
        // row, or 4 pairs of one that is not. The row's first and last vectors go one by one.
        uint32_t rest;
        if (load.aligned()) {
            rest = min(all, max(load.whole(), v0) - v0);
            for (uint32_t v = tid; v < rest; v += 8 * kSlice) {
                uint4 q[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (v + i * kSlice < rest) q[i] = __ldg(src + v + i * kSlice);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (v + i * kSlice < rest) put(v + i * kSlice, q[i]);
            }
        } else {
            rest = min(all, max(load.inner(), v0) - v0);
            const uint32_t start = v0 == 0 ? 1 : 0;
            if (start && tid == 0 && all) put(0, load(0));
            for (uint32_t v = start + tid; v < rest; v += 4 * kSlice) {
                uint4 lo[4], hi[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (v + i * kSlice < rest) {
                        lo[i] = __ldg(src + v + i * kSlice);
                        hi[i] = __ldg(src + v + i * kSlice + 1);
                    }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (v + i * kSlice < rest) put(v + i * kSlice, load.shifted(lo[i], hi[i]));
            }
            rest = max(rest, start);
        }
        for (uint32_t v = rest + tid; v < all; v += kSlice) put(v, load(v0 + v));
        for (int b = tid; b < kBins; b += kSlice) sh.hist[b] = 0;
        if (tid == 0) sh.listed = 0;
        top = vec_max<T>(m) + 0.0f;
    }
    int turn = 0;
    cluster_wait();
    top = __uint_as_float(cluster_join<JoinMax>(make_uint4(__float_as_uint(top), 0, 0, 0), sh, turn, ctas, rank).x);
    if (top == -INFINITY) {             // nothing to choose from
        if (rank == 0 && tid == 0) {
            a.tokens[row] = -1;
            if (a.probs) a.probs[row] = 0.0f;
        }
        return;
    }
    if (top == INFINITY) {              // infinite logits share the mass: 0 for them, -inf for the rest
        for (uint32_t v = tid; v < all; v += kSlice) {
            uint4 q = slice[v];
            T* e = reinterpret_cast<T*>(&q);
            for (int j = 0; j < VEC; ++j) e[j] = logit<T>(e[j]) == INFINITY ? T(0.0f) : T(-INFINITY);
            slice[v] = q;
        }
        top = 0.0f;
    }

    const float c = factor(temp);       // w = 2^y with y = (x - top) * log2(e) / T
    auto weight = [&](float x) { return ex2((x - top) * c); };
    auto finish = [&](uint32_t token, float x, float z) {
        a.tokens[row] = (int32_t)token;
        if (a.probs) a.probs[row] = (x == top ? 1.0f : expf((x - top) / temp)) / z;
    };

    // What the pass that sums Z does beside it:
    //   race   no filter: every token races
    //   list   a min_p that cuts at 2^-6 or above: the tokens that it leaves are listed
    //   count  other filters: tokens are counted in bins of w, to find how far down the
    //          order the filters can reach
    //   first  temperature 0: the lowest index of the largest logit
    enum { kRace, kListing, kCount, kFirst };
    const int mode = k == 1 ? kFirst : floor_w >= 0.015625f ? kListing : by_count || by_mass || floor_w > 0.0f ? kCount : kRace;
    const float least_w = fmaxf(floor_w, 1.17549435e-38f);     // of the tokens that race (w > 0)
    uint4 race = JoinRace::none();
    // The race of the tokens that weigh(vector, its first token, w[]) gives a w of least_w or more:
    // the variates of 16 tokens per thread are requested before the first is used.
    auto hold_race = [&](auto&& weigh) {
        constexpr int U = 16 / VEC;
        for (uint32_t v = tid; v < all; v += U * kSlice) {
            float wx[U][VEC], e[U][VEC];
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) wx[u][j] = 0.0f;
                if (v + u * kSlice < all) weigh(slice[v + u * kSlice], (v0 + v + u * kSlice) * VEC, wx[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    e[u][j] = wx[u][j] >= least_w ? __ldg(noise + (v0 + v + u * kSlice) * VEC + j) : -1.0f;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    if (!races(e[u][j])) continue;
                    const uint32_t key = __float_as_uint(__fdividef(wx[u][j], e[u][j])) + 1;
                    const uint32_t i = (v0 + v + u * kSlice) * VEC + j;
                    if (key > race.x || (key == race.x && i < race.y)) {
                        race.x = key;
                        race.y = i;
                        race.z = __float_as_uint(logit<T>(reinterpret_cast<const T*>(slice)[(v + u * kSlice) * VEC + j]));
                    }
                }
        }
    };
    auto list = [&](float x, uint32_t i) {
        asm volatile("prefetch.global.L2 [%0];" ::"l"(noise + i));      // CTA 0 wants it soon
        const uint32_t slot = atomicAdd(&sh.listed, 1u);
        if (slot < kList) sh.mine[slot] = make_uint2(__float_as_uint(x), i);
    };
    float z = 0.0f;
    uint32_t first = 0xFFFFFFFFu;
    // a vector's exponents and w, and its part of Z
    auto weigh_all = [&](const uint4& q, float (&x)[VEC], float2 (&y)[VEC / 2], float (&wx)[VEC]) {
        unpack<T>(q, x);
        float2 zz = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
            y[j / 2] = __fmul2_rn(__fadd2_rn(make_float2(x[j], x[j + 1]), make_float2(-top, -top)), make_float2(c, c));
            wx[j] = ex2(y[j / 2].x);
            wx[j + 1] = ex2(y[j / 2].y);
            zz = __fadd2_rn(zz, make_float2(wx[j], wx[j + 1]));
        }
        z += zz.x + zz.y;
    };
    if (mode == kRace) {
        hold_race([&](const uint4& q, uint32_t, float (&wx)[VEC]) {
            float x[VEC];
            float2 y[VEC / 2];
            weigh_all(q, x, y, wx);
        });
    }
    for (uint32_t v = tid, i0 = i_own; mode != kRace && v < all; v += kSlice, i0 += kSlice * VEC) {
        float x[VEC], wx[VEC];
        float2 y[VEC / 2];
        weigh_all(slice[v], x, y, wx);
        if (mode == kListing) {
            float m = wx[0];
#pragma unroll
            for (int j = 1; j < VEC; ++j) m = fmaxf(m, wx[j]);
            if (m >= least_w) {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (wx[j] >= least_w) list(x[j], i0 + j);
            }
        } else if (mode == kCount) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float t = (j & 1 ? y[j / 2].y : y[j / 2].x) * -kBinsPerOctave;
                if (t < (float)kBins) atomicAdd(&sh.hist[(int)t], 1u);
            }
        } else if (first == 0xFFFFFFFFu) {
#pragma unroll
            for (int j = VEC - 1; j >= 0; --j)
                if (x[j] == top) first = i0 + j;
        }
    }

    const int room = kList / ctas;
    // this CTA's candidates to CTA 0; call with every thread, then join
    auto send = [&]() {
        __syncthreads();
        const uint32_t n = min(sh.listed, (uint32_t)room);
        for (uint32_t i = tid; i < n; i += kSlice) remote_store(&sh.list[rank * room + i], 0u, sh.mine[i]);
    };
    uint4 won = JoinRace::none();
    bool done = false, have = false;
    float limit;
    if (mode == kListing) {
        send();
        const uint4 w = cluster_join<JoinList>(make_uint4(tid ? 0 : sh.listed, tid ? 0 : sh.listed, 0, __float_as_uint(z)), sh, turn, ctas, rank);
        z = __uint_as_float(w.w);
        limit = p * z;
        if (w.x && w.y <= (uint32_t)room) {
            if (rank) return;
            won = choose(sh, reinterpret_cast<uint64_t*>(slice), (int)w.x, turn ^ 1, ctas, k, by_mass, limit, top, c, noise, shift);
            if (tid == 0) finish(won.y, __uint_as_float(won.z), z);
            return;
        }
        done = !w.x;            // min_p above 1: the first token
    } else {
        race.w = __float_as_uint(z);
        won = cluster_join<JoinRace>(race, sh, turn, ctas, rank);
        z = __uint_as_float(won.w);
        limit = p * z;
        done = mode != kCount;
    }
    if (mode == kCount) {
        // bin b holds tokens with w in (2^-((b + 1) / 16), 2^-(b / 16)]
        const int warp = tid >> 5, lane = tid & 31;
        float cnt = 0.0f, least = 0.0f, most = 0.0f;
        if (tid == 0) sh.cut = kBins;
        if (tid < kBins) {
            uint32_t n = 0;
            for (int r = 0; r < ctas; ++r) n += remote_u32(&sh.hist[tid], (uint32_t)r);
            cnt = (float)n;     // exact up to 2^24 tokens, more than the slices can hold
            least = cnt * ex2(-(float)(tid + 1) / kBinsPerOctave);
            most = cnt * ex2(-(float)tid / kBinsPerOctave);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const float c1 = __shfl_up_sync(~0u, cnt, o), l1 = __shfl_up_sync(~0u, least, o), m1 = __shfl_up_sync(~0u, most, o);
                if (lane >= o) { cnt += c1; least += l1; most += m1; }
            }
            if (lane == 31) { sh.scan[0][warp] = cnt; sh.scan[1][warp] = least; sh.scan[2][warp] = most; }
        }
        __syncthreads();
        if (tid < kBins) {
            for (int i = 0; i < warp; ++i) { cnt += sh.scan[0][i]; least += sh.scan[1][i]; most += sh.scan[2][i]; }
            sh.count[tid] = (uint32_t)cnt;
            sh.most[tid] = most;
            // every kept token is in this bin or one before it
            if ((by_count && cnt >= (float)k) || (by_mass && least >= limit * 1.0001f)) atomicMin(&sh.cut, tid);
        }
        __syncthreads();
        const int cut = sh.cut;
        // logits of the bins up to the cut, from a little below to be safe against rounding
        float from = -INFINITY;
        if (cut < kBins) {
            from = top - ((float)(cut + 1) / kBinsPerOctave) / c;
            from -= 1e-5f * (fabsf(top) + fabsf(from)) + 1e-5f / c;
        }
        // few enough to be listed (the margin may add some: then they do not all fit and the
        // race below goes on)
        const bool few = cut < kBins && sh.count[cut] <= (uint32_t)kList;
        if (few) cluster_barrier();     // the histograms have been read: CTA 0's list takes their place
        if (few) {
            for (uint32_t v = tid, i0 = i_own; v < all; v += kSlice, i0 += kSlice * VEC) {
                const uint4 q = slice[v];
                if (!(vec_max<T>(q) >= from)) continue;
                float x[VEC];
                unpack<T>(q, x);
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (x[j] >= from && weight(x[j]) >= least_w) list(x[j], i0 + j);
            }
        } else {
            hold_race([&](const uint4& q, uint32_t, float (&wx)[VEC]) {
                if (!(vec_max<T>(q) >= from)) return;
                float x[VEC];
                unpack<T>(q, x);
#pragma unroll
                for (int j = 0; j < VEC; ++j) wx[j] = x[j] >= from ? weight(x[j]) : 0.0f;
            });
        }
        if (few) {
            send();
            const uint4 w = cluster_join<JoinList>(make_uint4(tid ? 0 : sh.listed, tid ? 0 : sh.listed, 0, 0), sh, turn, ctas, rank);
            if (w.x && w.y <= (uint32_t)room) {
                if (rank) return;
                won = choose(sh, reinterpret_cast<uint64_t*>(slice), (int)w.x, turn ^ 1, ctas, k, by_mass, limit, top, c, noise, shift);
                if (tid == 0) finish(won.y, __uint_as_float(won.z), z);
                return;
            }
        } else {
            won = cluster_join<JoinRace>(race, sh, turn, ctas, rank);
            have = true;
            // surely kept: even all tokens of its bin and those before are few and light enough
            if (won.x) {
                const float t = (__uint_as_float(won.z) - top) * c * -kBinsPerOctave;
                if (t < (float)kBins) {
                    const int b = (int)t;
                    done = (!by_count || sh.count[b] <= (uint32_t)k) && (!by_mass || sh.most[b] < limit * 0.9999f);
                }
            }
        }
    }
    // Rounds: is the winner kept? If not, race again before it. From the third round on the
    // midpoint between what is known to be in and to be out is tested too.
    uint64_t lo = position(top, 0, shift), hi = position(-INFINITY, 0, shift);
    for (int round = 0; !done; ++round) {
        if (!have) {
            race = JoinRace::none();
            const float from = value_of(hi, shift);
            hold_race([&](const uint4& q, uint32_t i0, float (&wx)[VEC]) {
                if (vec_max<T>(q) < from) return;
                float x[VEC];
                unpack<T>(q, x);
#pragma unroll
                for (int j = 0; j < VEC; ++j) wx[j] = position(x[j] + 0.0f, i0 + j, shift) < hi ? weight(x[j]) : 0.0f;
            });
            won = cluster_join<JoinRace>(race, sh, turn, ctas, rank);
        }
        have = false;
        if (!won.x) break;
        const float x_won = __uint_as_float(won.z);
        const uint64_t at_won = position(x_won + 0.0f, won.y, shift);
        if (at_won <= lo) break;
        const uint64_t mid = round < 2 ? lo : lo + (hi - lo) / 2;
        const float from = fminf(x_won, value_of(mid, shift));
        uint32_t n0 = 0, n1 = 0;
        float m0 = 0.0f, m1 = 0.0f;
        for (uint32_t v = tid, i0 = i_own; v < all; v += kSlice, i0 += kSlice * VEC) {
            const uint4 q = slice[v];
            if (vec_max<T>(q) < from) continue;
            float x[VEC];
            unpack<T>(q, x);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const uint64_t at = position(x[j] + 0.0f, i0 + j, shift);
                if (at >= at_won && at >= mid) continue;
                const float wx = weight(x[j]);
                if (at < at_won) { ++n0; m0 += wx; }
                if (at < mid) { ++n1; m1 += wx; }
            }
        }
        const uint4 w = cluster_join<JoinCounts>(make_uint4(n0, n1, __float_as_uint(m0), __float_as_uint(m1)), sh, turn, ctas, rank);
        if ((int)w.x < k && (!by_mass || __uint_as_float(w.z) < limit)) break;
        hi = at_won;
        if (round >= 2) {
            if ((int)w.y < k && (!by_mass || __uint_as_float(w.w) < limit)) lo = max(lo, mid);
            else hi = min(hi, mid);
        }
    }
    if (!won.x) {                       // temperature 0, or no usable variate: the first token
        if (mode != kFirst) {
            for (uint32_t v = tid, i0 = i_own; v < all && first == 0xFFFFFFFFu; v += kSlice, i0 += kSlice * VEC) {
                float x[VEC];
                unpack<T>(slice[v], x);
#pragma unroll
                for (int j = VEC - 1; j >= 0; --j)
                    if (x[j] == top) first = i0 + j;
            }
        }
        won.y = cluster_join<JoinLeast>(make_uint4(first, 0, 0, 0), sh, turn, ctas, rank).x;
        won.z = __float_as_uint(top);
    }
    if (rank == 0 && tid == 0) finish(won.y, __uint_as_float(won.z), z);
}

constexpr int64_t kMost = 200 * 1024, kTwoFit = 100 * 1024;     // bytes of a slice, and where two CTAs fit an SM

// CTAs per row, 0 where no cluster holds it: a power of two (others pack badly into the clusters'
// groups of SMs: 48 rows of 32000, 6 CTAs 43.2, 4 32.3), as many as leave every row's cluster resident
// at once, but no slices under 3 KB, where exchanges cost more than the slices save, and enough for
// slices of 100 KB, two of which fit an SM. A B200 holds 33 clusters of 8, 71 of 4 and 148 of 2; the last
// few share SMs with all others, so the limits are 30 and 68. Measured (us, sums over three kinds of filters,
// bf16 unless said), 8 CTAs against 4: 30 rows of 16000 26.2, 26.0; of 32000 28.9, 30.2; of 50257 36.2, 42.4;
// 33 rows of 16000 32.3, 26.1; of 32000 34.2, 30.2; of 40000 f32 37.5, 33.6; of 50257 40.8, 42.2; of 80000 45.9,
// 44.0; of 100001 50.6, 54.9; 34 of 50257 45.6, 42.1; 36 of 100001 57.3, 54.1. 4 against 2: 68 rows of 8000 28.7, 30.2;
// of 32000 33.8, 38.6; 71 of 8000 32.1, 30.0; of 32000 35.7, 38.1; 72 of 32000 43.8, 38.0; 148 of 36000 f32 81.7,
// 58.8. From 80000 tokens on half the rows may wait instead: 72 of 80000 68.8, 76.2; 110 of 80000 86.4, 94.9; 100
// of 100001 100.0, 111.9; 148 of 100001 134.1, 128.2; but 72 of 64000 53.0, 51.6; 110 of 64000 74.1, 63.9. 2 against 1:
// 256 of 32000 76.6, 73.9. Longer slices than need be: 256 of 50257 f32: 2 128.9, 4 148.8; 256 of 100001 f32:
// 4 229.4, 8 284.5; 256 of 131072, top-k and top-p: 4 48.6, 2 54.7, 8 66.9; 32 of 1000: 1 23.2, 8 30.3; 8 of 8000: 4 20.8, 8 21.5.
int ctas_per_row(int64_t rows, int64_t vocab, int64_t size) {
    const int64_t bytes = vocab * size;
    if (bytes / kMostCtas > kMost) return 0;
    const int fit = rows <= 30 ? 8 : rows <= (vocab >= 80000 ? 110 : 68) ? 4 : rows <= 148 ? 2 : 1;
    int need = 1, most = 1;
    while (need < kMostCtas && bytes > need * kTwoFit) need *= 2;
    while (most < kMostCtas && bytes >= 2 * most * 3072) most *= 2;
    return std::max(need, std::min(fit, most));
}

template <typename T>
bool launch_cluster(const SampleArgs& a, int shift, cudaStream_t s) {
    const int ctas = ctas_per_row(a.rows, a.vocab, sizeof(T));
    if (!ctas) return false;
    const size_t smem = std::max<size_t>((size_t)(((a.vocab + kVec<T> - 1) / kVec<T> + ctas - 1) / ctas) * 16, 2 * kList * 8);
    static bool ready[64] = {};
    int device = 0;
    PB_CUDA(cudaGetDevice(&device));
    if (device >= 64 || !ready[device]) {
        PB_CUDA(cudaFuncSetAttribute(sample_cluster_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMost + 1024));
        if (device < 64) ready[device] = true;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(a.rows * ctas));
    cfg.blockDim = dim3(kSlice);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0] = dependent_launch();
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)ctas;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    PB_CUDA(cudaLaunchKernelEx(&cfg, sample_cluster_kernel<T>, a, shift, ctas));
    return true;
}

}  // namespace

int sample_plan(int64_t rows, int64_t vocab, int dtype) { return ctas_per_row(rows, vocab, dtype == ENGINE_F32 ? 4 : 2); }

void launch_sample(const SampleArgs& a, cudaStream_t s) {
    if (a.rows == 0) return;
    int shift = 1;                             // bits of an index
    while ((1ll << shift) < a.vocab) ++shift;
    const bool done = a.dtype == ENGINE_F32 ? launch_cluster<float>(a, shift, s)
                      : a.dtype == ENGINE_F16 ? launch_cluster<__half>(a, shift, s)
                      : a.dtype == ENGINE_BF16 && launch_cluster<__nv_bfloat16>(a, shift, s);
    if (done) return;
    switch (a.dtype) {
        case ENGINE_F32: sample_rows_kernel<float><<<(unsigned)a.rows, kThreads, 0, s>>>(a, shift); break;
        case ENGINE_F16: sample_rows_kernel<__half><<<(unsigned)a.rows, kThreads, 0, s>>>(a, shift); break;
        case ENGINE_BF16: sample_rows_kernel<__nv_bfloat16><<<(unsigned)a.rows, kThreads, 0, s>>>(a, shift); break;
        default: fail(ENGINE_ERR_INVALID_ARG, "sample: dtype must be F32, F16 or BF16");
    }
    PB_CUDA(cudaGetLastError());
}

}  // namespace pb
