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
#include <cuda_fp16.h>

#include "common.h"
#include "device_common.cuh"

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
    const float c = kLog2e / temp;
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
            if (e >= 0.0f) r.take(w / e, i, x);
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
constexpr int kSlice = 256;             // threads of a CTA
constexpr int kWarps = kSlice / 32;
constexpr int kBins = 256;
constexpr float kBinsPerOctave = 16.0f; // the bins cover w from 1 down to 2^-16

template <typename T> constexpr int kVec = 16 / (int)sizeof(T);
template <typename T> constexpr bool kIsHalf = false;
template <> constexpr bool kIsHalf<__half> = true;

// 16 bytes of logits -> NaN replaced by -inf
template <typename T> __device__ __forceinline__ uint4 clean_vec(uint4 v);
template <> __device__ __forceinline__ uint4 clean_vec<float>(uint4 v) {
    uint32_t* w = &v.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(fmaxf(__uint_as_float(w[i]), -INFINITY));
    return v;
}
template <> __device__ __forceinline__ uint4 clean_vec<__half>(uint4 v) {
    const __half2 low = __half2half2(__ushort_as_half(0xFC00));
    __half2* w = reinterpret_cast<__half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __hmax2(w[i], low);
    return v;
}
template <> __device__ __forceinline__ uint4 clean_vec<__nv_bfloat16>(uint4 v) {
    const __nv_bfloat162 low = __bfloat162bfloat162(__ushort_as_bfloat16(0xFF80));
    __nv_bfloat162* w = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __hmax2(w[i], low);
    return v;
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
    float x[kVec<T>];
    unpack<T>(v, x);
    float m = x[0];
#pragma unroll
    for (int i = 1; i < kVec<T>; ++i) m = fmaxf(m, x[i]);
    return m;
}

// Vectors of a row that may start anywhere: one aligned load, or two and a shift by the
// row's offset within 16 bytes. Nothing outside the row is read.
template <typename T>
struct RowLoader {
    const T* row;
    uint32_t n;                 // elements
    const uint4* base;          // the aligned vector that holds the row's first element
    int words, bits;            // the row's offset in it
    __device__ __forceinline__ RowLoader(const T* r, uint32_t len) : row(r), n(len) {
        const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(r) & 15);
        base = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(r) - off);
        words = (int)(off >> 2);
        bits = (int)(off & 3) * 8;
    }
    __device__ __forceinline__ uint4 operator()(uint32_t v) const {
        const uint32_t i = v * kVec<T>;
        const bool whole = i + kVec<T> <= n;
        if ((words | bits) == 0 && whole) return __ldg(base + v);
        // the two vectors lie inside the row unless v is its first or its last
        if (v > 0 && i + 2 * kVec<T> <= n) {
            const uint4 lo = __ldg(base + v), hi = __ldg(base + v + 1);
            uint32_t s[5];
            switch (words) {
                case 0: s[0] = lo.x; s[1] = lo.y; s[2] = lo.z; s[3] = lo.w; s[4] = hi.x; break;
                case 1: s[0] = lo.y; s[1] = lo.z; s[2] = lo.w; s[3] = hi.x; s[4] = hi.y; break;
                case 2: s[0] = lo.z; s[1] = lo.w; s[2] = hi.x; s[3] = hi.y; s[4] = hi.z; break;
                default: s[0] = lo.w; s[1] = hi.x; s[2] = hi.y; s[3] = hi.z; s[4] = hi.w; break;
            }
            return make_uint4(__funnelshift_r(s[0], s[1], bits), __funnelshift_r(s[1], s[2], bits),
                              __funnelshift_r(s[2], s[3], bits), __funnelshift_r(s[3], s[4], bits));
        }
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (sizeof(T) == 4) {
                w[j] = i + j < n ? __float_as_uint((float)row[i + j]) : 0xFF800000u;
            } else {
                const uint16_t* h = reinterpret_cast<const uint16_t*>(row);
                const uint32_t low = kIsHalf<T> ? 0xFC00u : 0xFF80u;     // -inf
                w[j] = (i + 2 * j < n ? h[i + 2 * j] : low) | ((i + 2 * j + 1 < n ? h[i + 2 * j + 1] : low) << 16);
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// What the CTAs of a cluster tell each other; one field per kind of join.
struct Word {
    float sum0, sum1;           // added
    int n0, n1;                 // added
    float key, x;               // a race
    uint32_t idx;
    uint32_t least;             // minimum
};

__device__ __forceinline__ Word word_none() { return Word{0.0f, 0.0f, 0, 0, -1.0f, 0.0f, 0xFFFFFFFFu, 0xFFFFFFFFu}; }

// Joins `w` over lanes `width` apart and less; every lane gets the result.
__device__ __forceinline__ Word warp_join(Word w, int width) {
    for (int o = width >> 1; o; o >>= 1) {
        w.sum0 += __shfl_xor_sync(~0u, w.sum0, o);
        w.sum1 += __shfl_xor_sync(~0u, w.sum1, o);
        w.n0 += __shfl_xor_sync(~0u, w.n0, o);
        w.n1 += __shfl_xor_sync(~0u, w.n1, o);
        const float k = __shfl_xor_sync(~0u, w.key, o), x = __shfl_xor_sync(~0u, w.x, o);
        const uint32_t i = __shfl_xor_sync(~0u, w.idx, o);
        if (k > w.key || (k == w.key && i < w.idx)) { w.key = k; w.idx = i; w.x = x; }
        w.least = min(w.least, __shfl_xor_sync(~0u, w.least, o));
    }
    return w;
}

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t remote_u32(const void* p, uint32_t rank) {
    uint32_t v;
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.u32 %0, [a];\n\t}"
                 : "=r"(v) : "r"(smem_u32(p)), "r"(rank) : "memory");
    return v;
}

struct Shared {
    Word part[kWarps];
    Word told[2];               // this CTA's word of the last two joins
    uint32_t hist[kBins];
    uint32_t count[kBins];      // tokens of bins <= b, over the row
    float most[kBins];          // upper bound of their mass
    float scan[3][kWarps];
    int cut;
};

// One join over the cluster. Two slots suffice: a CTA writes a slot again only after the
// next join's barrier, which every CTA reaches after it has read this one.
__device__ __forceinline__ Word cluster_join(Word w, Shared& sh, int& turn, int ctas) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    w = warp_join(w, 32);
    if (lane == 0) sh.part[warp] = w;
    __syncthreads();
    if (warp == 0) {
        w = lane < kWarps ? sh.part[lane] : word_none();
        w = warp_join(w, 32);
        if (lane == 0) sh.told[turn] = w;
        __syncwarp();
    }
    cluster_barrier();
    Word r = word_none();
    if (lane < ctas) {
        const uint32_t* src = reinterpret_cast<const uint32_t*>(&sh.told[turn]);
        uint32_t* dst = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
        for (int i = 0; i < (int)(sizeof(Word) / 4); ++i) dst[i] = remote_u32(src + i, (uint32_t)lane);
    }
    turn ^= 1;
    return warp_join(r, 32);
}

template <typename T>
__global__ void __launch_bounds__(kSlice, 4)
sample_cluster_kernel(SampleArgs a, int shift, int ctas) {
    constexpr int VEC = kVec<T>;
    extern __shared__ uint4 slice[];
    __shared__ Shared sh;
    const int tid = threadIdx.x;
    uint32_t rank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const int64_t row = blockIdx.x / ctas;
    const T* lg = static_cast<const T*>(a.logits) + row * a.logits_stride;
    const float* noise = a.noise + row * a.noise_stride;
    const uint32_t V = (uint32_t)a.vocab;
    float temp = a.temperature ? a.temperature[row] : 1.0f;
    int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    const float floor_w = a.min_p ? a.min_p[row] : 0.0f;
    if (!(temp > 0.0f)) { temp = 1.0f; k = 1; }
    const bool by_count = k > 0, by_mass = !(p >= 1.0f);
    if (!by_count) k = 0x7FFFFFFF;

    // Vector v holds the elements from v * VEC on (-inf past the end), wherever the row
    // starts in memory, so that sums do not depend on that.
    const uint32_t nv = (V + VEC - 1) / VEC;
    const uint32_t v0 = (uint32_t)((uint64_t)nv * rank / ctas), all = (uint32_t)((uint64_t)nv * (rank + 1) / ctas) - v0;
    auto index_of = [&](uint32_t v) { return (v0 + v) * VEC; };

    const RowLoader<T> load(lg, V);
    float mx = -INFINITY;
    uint32_t at_max = 0;
#pragma unroll 4
    for (uint32_t v = tid; v < all; v += kSlice) {
        const uint4 q = clean_vec<T>(load(v0 + v));
        slice[v] = q;
        const float m = vec_max<T>(q);
        if (m > mx) { mx = m; at_max = v; }
    }
    for (int b = tid; b < kBins; b += kSlice) sh.hist[b] = 0;
    int turn = 0;
    float tmax = mx;
    {
        // maximum over the cluster
        const int warp = tid >> 5, lane = tid & 31;
#pragma unroll
        for (int o = 16; o; o >>= 1) tmax = fmaxf(tmax, __shfl_xor_sync(~0u, tmax, o));
        if (lane == 0) sh.part[warp].x = tmax;
        __syncthreads();
        if (tid == 0) {
            for (int i = 1; i < kWarps; ++i) tmax = fmaxf(tmax, sh.part[i].x);
            sh.told[turn].x = tmax;
        }
        __syncwarp();
        cluster_barrier();
        tmax = lane < ctas ? __uint_as_float(remote_u32(&sh.told[turn].x, (uint32_t)lane)) : -INFINITY;
#pragma unroll
        for (int o = 16; o; o >>= 1) tmax = fmaxf(tmax, __shfl_xor_sync(~0u, tmax, o));
        turn ^= 1;
    }
    const float top = tmax + 0.0f;      // the row's largest logit
    if (top == -INFINITY) {
        if (rank == 0 && tid == 0) {
            a.tokens[row] = -1;
            if (a.probs) a.probs[row] = 0.0f;
        }
        cluster_barrier();              // no CTA leaves while another may read its memory
        return;
    }

    // w = 2^y with y = (x - top) * log2(e) / T. The clamps keep two products from becoming
    // NaN: inf - inf (the top itself, y = 0) and -inf * 0 (an infinite temperature).
    const float c = fmaxf(kLog2e / temp, 1.17549435e-38f);
    auto exponent = [&](float x) { return fminf((x - top) * c, 0.0f); };

    // Which tokens can be kept? With a min_p that cuts at 2^-6 or above, those it leaves, and
    // they race in this pass; with no filter at all, every token. Otherwise count the tokens in
    // bins of w, to find how far down the order the filters can reach.
    const bool filtered = by_count || by_mass || floor_w > 0.0f;
    const bool greedy = k == 1;
    const bool race_now = !greedy && (!filtered || floor_w >= 0.015625f);
    const bool count_now = !greedy && !race_now;
    Word w = word_none();
    float z = 0.0f;
    Race race;
    auto enter = [&](float x, uint32_t i, float wx) {
        const float e = __ldg(noise + i);
        if (e >= 0.0f && wx > 0.0f) race.take(__fdividef(wx, e), i, x);
    };
    for (uint32_t v = tid; v < all; v += kSlice) {
        float x[VEC], y[VEC], wx[VEC];
        unpack<T>(slice[v], x);
        float zz = 0.0f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            y[j] = exponent(x[j]);
            wx[j] = ex2(y[j]);
            zz += wx[j];
        }
        z += zz;
        if (race_now) {
            float m = wx[0];
#pragma unroll
            for (int j = 1; j < VEC; ++j) m = fmaxf(m, wx[j]);
            if (m >= floor_w) {
                const uint32_t i0 = index_of(v);
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (wx[j] >= floor_w && x[j] > -INFINITY) enter(x[j], i0 + j, wx[j]);
            }
        } else if (count_now) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float t = y[j] * -kBinsPerOctave;
                if (t < (float)kBins) atomicAdd(&sh.hist[(int)t], 1u);
            }
        }
    }
    w.sum0 = z;
    w.key = race.key; w.idx = race.idx; w.x = race.x;
    // lowest index of the largest logit
    if (mx == top) {
        float x[VEC];
        unpack<T>(slice[at_max], x);
        for (int j = VEC - 1; j >= 0; --j)
            if (x[j] == top) w.least = index_of(at_max) + j;
    }
    w = cluster_join(w, sh, turn, ctas);
    z = w.sum0;
    const uint32_t first = w.least;
    const float limit = p * z;
    Race won;
    won.key = w.key; won.idx = w.idx; won.x = w.x;

    bool done = greedy || (race_now && !by_count && !by_mass);
    if (greedy) won.idx = 0xFFFFFFFFu;      // the first token
    uint64_t lo = position(top, first, shift), hi = position(-INFINITY, 0, shift);
    bool have = race_now;
    if (count_now) {
        // bin b holds tokens with w in (2^(-(b + 1) / 16), 2^(-b / 16)]
        const int warp = tid >> 5, lane = tid & 31;
        uint32_t n = 0;
        for (int r = 0; r < ctas; ++r) n += remote_u32(&sh.hist[tid], (uint32_t)r);
        float least = (float)n * ex2(-(float)(tid + 1) / kBinsPerOctave);
        float most = (float)n * ex2(-(float)tid / kBinsPerOctave);
        float cnt = (float)n;               // exact: at most 2^24 matter, and more only say "many"
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const float c1 = __shfl_up_sync(~0u, cnt, o), l1 = __shfl_up_sync(~0u, least, o), m1 = __shfl_up_sync(~0u, most, o);
            if (lane >= o) { cnt += c1; least += l1; most += m1; }
        }
        if (lane == 31) { sh.scan[0][warp] = cnt; sh.scan[1][warp] = least; sh.scan[2][warp] = most; }
        if (tid == 0) sh.cut = kBins;
        __syncthreads();
        for (int i = 0; i < warp; ++i) { cnt += sh.scan[0][i]; least += sh.scan[1][i]; most += sh.scan[2][i]; }
        sh.count[tid] = (uint32_t)fminf(cnt, 2147483520.0f);
        sh.most[tid] = most;
        // every kept token is in this bin or one before it
        if ((by_count && cnt >= (float)k) || (by_mass && least >= limit * 1.0001f)) atomicMin(&sh.cut, tid);
        __syncthreads();
        const int cut = sh.cut;
        // logits of the bins up to the cut, a little below to be safe against rounding
        float from = -INFINITY;
        if (cut < kBins) {
            from = top - ((float)(cut + 1) / kBinsPerOctave) / c;
            if (top < INFINITY) from -= 1e-5f * (fabsf(top) + fabsf(from)) + 1e-5f / c;
        }
        race = Race();
        for (uint32_t v = tid; v < all; v += kSlice) {
            const uint4 q = slice[v];
            if (!(vec_max<T>(q) >= from)) continue;
            float x[VEC];
            unpack<T>(q, x);
            const uint32_t i0 = index_of(v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if (!(x[j] >= from) || x[j] == -INFINITY) continue;
                const float wx = ex2(exponent(x[j]));
                if (wx >= floor_w) enter(x[j], i0 + j, wx);
            }
        }
        w = word_none();
        w.key = race.key; w.idx = race.idx; w.x = race.x;
        w = cluster_join(w, sh, turn, ctas);
        won.key = w.key; won.idx = w.idx; won.x = w.x;
        have = true;
        // surely kept: even all tokens of its bin and those before are few and light enough
        if (won.idx != 0xFFFFFFFFu) {
            const float t = exponent(won.x) * -kBinsPerOctave;
            if (t < (float)kBins) {
                const int b = (int)t;
                if ((!by_count || sh.count[b] <= (uint32_t)k) && (!by_mass || sh.most[b] < limit * 0.9999f)) done = true;
            }
        }
    }
    // Rounds: is the winner kept? If not, race again before it. From the third round on the
    // midpoint between what is known to be in and to be out is tested too.
    for (int round = 0; !done; ++round) {
        if (!have) {
            race = Race();
            const float from = value_of(hi, shift);
            for (uint32_t v = tid; v < all; v += kSlice) {
                const uint4 q = slice[v];
                if (vec_max<T>(q) < from) continue;
                float x[VEC];
                unpack<T>(q, x);
                const uint32_t i0 = index_of(v);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    if (x[j] == -INFINITY || position(x[j] + 0.0f, i0 + j, shift) >= hi) continue;
                    const float wx = ex2(exponent(x[j]));
                    if (wx >= floor_w) enter(x[j], i0 + j, wx);
                }
            }
            w = word_none();
            w.key = race.key; w.idx = race.idx; w.x = race.x;
            w = cluster_join(w, sh, turn, ctas);
            won.key = w.key; won.idx = w.idx; won.x = w.x;
        }
        have = false;
        if (won.idx == 0xFFFFFFFFu) break;
        const uint64_t at_won = position(won.x + 0.0f, won.idx, shift);
        if (at_won <= lo) break;
        const uint64_t mid = round < 2 ? lo : lo + (hi - lo) / 2;
        const float from = fminf(won.x, value_of(mid, shift));
        w = word_none();
        for (uint32_t v = tid; v < all; v += kSlice) {
            const uint4 q = slice[v];
            if (vec_max<T>(q) < from) continue;
            float x[VEC];
            unpack<T>(q, x);
            const uint32_t i0 = index_of(v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if (x[j] == -INFINITY) continue;
                const uint64_t at = position(x[j] + 0.0f, i0 + j, shift);
                if (at >= at_won && at >= mid) continue;
                const float wx = ex2(exponent(x[j]));
                if (at < at_won) { ++w.n0; w.sum0 += wx; }
                if (at < mid) { ++w.n1; w.sum1 += wx; }
            }
        }
        w = cluster_join(w, sh, turn, ctas);
        if (w.n0 < k && (!by_mass || w.sum0 < limit)) break;
        hi = at_won;
        if (round >= 2) {
            if (w.n1 < k && (!by_mass || w.sum1 < limit)) lo = max(lo, mid);
            else hi = min(hi, mid);
        }
    }
    if (rank == 0 && tid == 0) {
        const bool none = won.idx == 0xFFFFFFFFu;       // no usable variate: the first token
        a.tokens[row] = (int32_t)(none ? first : won.idx);
        if (a.probs) a.probs[row] = (none || won.x == top ? 1.0f : expf((won.x - top) / temp)) / z;
    }
    cluster_barrier();
}

template <typename T>
bool launch_cluster(const SampleArgs& a, int shift, cudaStream_t s) {
    const int64_t bytes = a.vocab * (int64_t)sizeof(T);
    constexpr int64_t kMost = 200 * 1024;
    int ctas = 8;
    if (bytes / ctas > kMost) return false;
    const size_t smem = (size_t)(((a.vocab + kVec<T> - 1) / kVec<T> + ctas - 1) / ctas) * 16;
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
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)ctas;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    PB_CUDA(cudaLaunchKernelEx(&cfg, sample_cluster_kernel<T>, a, shift, ctas));
    return true;
}

}  // namespace

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
