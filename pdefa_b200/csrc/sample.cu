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

}  // namespace

void launch_sample(const SampleArgs& a, cudaStream_t s) {
    if (a.rows == 0) return;
    int shift = 1;                             // bits of an index
    while ((1ll << shift) < a.vocab) ++shift;
    switch (a.dtype) {
        case ENGINE_F32: sample_rows_kernel<float><<<(unsigned)a.rows, kThreads, 0, s>>>(a, shift); break;
        case ENGINE_F16: sample_rows_kernel<__half><<<(unsigned)a.rows, kThreads, 0, s>>>(a, shift); break;
        case ENGINE_BF16: sample_rows_kernel<__nv_bfloat16><<<(unsigned)a.rows, kThreads, 0, s>>>(a, shift); break;
        default: fail(ENGINE_ERR_INVALID_ARG, "sample: dtype must be F32, F16 or BF16");
    }
    PB_CUDA(cudaGetLastError());
}

}  // namespace pb
