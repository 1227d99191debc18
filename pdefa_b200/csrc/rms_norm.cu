// Root-mean-square norm of rows, with the addition of a residual before it and, if
// wanted, the 8-bit form of the result with one scale for each 128 columns.
//
//   h = x + residual (32 bits), h_out = round(h)
//   y = h * w / sqrt(mean(h^2) + eps)
//   8-bit: scale = max(max|y| over 128 columns, 1e-10) / 448, q = e4m3(y / scale)
//
// Bound by memory: the values are read once and written once, 16384 x 8192 bf16 with a
// residual and an 8-bit output in 140 us from a graph (6.8 TB/s, 105% of a plain copy's rate on
// B200) and 157 in a loop of calls (6.0 TB/s).
//
// The statistic and the scales come from the unrounded 32-bit sum. A NaN in a row makes its
// whole output NaN. An infinity makes the root infinite: it becomes NaN, the row's others 0.
#include <algorithm>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <type_traits>

#include "common.h"
#include "device_common.cuh"
#include "row_vec.cuh"

namespace pb {

namespace {

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }

// max that keeps NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

constexpr float kE4m3Max = 448.0f;
constexpr float kTiny = 1e-10f;
constexpr int kGroup = 128;

// A group's scale m / 448 and what quotients by it take, both as the 32-bit division rounds them:
// a product by an inverse that is good to a few ulps, then one step on the residue, which a fused
// product leaves exact (Markstein's method). Values between two 8-bit ones are quotients that 32
// bits hold, so they must not be off by an ulp. (Bit by bit the division's bytes and scales. On
// pairs the step costs next to nothing: 16384 x 8192 bf16, residual: 139.7 us, 139.1 without it,
// 176 with divisions; 5000 x 4096 f32 27.3, 26.5 and 31.4.) The residue of an infinite scale would be
// NaN, so a finite one stands for it there. A quarter of both in the inverse, since the fast division
// takes divisors to 2^126.
struct Scale {
    float s, inv, minus;
};
__device__ __forceinline__ Scale scale_of(float m) {
    constexpr float c = 1.0f / kE4m3Max, most = 3.0e38f;
    Scale d;
    const float s = fminf(m * c, most);
    d.s = fmaf(fmaf(-kE4m3Max, s, m), c, s);
    d.inv = __fdividef(0.25f * kE4m3Max, 0.25f * m);
    d.minus = fmaxf(-d.s, -most);
    return d;
}
__device__ __forceinline__ float2 quotients(float2 v, float2 inv, float2 minus) {
    const float2 q = __fmul2_rn(v, inv);
    return __ffma2_rn(__ffma2_rn(q, minus, v), inv, q);
}
__device__ __forceinline__ float2 times(float2 h, float r, float2 w) { return __fmul2_rn(__fmul2_rn(h, make_float2(r, r)), w); }
__device__ __forceinline__ uint32_t four_fp8(float2 a, float2 b) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3);
    return lo | (uint32_t)__nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3) << 16;
}

// One CTA per row; every pass reads the row again (from L2 after the first). For rows of more
// than 4096 pieces, which the registers do not hold (1000 x 32776 bf16 with a residual and an
// 8-bit output: 161 us; 1000 x 32760 in registers 51).
template <typename T, typename W>
__global__ void __launch_bounds__(256)
rms_norm_rows_kernel(RmsNormArgs a) {
    __shared__ float part[8];
    grid_trigger();
    grid_wait();
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
    const W* w = static_cast<const W*>(a.weight);
    T* h_out = a.h_out ? static_cast<T*>(a.h_out) + row * a.h_stride : nullptr;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto value = [&](int64_t c) {
        float v = to_f32(x[c]);
        return res ? v + to_f32(res[c]) : v;
    };
    float sum = 0.0f;
    for (int64_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
        const float v = value(c);
        sum = fmaf(v, v, sum);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (lane == 0) part[warp] = sum;
    __syncthreads();
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) total += part[i];
    const float r = rsqrtf(total / (float)a.cols + a.eps);
    // One warp per 128 columns, so that a group's largest value stays inside the
    // warp; h_out is written here, by the thread that read x and the residual, which
    // makes h_out == residual (or x) safe.
    for (int64_t g = warp; g * kGroup < a.cols; g += 8) {
        float v[4], m = kTiny;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t c = g * kGroup + i * 32 + lane;
            v[i] = 0.0f;
            if (c < a.cols) {
                const float h = value(c);
                if (h_out) h_out[c] = from_f32<T>(h);
                v[i] = h * r * to_f32(w[c]);
                m = max_nan(m, fabsf(v[i]));
            }
        }
        if (a.quantize) {
#pragma unroll
            for (int o = 16; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(~0u, m, o));
            const float scale = m / kE4m3Max;
            if (lane == 0) a.scales[row * a.scales_stride + g] = scale;
            uint8_t* y = static_cast<uint8_t*>(a.y) + row * a.y_stride;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t c = g * kGroup + i * 32 + lane;
                if (c < a.cols) y[c] = __nv_cvt_float_to_fp8(v[i] / scale, __NV_SATFINITE, __NV_E4M3);
            }
        } else {
            T* y = static_cast<T*>(a.y) + row * a.y_stride;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t c = g * kGroup + i * 32 + lane;
                if (c < a.cols) y[c] = from_f32<T>(v[i]);
            }
        }
    }
}

// 16-byte pieces of a row: 8 values of 16 bits or 4 of 32.
template <typename T> constexpr int kPiece = 16 / (int)sizeof(T);

template <typename T>
__device__ __forceinline__ void unpack(const uint4& q, float (&v)[kPiece<T>]) {
    const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
    for (int i = 0; i < kPiece<T>; ++i) v[i] = to_f32(e[i]);
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float (&v)[kPiece<T>]) {
    uint4 q;
    T* e = reinterpret_cast<T*>(&q);
#pragma unroll
    for (int i = 0; i < kPiece<T>; ++i) e[i] = from_f32<T>(v[i]);
    return q;
}

// STREAM: the data passes through the L2 cache without staying there.
template <bool STREAM>
__device__ __forceinline__ uint4 load_piece(const void* p) {
    const uint4* q = static_cast<const uint4*>(p);
    return STREAM ? __ldcs(q) : *q;
}
template <bool STREAM, typename V>
__device__ __forceinline__ void store_piece(void* p, V v) {
    if (STREAM) __stcs(static_cast<V*>(p), v);
    else *static_cast<V*>(p) = v;
}

// Stores the pieces of a row that starts anywhere: a thread writes the aligned piece that
// begins inside its own and ends in the next thread's (`next`), element by element only at
// the row's two ends. B: bytes of a piece, V the vector type of that size, E the element's.
__device__ __forceinline__ uint4 join_pieces(const uint4& own, const uint4& next, int bytes) {
    return shift_pair(own, next, bytes >> 2, (bytes & 3) * 8);
}
__device__ __forceinline__ uint2 join_pieces(const uint2& own, const uint2& next, int bytes) {
    const uint4 r = shift_pair(make_uint4(own.x, own.y, next.x, next.y), make_uint4(0, 0, 0, 0), bytes >> 2, (bytes & 3) * 8);
    return make_uint2(r.x, r.y);
}
__device__ __forceinline__ uint32_t join_pieces(uint32_t own, uint32_t next, int bytes) {
    return __funnelshift_r(own, next, bytes * 8);
}
template <typename E, typename V>
__device__ __forceinline__ void store_shifted(E* row, int cols, int c, const V& own, const V& next) {
    constexpr int B = sizeof(V), P = B / sizeof(E);
    const int off = (int)(reinterpret_cast<uintptr_t>(row) % B);
    const int lead = off ? (B - off) / (int)sizeof(E) : 0;      // elements before the first aligned piece
    if (c == 0 && lead) {
        const E* e = reinterpret_cast<const E*>(&own);
#pragma unroll
        for (int j = 0; j < P; ++j)
            if (j < lead && j < cols) row[j] = e[j];
    }
    const int first = c + lead;
    if (first >= cols) return;
    const V out = lead ? join_pieces(own, next, lead * (int)sizeof(E)) : own;
    if (first + P <= cols) {
        *reinterpret_cast<V*>(row + first) = out;
    } else {
        const E* e = reinterpret_cast<const E*>(&out);
#pragma unroll
        for (int j = 0; j < P; ++j)
            if (first + j < cols) row[first + j] = e[j];
    }
}
__device__ __forceinline__ uint4 shuffle_down(const uint4& v) {
    return make_uint4(__shfl_down_sync(~0u, v.x, 1), __shfl_down_sync(~0u, v.y, 1), __shfl_down_sync(~0u, v.z, 1),
                      __shfl_down_sync(~0u, v.w, 1));
}
__device__ __forceinline__ uint2 shuffle_down(const uint2& v) {
    return make_uint2(__shfl_down_sync(~0u, v.x, 1), __shfl_down_sync(~0u, v.y, 1));
}
__device__ __forceinline__ uint32_t shuffle_down(uint32_t v) { return __shfl_down_sync(~0u, v, 1); }
// The next thread's piece: from the next lane, and for the last one what the next warp's
// first lane left in shared memory.
template <typename V>
__device__ __forceinline__ V next_piece(const V& own, const V* edge, bool last_lane) {
    V n = shuffle_down(own);
    if (last_lane) n = *edge;
    return n;
}

// A piece with only elements lo .. hi - 1 kept.
template <int BITS>
__device__ __forceinline__ uint4 keep_range(const uint4& q, int lo, int hi) {
    auto word = [&](uint32_t w, int k) {
        const int from = min(max(lo * BITS - k * 32, 0), 32), to = min(max(hi * BITS - k * 32, 0), 32);
        return w & __funnelshift_lc(~0u, 0u, to) & ~__funnelshift_lc(~0u, 0u, from);
    };
    return make_uint4(word(q.x, 0), word(q.y, 1), word(q.z, 2), word(q.w, 3));
}
// The first n elements (0 < n < 8 or 4) of an aligned piece, by words.
template <typename E>
__device__ __forceinline__ uint4 load_start(const E* p, int n) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(p);
    const int words = n * (int)sizeof(E) / 4;
    uint32_t q[4] = {0, 0, 0, 0}, last = 0;
    if (sizeof(E) == 2 && (n & 1)) last = reinterpret_cast<const uint16_t*>(p)[n - 1];
#pragma unroll
    for (int k = 0; k < 4; ++k) q[k] = k < words ? w[k] : k == words ? last : 0;
    return make_uint4(q[0], q[1], q[2], q[3]);
}
// A piece of an array of n elements from anywhere in it, 0 outside: the two aligned pieces
// around it, shifted.
template <typename E>
__device__ __forceinline__ uint4 load_anywhere(const E* array, int c, int n) {
    constexpr int P = kPiece<E>;
    const int off = (int)((reinterpret_cast<uintptr_t>(array) + (int64_t)c * (int)sizeof(E)) & 15);
    const int first = c - off / (int)sizeof(E);
    auto piece = [&](int at) {
        if (at >= 0 && at + P <= n) return *reinterpret_cast<const uint4*>(array + at);
        if (at >= n || at + P <= 0) return make_uint4(0, 0, 0, 0);
        if (at >= 0) return load_start(array + at, n - at);
        uint4 q = make_uint4(0, 0, 0, 0);           // the piece that holds an unaligned array's start
        E* e = reinterpret_cast<E*>(&q);
#pragma unroll
        for (int j = 0; j < P; ++j)
            if (at + j >= 0 && at + j < n) e[j] = array[at + j];
        return q;
    };
    const uint4 lo = piece(first);
    return off ? shift_pair(lo, piece(first + P), off >> 2, (off & 3) * 8) : lo;
}
// The bytes of a piece from `lo` on: halves of what is left, the smallest first where the piece
// ends a row's lead (its end is aligned), the largest first where it starts a row's tail.
__device__ __forceinline__ void put_bytes(uint8_t* at, uint4 q, int bytes, bool tail) {
    auto drop = [&](int n) { q = shift_pair(q, make_uint4(0, 0, 0, 0), n >> 2, (n & 3) * 8); };
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int n = tail ? 8 >> k : 1 << k;
        if (!(bytes & n)) continue;
        if (n == 8) *reinterpret_cast<uint2*>(at) = make_uint2(q.x, q.y);
        else if (n == 4) *reinterpret_cast<uint32_t*>(at) = q.x;
        else if (n == 2) *reinterpret_cast<uint16_t*>(at) = (uint16_t)q.x;
        else *at = (uint8_t)q.x;
        at += n;
        drop(n);
    }
}
__device__ __forceinline__ uint4 widen(const uint4& q) { return q; }
__device__ __forceinline__ uint4 widen(const uint2& q) { return make_uint4(q.x, q.y, 0, 0); }
__device__ __forceinline__ uint4 widen(uint32_t q) { return make_uint4(q, 0, 0, 0); }
// Stores the part of an aligned piece that lies in the row (of one piece at least).
template <typename E, typename V>
__device__ __forceinline__ void put_piece(E* row, int c, int cols, const V& v) {
    constexpr int P = sizeof(V) / sizeof(E), S = sizeof(E);
    if (c >= 0 && c + P <= cols) {
        store_piece<false>(row + c, v);
    } else if (c < 0) {
        put_bytes(reinterpret_cast<uint8_t*>(row), shift_pair(widen(v), make_uint4(0, 0, 0, 0), -c * S >> 2, (-c * S & 3) * 8), (P + c) * S, false);
    } else if (c < cols) {
        put_bytes(reinterpret_cast<uint8_t*>(row + c), widen(v), (cols - c) * S, true);
    }
}

template <int P> struct BytePiece;
template <> struct BytePiece<8> { using type = uint2; };
template <> struct BytePiece<4> { using type = uint32_t; };

// The row stays in registers: N pieces per thread, piece i of thread t at column
// (i * threads + t) * kPiece. A group of 128 columns is 16 (or 32) neighbouring lanes.
// !ALIGNED: rows of any alignment and length, read and written as aligned pieces that are
// shifted into place. That takes twice the instructions, which then bound it (4000 x 8191 bf16
// with a residual and an 8-bit output: 84 us, 2.7 TB/s; element by element 114 us).
template <typename T, typename W, int N, bool QUANT, bool ALIGNED, bool STREAM>
__global__ void __launch_bounds__(1024)
rms_norm_kernel(RmsNormArgs a) {
    constexpr int P = kPiece<T>;
    using Q = typename BytePiece<P>::type;
    __shared__ float part[32];
    __shared__ uint4 edge_h[ALIGNED ? 1 : N * 32 + 1];
    __shared__ uint4 edge_y[ALIGNED ? 1 : N * 32 + 1];
    grid_trigger();
    grid_wait();
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
    const W* w = static_cast<const W*>(a.weight);
    T* h_out = a.h_out ? static_cast<T*>(a.h_out) + row * a.h_stride : nullptr;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int threads = blockDim.x, warps = threads >> 5, cols = (int)a.cols;
    uint4 qx[N], qr[N];
    float v[N][P];
    if (ALIGNED) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = (i * threads + (int)threadIdx.x) * P;
            qx[i] = qr[i] = make_uint4(0, 0, 0, 0);
            if (c < cols) {
                qx[i] = load_piece<STREAM>(x + c);
                if (res) qr[i] = load_piece<STREAM>(res + c);
            }
        }
    } else {
        const RowLoader<T> lx(x, (uint32_t)cols, 0), lr(res, (uint32_t)cols, 0);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int u = i * threads + (int)threadIdx.x;
            qx[i] = qr[i] = make_uint4(0, 0, 0, 0);
            if (u * P < cols) {
                qx[i] = lx(u);
                if (res) qr[i] = lr(u);
            }
        }
    }
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        unpack<T>(qx[i], v[i]);
        if (res) {
            float r[P];
            unpack<T>(qr[i], r);
#pragma unroll
            for (int j = 0; j < P; ++j) v[i][j] += r[j];
        }
#pragma unroll
        for (int j = 0; j < P; ++j) sum = fmaf(v[i][j], v[i][j], sum);
        if (!ALIGNED && h_out && lane == 0) edge_h[i * warps + warp] = pack<T>(v[i]);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (lane == 0) part[warp] = sum;
    __syncthreads();
    sum = lane < warps ? part[lane] : 0.0f;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    const float r = rsqrtf(sum * a.inv_cols + a.eps);
    uint4 out[N];               // the pieces of y
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = (i * threads + (int)threadIdx.x) * P;
        if (ALIGNED) {
            if (h_out && c < cols) store_piece<STREAM>(h_out + c, pack<T>(v[i]));
        } else if (h_out) {
            const uint4 own = pack<T>(v[i]);
            const uint4 next = next_piece(own, edge_h + i * warps + warp + 1, lane == 31);
            if (c < cols) store_shifted<T, uint4>(h_out, cols, c, own, next);
        }
        float wv[P];
        if (!ALIGNED) {
            const RowLoader<W> lw(w, (uint32_t)cols, 0);
            constexpr int PW = kPiece<W>;
#pragma unroll
            for (int j = 0; j < P; j += PW) {
                float f[PW];
                unpack<W>(c + j < cols ? lw((uint32_t)(c + j) / PW) : make_uint4(0, 0, 0, 0), f);
#pragma unroll
                for (int t = 0; t < PW; ++t) wv[j + t] = f[t];
            }
        } else if (c < cols) {
            if (sizeof(W) == sizeof(T)) {
                unpack<T>(__ldg(reinterpret_cast<const uint4*>(w + c)), wv);
            } else {
#pragma unroll
                for (int j = 0; j < P; j += 4) {
                    const float4 f = __ldg(reinterpret_cast<const float4*>(w + c + j));
                    wv[j] = f.x; wv[j + 1] = f.y; wv[j + 2] = f.z; wv[j + 3] = f.w;
                }
            }
        }
        if (c < cols) {
#pragma unroll
            for (int j = 0; j < P; j += 2) {
                const float2 y = times(make_float2(v[i][j], v[i][j + 1]), r, make_float2(wv[j], wv[j + 1]));
                v[i][j] = y.x;
                v[i][j + 1] = y.y;
            }
        }
        if (!QUANT) {
            out[i] = pack<T>(v[i]);
            if (ALIGNED && c < cols) store_piece<STREAM>(static_cast<T*>(a.y) + row * a.y_stride + c, out[i]);
        } else {
            float m = kTiny;                // columns past the end count as 0
            if (c < cols) {
#pragma unroll
                for (int j = 0; j < P; ++j) m = max_nan(m, fabsf(v[i][j]));
            }
#pragma unroll
            for (int o = kGroup / P / 2; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(~0u, m, o));
            const Scale d = scale_of(m);
            if (c < cols && c % kGroup == 0) a.scales[row * a.scales_stride + c / kGroup] = d.s;
            uint32_t b[2] = {0, 0};
            const float2 inv = make_float2(d.inv, d.inv), minus = make_float2(d.minus, d.minus);
#pragma unroll
            for (int j = 0; j < P; j += 4)
                b[j / 4] = four_fp8(quotients(make_float2(v[i][j], v[i][j + 1]), inv, minus),
                                    quotients(make_float2(v[i][j + 2], v[i][j + 3]), inv, minus));
            out[i] = make_uint4(b[0], b[1], 0, 0);
            if (ALIGNED && c < cols) {
                uint8_t* y = static_cast<uint8_t*>(a.y) + row * a.y_stride + c;
                if (P == 8) store_piece<STREAM>(y, make_uint2(b[0], b[1]));
                else store_piece<STREAM>(y, b[0]);
            }
        }
        if (!ALIGNED && lane == 0) edge_y[i * warps + warp] = out[i];
    }
    if (ALIGNED) return;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = (i * threads + (int)threadIdx.x) * P;
        const uint4* edge = edge_y + i * warps + warp + 1;
        if (QUANT) {
            const Q own = *reinterpret_cast<const Q*>(&out[i]);
            const Q next = next_piece(own, reinterpret_cast<const Q*>(edge), lane == 31);
            if (c < cols) store_shifted<uint8_t, Q>(static_cast<uint8_t*>(a.y) + row * a.y_stride, cols, c, own, next);
        } else {
            const uint4 next = next_piece(out[i], edge, lane == 31);
            if (c < cols) store_shifted<T, uint4>(static_cast<T*>(a.y) + row * a.y_stride, cols, c, out[i], next);
        }
    }
}

// f(integral_constant of s), 0 <= s < P: a row's offset as a constant, so that which of a
// piece's elements belong to which group costs no instructions.
template <int P, typename F>
__device__ __forceinline__ void by_offset(int s, F f) {
    switch (s) {
        case 0: f(std::integral_constant<int, 0>()); break;
        case 1: f(std::integral_constant<int, 1>()); break;
        case 2: f(std::integral_constant<int, 2>()); break;
        case 3: f(std::integral_constant<int, 3>()); break;
        case 4: f(std::integral_constant<int, P == 8 ? 4 : 0>()); break;
        case 5: f(std::integral_constant<int, P == 8 ? 5 : 0>()); break;
        case 6: f(std::integral_constant<int, P == 8 ? 6 : 0>()); break;
        default: f(std::integral_constant<int, P == 8 ? 7 : 0>()); break;
    }
}

// Rows of one kind of offset: x, the residual, h and y of a row all start at the same element of
// an aligned piece, as those of contiguous tensors do whatever the number of columns. Pieces on
// memory's own grid, which begins s columns before the row, are read and written as they are
// and only the weights are shifted. A piece at the row's ends is read whole where the array goes
// on beyond the row, and written by halves. The order in which the squares are added depends on s.
// Bound by its instructions and its barriers, so registers are limited, to 40 with two or three pieces
// a thread, for two CTAs of 544 threads on an SM or four of 352 (4000 x 8191 bf16, residual, 8-bit output:
// 53 us, over two pieces 59, with one CTA on an SM 96, the general kernel 84; 4000 x 8190, 16-bit
// output: 43, general 84; 16000 x 2049, 8-bit: 50 against 57; 509 x 2050 f16: 2.6 against 3.0). Weights read
// early pay with one piece a thread only (2.6 against 2.75; 55 against 51 with two).
template <typename T, typename W, int N, bool QUANT>
__global__ void __launch_bounds__(N == 2 ? 768 : N == 3 ? 448 : 1024, N == 4 ? 1 : N == 3 ? 3 : 2)
rms_norm_alike_kernel(RmsNormArgs a) {
    constexpr int P = kPiece<T>, PW = kPiece<W>, H = kGroup / P;
    using Q = typename BytePiece<P>::type;
    __shared__ float part[32];
    // Largest |y| of a group without its end, and of that end, which is the first s elements of
    // the next group's first piece.
    __shared__ float top[QUANT ? N * 1024 / H : 1], low[QUANT ? N * 1024 / H : 1];
    __shared__ Scale scales[QUANT ? N * 1024 / H : 1];
    grid_trigger();
    grid_wait();
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
    const W* w = static_cast<const W*>(a.weight);
    T* h_out = a.h_out ? static_cast<T*>(a.h_out) + row * a.h_stride : nullptr;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int threads = blockDim.x, warps = threads >> 5, cols = (int)a.cols;
    const int s = (int)(reinterpret_cast<uintptr_t>(x) / sizeof(T) % P);
    const bool x_front = row * a.x_stride >= P, x_back = (a.rows - 1 - row) * a.x_stride >= P;
    const bool r_front = row * a.residual_stride >= P, r_back = (a.rows - 1 - row) * a.residual_stride >= P;
    uint4 qx[N], qr[N];
    float v[N][P];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = (i * threads + (int)threadIdx.x) * P - s;
        qx[i] = qr[i] = make_uint4(0, 0, 0, 0);
        // whole pieces, those at the row's ends too where the array goes on beyond the row
        const bool x_whole = (c >= 0 || x_front) && (c + P <= cols || x_back);
        const bool r_whole = (c >= 0 || r_front) && (c + P <= cols || r_back);
        if (c < cols) {
            if (x_whole) qx[i] = load_piece<false>(x + c);
            if (res && r_whole) qr[i] = load_piece<false>(res + c);
            if (!x_whole) qx[i] = load_anywhere(x, c, cols);
            if (res && !r_whole) qr[i] = load_anywhere(res, c, cols);
        }
    }
    uint4 wq[P / PW];                       // one piece's weights are read before the sum is known
    if (N == 1) {
#pragma unroll
        for (int j = 0; j < P / PW; ++j) wq[j] = load_anywhere(w, (int)threadIdx.x * P - s + j * PW, cols);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = (i * threads + (int)threadIdx.x) * P - s;
        if (c < 0 || c + P > cols) {
            qx[i] = keep_range<8 * sizeof(T)>(qx[i], -c, cols - c);
            qr[i] = keep_range<8 * sizeof(T)>(qr[i], -c, cols - c);
        }
    }
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        unpack<T>(qx[i], v[i]);
        if (res) {
            float r[P];
            unpack<T>(qr[i], r);
#pragma unroll
            for (int j = 0; j < P; ++j) v[i][j] += r[j];
        }
#pragma unroll
        for (int j = 0; j < P; ++j) sum = fmaf(v[i][j], v[i][j], sum);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (lane == 0) part[warp] = sum;
    __syncthreads();
    sum = lane < warps ? part[lane] : 0.0f;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    const float r = rsqrtf(sum * a.inv_cols + a.eps);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int u = i * threads + (int)threadIdx.x, c = u * P - s;
        if (h_out) put_piece(h_out, c, cols, pack<T>(v[i]));
#pragma unroll
        for (int j = 0; j < P; j += PW) {
            float f[PW];
            unpack<W>(N == 1 ? wq[j / PW] : load_anywhere(w, c + j, cols), f);
#pragma unroll
            for (int t = 0; t < PW; t += 2) {
                const float2 y = times(make_float2(v[i][j + t], v[i][j + t + 1]), r, make_float2(f[t], f[t + 1]));
                v[i][j + t] = y.x;
                v[i][j + t + 1] = y.y;
            }
        }
        if (!QUANT) {
            put_piece(static_cast<T*>(a.y) + row * a.y_stride, c, cols, pack<T>(v[i]));
        } else {
            float m = kTiny, end = kTiny;
            by_offset<P>(s, [&](auto S) {
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    if (j < S.value) end = max_nan(end, fabsf(v[i][j]));
                    else m = max_nan(m, fabsf(v[i][j]));
                }
            });
            if (lane % H) m = max_nan(m, end);
#pragma unroll
            for (int o = H / 2; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(~0u, m, o));
            if (lane % H == 0) {
                top[u / H] = m;
                low[u / H] = end;
            }
        }
    }
    if (!QUANT) return;
    __syncthreads();
    const int groups = N * threads / H;             // fewer than threads
    if ((int)threadIdx.x < groups && (int)threadIdx.x * kGroup < cols) {
        const int g = threadIdx.x;
        const float m = g + 1 < groups ? max_nan(top[g], low[g + 1]) : top[g];
        scales[g] = scale_of(m);
        a.scales[row * a.scales_stride + g] = scales[g].s;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int u = i * threads + (int)threadIdx.x, c = u * P - s;
        if (c >= cols) continue;
        const int own = min(u / H, (cols - 1) / kGroup);        // the last piece may only end a group
        const Scale d_own = scales[own], d_end = scales[lane % H || u == 0 ? own : u / H - 1];
        uint32_t b[2] = {0, 0};
        by_offset<P>(s, [&](auto S) {
#pragma unroll
            for (int j = 0; j < P; j += 4) {
                float2 f[2];
#pragma unroll
                for (int t = 0; t < 4; t += 2) {
                    const Scale &d0 = j + t < S.value ? d_end : d_own, &d1 = j + t + 1 < S.value ? d_end : d_own;
                    f[t / 2] = quotients(make_float2(v[i][j + t], v[i][j + t + 1]), make_float2(d0.inv, d1.inv),
                                         make_float2(d0.minus, d1.minus));
                }
                b[j / 4] = four_fp8(f[0], f[1]);
            }
        });
        const uint2 q = make_uint2(b[0], b[1]);
        put_piece(static_cast<uint8_t*>(a.y) + row * a.y_stride, c, cols, *reinterpret_cast<const Q*>(&q));
    }
}

// A CTA per row.
void launch_rows(void (*kernel)(RmsNormArgs), const RmsNormArgs& a, int threads, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)a.rows);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = s;
    cudaLaunchAttribute at = dependent_launch();
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    PB_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
}

enum class Rows { kWhole, kAlike, kAny };       // whole aligned pieces, one kind of offset, any

template <typename T, typename W, int N, bool QUANT, Rows ROWS>
void launch_n(const RmsNormArgs& a, int64_t pieces, cudaStream_t s) {
    const int threads = (int)std::max<int64_t>(32, ((pieces + N - 1) / N + 31) / 32 * 32);
    if constexpr (ROWS == Rows::kAny) {
        launch_rows(rms_norm_kernel<T, W, N, QUANT, false, false>, a, threads, s);
    } else if constexpr (ROWS == Rows::kAlike) {
        launch_rows(rms_norm_alike_kernel<T, W, N, QUANT>, a, threads, s);
    } else {
        // With a residual, four arrays go through the L2 cache; beyond half of its 126 MB they only
        // push each other out, and passing them through is faster (16384 x 8192 bf16, 8-bit output:
        // 139 us against 173; 8192 x 4096: 37.9 against 40.9). Without one it is not (40000 x 2048
        // bf16: 53.3 against 50.4), nor where rows share their ends' lines (8000 x 4001: 49.1
        // against 47.5).
        const bool streams = a.residual && a.rows * a.cols * (int64_t)sizeof(T) * 3 > (int64_t(64) << 20);
        launch_rows(streams ? rms_norm_kernel<T, W, N, QUANT, true, true> : rms_norm_kernel<T, W, N, QUANT, true, false>, a, threads, s);
    }
}

// Pieces per thread: one where all rows run at once (550 x 4096 bf16, residual, 8-bit: 3.5 us, with
// two 4.5; 509 x 2050 f16: 2.6 and 4.1), two for more rows (16384 x 8192: 139 us, one 182, four 142;
// 500 x 6001: 6.4, one 8.2), four for rows that two do not hold.
// Contiguous odd rows that do not run at once take three where that leaves fewer of the threads'
// slots empty than two (4000 x 8190 bf16: 43.0, two 51.3; 16000 x 2050: 32.5 and 38.3; where it
// does not: 8000 x 4001, 8-bit, 56.2 and 47.5; at once: 200 x 8191 7.7 and 5.0).
template <typename T, typename W, bool QUANT, Rows ROWS>
bool launch_pieces(const RmsNormArgs& a, cudaStream_t s) {
    const int64_t ends = ROWS == Rows::kAlike ? kPiece<T> - 1 : 0;      // columns before the row in its first piece
    const int64_t pieces = (a.cols + ends + kPiece<T> - 1) / kPiece<T>;
    if (pieces > 4 * 1024) return false;
    const int64_t most = ROWS == Rows::kAlike ? 768 : 1024;     // threads, with two pieces each
    auto slots = [&](int64_t n) { return ((pieces + n - 1) / n + 31) / 32 * 32 * n; };      // of a CTA's threads, n each
    const bool at_once = a.rows * ((pieces + 31) / 32 * 32) <= 148 * 2048;
    const bool three = ROWS == Rows::kAlike && !at_once && pieces <= 3 * 448 && slots(3) < slots(2);
    if (pieces > 2 * most) launch_n<T, W, 4, QUANT, ROWS>(a, pieces, s);
    else if (three) launch_n<T, W, ROWS == Rows::kAlike ? 3 : 2, QUANT, ROWS>(a, pieces, s);
    else if (pieces > 1024 || (!at_once && pieces > 32)) launch_n<T, W, 2, QUANT, ROWS>(a, pieces, s);
    else launch_n<T, W, 1, QUANT, ROWS>(a, pieces, s);
    return true;
}

template <typename T, typename W, bool QUANT>
void launch_typed(const RmsNormArgs& a, cudaStream_t s) {
    // Do an array's rows start at the same element of an aligned piece as x's?
    auto alike = [&](const void* p, int64_t stride, int64_t bytes) {
        const int64_t at = (int64_t)(reinterpret_cast<uintptr_t>(p) / bytes) - (int64_t)(reinterpret_cast<uintptr_t>(a.x) / sizeof(T));
        return !p || (at % kPiece<T> == 0 && (a.rows <= 1 || (stride - a.x_stride) % kPiece<T> == 0));
    };
    const int64_t e = sizeof(T);
    const bool same = alike(a.residual, a.residual_stride, e) && alike(a.h_out, a.h_stride, e) && alike(a.y, a.y_stride, QUANT ? 1 : e);
    const bool whole = same && a.cols % kPiece<T> == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0 &&
                       (a.rows <= 1 || a.x_stride % kPiece<T> == 0) && reinterpret_cast<uintptr_t>(a.weight) % 16 == 0;
    if (whole && launch_pieces<T, W, QUANT, Rows::kWhole>(a, s)) return;
    if (!whole && same && a.cols >= 2 * kPiece<T> && launch_pieces<T, W, QUANT, Rows::kAlike>(a, s)) return;
    if (!whole && launch_pieces<T, W, QUANT, Rows::kAny>(a, s)) return;
    launch_rows(rms_norm_rows_kernel<T, W>, a, 256, s);      // rows too long for the registers
}

template <typename T>
void launch_weights(const RmsNormArgs& a, cudaStream_t s) {
    if (a.weight_dtype == ENGINE_F32) a.quantize ? launch_typed<T, float, true>(a, s) : launch_typed<T, float, false>(a, s);
    else a.quantize ? launch_typed<T, T, true>(a, s) : launch_typed<T, T, false>(a, s);
}

}  // namespace

void launch_rms_norm(const RmsNormArgs& args, cudaStream_t s) {
    if (args.rows == 0 || args.cols == 0) return;
    RmsNormArgs a = args;
    a.inv_cols = 1.0f / (float)a.cols;
    switch (a.dtype) {
        case ENGINE_F32: launch_weights<float>(a, s); break;
        case ENGINE_F16: launch_weights<__half>(a, s); break;
        case ENGINE_BF16: launch_weights<__nv_bfloat16>(a, s); break;
        default: fail(ENGINE_ERR_INVALID_ARG, "rms_norm: dtype must be F32, F16 or BF16");
    }
}

}  // namespace pb
