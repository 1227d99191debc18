// Root-mean-square norm of rows, with the addition of a residual before it and, if
// wanted, the 8-bit form of the result with one scale for each 128 columns.
//
//   h = x + residual (32 bits), h_out = round(h)
//   y = h * w / sqrt(mean(h^2) + eps)
//   8-bit: scale = max(max|y| over 128 columns, 1e-10) / 448, q = e4m3(y / scale)
//
// The statistic and the scales come from the unrounded 32-bit sum. A NaN in a row
// makes its whole output NaN (an infinity makes the statistic 0 and itself NaN).
#include <algorithm>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.h"
#include "device_common.cuh"

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

// One CTA per row; every pass reads the row again (from L2 after the first).
template <typename T, typename W>
__global__ void __launch_bounds__(256)
rms_norm_rows_kernel(RmsNormArgs a) {
    __shared__ float part[8];
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

// The row stays in registers: N pieces per thread, piece i of thread t at column
// (i * threads + t) * kPiece. A group of 128 columns is 16 (or 32) neighbouring lanes.
template <typename T, typename W, int N, bool QUANT>
__global__ void __launch_bounds__(1024)
rms_norm_kernel(RmsNormArgs a) {
    constexpr int P = kPiece<T>;
    __shared__ float part[32];
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
    const W* w = static_cast<const W*>(a.weight);
    T* h_out = a.h_out ? static_cast<T*>(a.h_out) + row * a.h_stride : nullptr;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int threads = blockDim.x, cols = (int)a.cols;
    uint4 qx[N], qr[N];
    float v[N][P];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = (i * threads + (int)threadIdx.x) * P;
        qx[i] = qr[i] = make_uint4(0, 0, 0, 0);
        if (c < cols) {
            qx[i] = *reinterpret_cast<const uint4*>(x + c);
            if (res) qr[i] = *reinterpret_cast<const uint4*>(res + c);
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
    sum = lane < (threads >> 5) ? part[lane] : 0.0f;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    const float r = rsqrtf(sum / (float)cols + a.eps);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = (i * threads + (int)threadIdx.x) * P;
        if (c < cols) {
            if (h_out) *reinterpret_cast<uint4*>(h_out + c) = pack<T>(v[i]);
            float wv[P];
            if (sizeof(W) == sizeof(T)) {
                unpack<T>(__ldg(reinterpret_cast<const uint4*>(w + c)), wv);
            } else {
#pragma unroll
                for (int j = 0; j < P; j += 4) {
                    const float4 f = __ldg(reinterpret_cast<const float4*>(w + c + j));
                    wv[j] = f.x; wv[j + 1] = f.y; wv[j + 2] = f.z; wv[j + 3] = f.w;
                }
            }
#pragma unroll
            for (int j = 0; j < P; ++j) v[i][j] = v[i][j] * r * wv[j];
        }
        if (!QUANT) {
            if (c < cols) *reinterpret_cast<uint4*>(static_cast<T*>(a.y) + row * a.y_stride + c) = pack<T>(v[i]);
            continue;
        }
        float m = kTiny;                    // columns past the end count as 0
        if (c < cols) {
#pragma unroll
            for (int j = 0; j < P; ++j) m = max_nan(m, fabsf(v[i][j]));
        }
#pragma unroll
        for (int o = kGroup / P / 2; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(~0u, m, o));
        if (c >= cols) continue;
        if (c % kGroup == 0) a.scales[row * a.scales_stride + c / kGroup] = m / kE4m3Max;
        // the quotient by the scale as a product: one division per thread and not per value,
        // within an ulp of 32 bits of it
        const float inv = kE4m3Max / m;
        uint8_t* y = static_cast<uint8_t*>(a.y) + row * a.y_stride + c;
        uint32_t out[P / 4];
#pragma unroll
        for (int j = 0; j < P; j += 4) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[i][j] * inv, v[i][j + 1] * inv), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[i][j + 2] * inv, v[i][j + 3] * inv), __NV_SATFINITE, __NV_E4M3);
            out[j / 4] = lo | hi << 16;
        }
        if (P == 8) *reinterpret_cast<uint2*>(y) = make_uint2(out[0], out[P / 4 - 1]);
        else *reinterpret_cast<uint32_t*>(y) = out[0];
    }
}

// Pieces per thread and threads: few rows get many threads with a piece each (the time is
// that of one row), many rows get up to 4 pieces per thread.
template <typename T, typename W, bool QUANT>
bool launch_pieces(const RmsNormArgs& a, cudaStream_t s) {
    const int64_t pieces = (a.cols + kPiece<T> - 1) / kPiece<T>;
    int n = a.rows <= 296 ? 1 : 4;
    while (n > 1 && pieces <= 128 * (n / 2)) n /= 2;
    while (n < 4 && pieces > 1024 * n) n *= 2;
    if (pieces > 1024 * n) return false;
    const int threads = (int)std::max<int64_t>(32, ((pieces + n - 1) / n + 31) / 32 * 32);
    const unsigned grid = (unsigned)a.rows;
    if (n == 1) rms_norm_kernel<T, W, 1, QUANT><<<grid, threads, 0, s>>>(a);
    else if (n == 2) rms_norm_kernel<T, W, 2, QUANT><<<grid, threads, 0, s>>>(a);
    else rms_norm_kernel<T, W, 4, QUANT><<<grid, threads, 0, s>>>(a);
    return true;
}

template <typename T, typename W>
void launch_typed(const RmsNormArgs& a, cudaStream_t s) {
    // 16-byte pieces need their alignment everywhere, and rows that end with one; other rows
    // and those too long for the registers go element by element.
    auto whole = [&](const void* p, int64_t stride, int64_t bytes, int64_t piece) {
        return !p || (reinterpret_cast<uintptr_t>(p) % piece == 0 && (a.rows <= 1 || stride * bytes % piece == 0));
    };
    const int64_t e = sizeof(T);
    const bool pieces = a.cols % kPiece<T> == 0 && whole(a.x, a.x_stride, e, 16) && whole(a.residual, a.residual_stride, e, 16) &&
                        whole(a.h_out, a.h_stride, e, 16) && reinterpret_cast<uintptr_t>(a.weight) % 16 == 0 &&
                        (a.quantize ? whole(a.y, a.y_stride, 1, kPiece<T>) : whole(a.y, a.y_stride, e, 16));
    if (pieces && (a.quantize ? launch_pieces<T, W, true>(a, s) : launch_pieces<T, W, false>(a, s))) return;
    rms_norm_rows_kernel<T, W><<<(unsigned)a.rows, 256, 0, s>>>(a);
}

template <typename T>
void launch_weights(const RmsNormArgs& a, cudaStream_t s) {
    if (a.weight_dtype == ENGINE_F32) launch_typed<T, float>(a, s);
    else launch_typed<T, T>(a, s);
}

}  // namespace

void launch_rms_norm(const RmsNormArgs& a, cudaStream_t s) {
    if (a.rows == 0 || a.cols == 0) return;
    switch (a.dtype) {
        case ENGINE_F32: launch_typed<float, float>(a, s); break;
        case ENGINE_F16: launch_weights<__half>(a, s); break;
        case ENGINE_BF16: launch_weights<__nv_bfloat16>(a, s); break;
        default: fail(ENGINE_ERR_INVALID_ARG, "rms_norm: dtype must be F32, F16 or BF16");
    }
    PB_CUDA(cudaGetLastError());
}

}  // namespace pb
