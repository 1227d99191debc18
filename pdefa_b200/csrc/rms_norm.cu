// Root-mean-square norm of rows, with the addition of a residual before it and, if
// wanted, the 8-bit form of the result with one scale for each 128 columns.
//
//   h = x + residual (32 bits), h_out = round(h)
//   y = h * w / sqrt(mean(h^2) + eps)
//   8-bit: scale = max(max|y| over 128 columns, 1e-10) / 448, q = e4m3(y / scale)
//
// The statistic and the scales come from the unrounded 32-bit sum. A NaN in a row
// makes its whole output NaN (an infinity makes the statistic 0 and itself NaN).
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

template <typename T>
void launch_typed(const RmsNormArgs& a, cudaStream_t s) {
    if (a.weight_dtype == ENGINE_F32) rms_norm_rows_kernel<T, float><<<(unsigned)a.rows, 256, 0, s>>>(a);
    else rms_norm_rows_kernel<T, T><<<(unsigned)a.rows, 256, 0, s>>>(a);
}

}  // namespace

void launch_rms_norm(const RmsNormArgs& a, cudaStream_t s) {
    if (a.rows == 0 || a.cols == 0) return;
    switch (a.dtype) {
        case ENGINE_F32: launch_typed<float>(a, s); break;
        case ENGINE_F16: launch_typed<__half>(a, s); break;
        case ENGINE_BF16: launch_typed<__nv_bfloat16>(a, s); break;
        default: fail(ENGINE_ERR_INVALID_ARG, "rms_norm: dtype must be F32, F16 or BF16");
    }
    PB_CUDA(cudaGetLastError());
}

}  // namespace pb
