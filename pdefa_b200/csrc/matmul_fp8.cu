// Matrix product of 8-bit floating-point operands (e4m3) with block scales:
//
//   out[m, n] = sum over kb of sa[m, kb] * sb[n / 128, kb] *
//               (sum over the 128 k of block kb of a[m, k] * b[n, k])
//
// a is [M, K] (rows are tokens), b is [N, K] (a weight as it is stored), or
// [experts, N, K] with `offsets` giving each expert's range of rows of a. The inner
// sum of a block is exact products in 32-bit accumulation; blocks are joined in
// 32 bits.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.h"
#include "device_common.cuh"

namespace pb {

namespace {

constexpr int kBlock = 128;

__device__ __forceinline__ float e4m3(uint8_t v) {
    __nv_fp8_e4m3 f;
    f.__x = v;
    return (float)f;
}

__device__ __forceinline__ void store_out(void* out, int dtype, int64_t i, float v) {
    if (dtype == ENGINE_F32) static_cast<float*>(out)[i] = v;
    else if (dtype == ENGINE_F16) static_cast<__half*>(out)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
}

// One thread per output.
__global__ void __launch_bounds__(256)
matmul_fp8_simple_kernel(MatmulFp8Args p) {
    const int64_t n = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
    const int64_t m = (int64_t)blockIdx.y * 8 + (threadIdx.x >> 5);
    if (m >= p.m || n >= p.n) return;
    const uint8_t* b = static_cast<const uint8_t*>(p.b);
    const float* sb = p.b_scales;
    if (p.offsets) {
        int e = 0;
        while (e < p.experts && !(p.offsets[e] <= m && m < p.offsets[e + 1])) ++e;
        if (e == p.experts) {
            store_out(p.out, p.out_dtype, m * p.ldo + n, 0.0f);
            return;
        }
        b += e * p.b_expert;
        sb += e * p.b_scales_expert;
    }
    const uint8_t* ar = static_cast<const uint8_t*>(p.a) + m * p.lda;
    const uint8_t* br = b + n * p.ldb;
    float sum = 0.0f;
    for (int64_t k0 = 0; k0 < p.k; k0 += kBlock) {
        float part = 0.0f;
        const int64_t k1 = k0 + kBlock < p.k ? k0 + kBlock : p.k;
        for (int64_t k = k0; k < k1; ++k) part = fmaf(e4m3(ar[k]), e4m3(br[k]), part);
        sum = fmaf(part, p.a_scales[m * p.lda_scales + k0 / kBlock] * sb[n / kBlock * p.ldb_scales + k0 / kBlock], sum);
    }
    store_out(p.out, p.out_dtype, m * p.ldo + n, sum);
}

}  // namespace

void launch_matmul_fp8(const MatmulFp8Args& p, cudaStream_t s) {
    if (p.m == 0 || p.n == 0) return;
    for (int64_t m0 = 0; m0 < p.m; m0 += 65535 * 8) {      // grid rows are limited to 65535
        if (m0) fail(ENGINE_ERR_NOT_IMPL, "matmul_fp8: more than 524280 rows");
    }
    dim3 grid((unsigned)((p.n + 31) / 32), (unsigned)((p.m + 7) / 8));
    matmul_fp8_simple_kernel<<<grid, 256, 0, s>>>(p);
    PB_CUDA(cudaGetLastError());
}

}  // namespace pb
