// Entry points of the language-model operators (include/pdefa_b200_ext.h): argument
// checks, the device of the call and the launch. Device pointers only; every call just
// enqueues on the caller's stream.
#include <cmath>

#include "../../include/pdefa_b200_ext.h"
#include "kernels.h"
#include "runtime.h"

using namespace pb;

namespace {

constexpr int64_t kMaxExtent = 0x7FFFFFFF;
constexpr int64_t kMaxReach = int64_t(1) << 60;   // of a stride times its rows: byte offsets stay within 63 bits
constexpr int64_t kBlock = 128;

// Makes `device` current for a call and puts the caller's device back.
struct DeviceScope {
    int before = 0;
    bool moved = false;
    explicit DeviceScope(int device) {
        PB_CUDA(cudaGetDevice(&before));
        if (before == device) return;
        require_device(device);
        PB_CUDA(cudaSetDevice(device));
        moved = true;
    }
    ~DeviceScope() { if (moved) cudaSetDevice(before); }
};

void need(bool ok, EngineStatus s, const char* what) { if (!ok) fail(s, what); }

void need_extent(int64_t n, const char* what) {
    need(n >= 0 && n <= kMaxExtent, ENGINE_ERR_INVALID_SHAPE, what);
}

// An output's row stride: rows may not overlap, unless there is one at most.
void need_stride(int64_t stride, int64_t width, int64_t rows, const char* what) {
    need(rows <= 1 || (stride >= width && stride <= kMaxReach / rows), ENGINE_ERR_INVALID_ARG, what);
}
// An input's: its rows may overlap or be one and the same (stride 0).
void need_input_stride(int64_t stride, int64_t rows, const char* what) {
    need(rows <= 1 || (stride >= 0 && stride <= kMaxReach / rows), ENGINE_ERR_INVALID_ARG, what);
}

bool float_type(int32_t t) { return t == ENGINE_F32 || t == ENGINE_F16 || t == ENGINE_BF16; }
size_t align_of(int32_t t) { return t == ENGINE_F32 ? 4 : 2; }

void need_aligned(const void* p, size_t n, const char* what) {
    need(reinterpret_cast<uintptr_t>(p) % n == 0, ENGINE_ERR_INVALID_ARG, what);
}

EngineStatus matmul_fp8(MatmulFp8Args p, int32_t device, void* stream) {
    clear_error();
    need_extent(p.m, "matmul_fp8: bad number of rows");
    need_extent(p.n, "matmul_fp8: bad number of columns");
    need_extent(p.k, "matmul_fp8: bad inner extent");
    need(float_type(p.out_dtype), ENGINE_ERR_INVALID_ARG, "matmul_fp8: the output type must be F32, F16 or BF16");
    const int64_t kb = (p.k + kBlock - 1) / kBlock;
    const int64_t nb = (p.n + kBlock - 1) / kBlock;
    if (p.m == 0 || p.n == 0) return ENGINE_OK;
    need(p.out != nullptr, ENGINE_ERR_NULL_PTR, "matmul_fp8: no output");
    if (p.k > 0) {
        need(p.a && p.b && p.a_scales && p.b_scales, ENGINE_ERR_NULL_PTR, "matmul_fp8: an operand or its scales are missing");
        need_aligned(p.a_scales, 4, "matmul_fp8: scales of a are not aligned");
        need_aligned(p.b_scales, 4, "matmul_fp8: scales of b are not aligned");
    }
    need_input_stride(p.lda, p.m, "matmul_fp8: stride of a");
    need_input_stride(p.ldb, p.n, "matmul_fp8: stride of b");
    need_input_stride(p.lda_scales, p.m, "matmul_fp8: stride of a's scales");
    need_input_stride(p.ldb_scales, nb, "matmul_fp8: stride of b's scales");
    need_stride(p.ldo, p.n, p.m, "matmul_fp8: stride of the output");
    need_aligned(p.out, align_of(p.out_dtype), "matmul_fp8: the output is not aligned");
    if (p.offsets) {
        need(p.experts >= 1 && p.experts <= 1024, ENGINE_ERR_INVALID_SHAPE, "matmul_fp8: 1 to 1024 experts");
        need_aligned(p.offsets, 4, "matmul_fp8: the offsets are not aligned");
        need_input_stride(p.b_expert, p.experts, "matmul_fp8: expert stride of b");
        need_input_stride(p.b_scales_expert, p.experts, "matmul_fp8: expert stride of b's scales");
    }
    DeviceScope scope(device);
    launch_matmul_fp8(p, static_cast<cudaStream_t>(stream));
    return ENGINE_OK;
}

}  // namespace

extern "C" {

ENGINE_API EngineStatus engine_rms_norm_device(const void* d_x, int64_t x_stride, const void* d_residual,
                                               int64_t residual_stride, const void* d_weight, void* d_h,
                                               int64_t h_stride, void* d_y, int64_t y_stride, float* d_scales,
                                               int64_t scales_stride, int64_t rows, int64_t cols, int32_t dtype,
                                               int32_t weight_dtype, float eps, int32_t device, void* stream) {
    return guarded([&]() -> EngineStatus {
        clear_error();
        need_extent(rows, "rms_norm: bad number of rows");
        need_extent(cols, "rms_norm: bad number of columns");
        need(float_type(dtype), ENGINE_ERR_INVALID_ARG, "rms_norm: dtype must be F32, F16 or BF16");
        need(weight_dtype == dtype || weight_dtype == ENGINE_F32, ENGINE_ERR_INVALID_ARG,
             "rms_norm: the weight must be of x's type or F32");
        need(std::isfinite(eps) && eps >= 0.0f, ENGINE_ERR_INVALID_ARG, "rms_norm: eps must be finite and >= 0");
        if (rows == 0 || cols == 0) return ENGINE_OK;
        need(d_x && d_weight && d_y, ENGINE_ERR_NULL_PTR, "rms_norm: x, weight and y are needed");
        need_input_stride(x_stride, rows, "rms_norm: stride of x");
        need_stride(y_stride, cols, rows, "rms_norm: stride of y");
        need_aligned(d_x, align_of(dtype), "rms_norm: x is not aligned");
        need_aligned(d_weight, align_of(weight_dtype), "rms_norm: the weight is not aligned");
        if (d_residual) {
            need_input_stride(residual_stride, rows, "rms_norm: stride of the residual");
            need_aligned(d_residual, align_of(dtype), "rms_norm: the residual is not aligned");
        }
        if (d_h) {
            need_stride(h_stride, cols, rows, "rms_norm: stride of h");
            need_aligned(d_h, align_of(dtype), "rms_norm: h is not aligned");
        }
        if (d_scales) {
            need_stride(scales_stride, (cols + kBlock - 1) / kBlock, rows, "rms_norm: stride of the scales");
            need_aligned(d_scales, 4, "rms_norm: the scales are not aligned");
        } else {
            need_aligned(d_y, align_of(dtype), "rms_norm: y is not aligned");
        }
        DeviceScope scope(device);
        RmsNormArgs a;
        a.x = d_x; a.residual = d_residual; a.weight = d_weight; a.h_out = d_h; a.y = d_y; a.scales = d_scales;
        a.rows = rows; a.cols = cols;
        a.x_stride = x_stride; a.residual_stride = residual_stride; a.h_stride = h_stride;
        a.y_stride = y_stride; a.scales_stride = scales_stride;
        a.eps = eps; a.dtype = dtype; a.weight_dtype = weight_dtype; a.quantize = d_scales != nullptr;
        launch_rms_norm(a, static_cast<cudaStream_t>(stream));
        return ENGINE_OK;
    });
}

ENGINE_API EngineStatus engine_matmul_fp8_device(const void* d_a, int64_t lda, const float* d_a_scales,
                                                 int64_t lda_scales, const void* d_b, int64_t ldb,
                                                 const float* d_b_scales, int64_t ldb_scales, void* d_out, int64_t ldo,
                                                 int32_t out_dtype, int64_t m, int64_t n, int64_t k, int32_t device,
                                                 void* stream) {
    return guarded([&]() -> EngineStatus {
        MatmulFp8Args p;
        p.a = d_a; p.b = d_b; p.a_scales = d_a_scales; p.b_scales = d_b_scales; p.out = d_out;
        p.m = m; p.n = n; p.k = k;
        p.lda = lda; p.ldb = ldb; p.lda_scales = lda_scales; p.ldb_scales = ldb_scales; p.ldo = ldo;
        p.out_dtype = out_dtype;
        return matmul_fp8(p, device, stream);
    });
}

ENGINE_API EngineStatus engine_matmul_grouped_fp8_device(const void* d_a, int64_t lda, const float* d_a_scales,
                                                         int64_t lda_scales, const void* d_b, int64_t ldb,
                                                         int64_t b_expert_stride, const float* d_b_scales,
                                                         int64_t ldb_scales, int64_t b_scales_expert_stride,
                                                         const int32_t* d_offsets, int64_t experts, void* d_out,
                                                         int64_t ldo, int32_t out_dtype, int64_t rows, int64_t n,
                                                         int64_t k, int32_t device, void* stream) {
    return guarded([&]() -> EngineStatus {
        if (!d_offsets) { set_error("matmul_fp8: no offsets"); return ENGINE_ERR_NULL_PTR; }
        MatmulFp8Args p;
        p.a = d_a; p.b = d_b; p.a_scales = d_a_scales; p.b_scales = d_b_scales; p.out = d_out;
        p.offsets = d_offsets; p.experts = experts;
        p.m = rows; p.n = n; p.k = k;
        p.lda = lda; p.ldb = ldb; p.lda_scales = lda_scales; p.ldb_scales = ldb_scales; p.ldo = ldo;
        p.b_expert = b_expert_stride; p.b_scales_expert = b_scales_expert_stride;
        p.out_dtype = out_dtype;
        return matmul_fp8(p, device, stream);
    });
}

ENGINE_API EngineStatus engine_matmul_fp8_plan(int64_t m, int64_t n, int64_t k, int64_t experts, int32_t out_dtype,
                                               int32_t aligned_out, int32_t sms, const int32_t clusters[3],
                                               int32_t plan[3]) {
    return guarded([&]() -> EngineStatus {
        clear_error();
        need_extent(m, "matmul_fp8: bad number of rows");
        need_extent(n, "matmul_fp8: bad number of columns");
        need_extent(k, "matmul_fp8: bad inner extent");
        need(m > 0 && n > 0 && k > 0 && experts >= 0 && experts <= 1024, ENGINE_ERR_INVALID_SHAPE, "matmul_fp8: nothing to plan");
        need(float_type(out_dtype), ENGINE_ERR_INVALID_ARG, "matmul_fp8: the output type must be F32, F16 or BF16");
        need(sms >= 2, ENGINE_ERR_INVALID_ARG, "matmul_fp8: too few SMs");
        need(clusters && plan, ENGINE_ERR_NULL_PTR, "matmul_fp8: nowhere to put the plan");
        static const int32_t none = 0;
        MatmulFp8Args p;
        p.m = m; p.n = n; p.k = k; p.out_dtype = out_dtype;
        if (experts) { p.offsets = &none; p.experts = experts; }       // not read
        const int32_t held[3] = {clusters[0], clusters[1], clusters[2]};
        int32_t found[3];
        matmul_fp8_plan(p, aligned_out != 0, sms, held, found);
        for (int i = 0; i < 3; ++i) plan[i] = found[i];
        return ENGINE_OK;
    });
}

ENGINE_API EngineStatus engine_sample_device(const void* d_logits, int64_t logits_stride, int32_t dtype,
                                             const float* d_noise, int64_t noise_stride, const float* d_temperature,
                                             const int32_t* d_top_k, const float* d_top_p, const float* d_min_p,
                                             int64_t rows, int64_t vocab, int32_t* d_tokens, float* d_probs,
                                             int32_t device, void* stream) {
    return guarded([&]() -> EngineStatus {
        clear_error();
        need_extent(rows, "sample: bad number of rows");
        need(vocab >= 1 && vocab <= kMaxExtent, ENGINE_ERR_INVALID_SHAPE, "sample: a row needs 1 to 2^31 - 1 logits");
        need(float_type(dtype), ENGINE_ERR_INVALID_ARG, "sample: dtype must be F32, F16 or BF16");
        if (rows == 0) return ENGINE_OK;
        need(d_logits && d_noise && d_tokens, ENGINE_ERR_NULL_PTR, "sample: logits, noise and tokens are needed");
        need_input_stride(logits_stride, rows, "sample: stride of the logits");
        need_input_stride(noise_stride, rows, "sample: stride of the noise");
        need_aligned(d_logits, align_of(dtype), "sample: the logits are not aligned");
        const void* words[] = {d_noise, d_temperature, d_top_k, d_top_p, d_min_p, d_tokens, d_probs};
        for (const void* w : words) need_aligned(w, 4, "sample: an array is not aligned");
        DeviceScope scope(device);
        SampleArgs a;
        a.logits = d_logits; a.noise = d_noise; a.temperature = d_temperature; a.top_k = d_top_k;
        a.top_p = d_top_p; a.min_p = d_min_p; a.tokens = d_tokens; a.probs = d_probs;
        a.rows = rows; a.vocab = vocab; a.logits_stride = logits_stride; a.noise_stride = noise_stride;
        a.dtype = dtype;
        launch_sample(a, static_cast<cudaStream_t>(stream));
        return ENGINE_OK;
    });
}

ENGINE_API EngineStatus engine_sample_plan(int64_t rows, int64_t vocab, int32_t dtype, int32_t* ctas) {
    return guarded([&]() -> EngineStatus {
        clear_error();
        need_extent(rows, "sample: bad number of rows");
        need(vocab >= 1 && vocab <= kMaxExtent, ENGINE_ERR_INVALID_SHAPE, "sample: a row needs 1 to 2^31 - 1 logits");
        need(float_type(dtype), ENGINE_ERR_INVALID_ARG, "sample: dtype must be F32, F16 or BF16");
        need(ctas != nullptr, ENGINE_ERR_NULL_PTR, "sample: nowhere to put the plan");
        *ctas = sample_plan(rows, vocab, dtype);
        return ENGINE_OK;
    });
}

}  // extern "C"
