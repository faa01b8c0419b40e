// glm_matrix_capi.cu -- the extern "C" entry points declared in include/glm_matrix_b200.h.
//
// Each checks its arguments before it touches a device, then launches on the
// caller's stream.
#include <cmath>

#include "glm_matrix_b200.h"
#include "glm_ortho.cuh"
#include "glm_q4.cuh"

static_assert(GLMM_MAX_STEPS == glmb::kOrthoMaxSteps);

namespace glmb {

int device_check();  // glm_capi.cu

namespace {

template <typename F>
int guarded_call(F&& f) {
    try {
        return f();
    } catch (...) {
        return GLMB_ERR_INVALID_VALUE;
    }
}

// Sizes whose element counts (and byte counts, with the library's own padding) stay within 2^58.
bool sizes_ok(int64_t a, int64_t b, int64_t c, int64_t d = 1) {
    int64_t n = 1;
    for (int64_t x : {a, b, c, d}) {
        if (x > (int64_t(1) << 40)) return false;
        if (x > 0 && n > (int64_t(1) << 58) / (x + 128)) return false;
        n *= x > 0 ? x + 128 : 1;
    }
    return true;
}

// Whether [p, p + pn) and [q, q + qn) share a byte.
bool overlap(const void* p, size_t pn, const void* q, size_t qn) {
    const auto a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
    return a < b + qn && b < a + pn;
}

bool group_ok(int group) { return group == 64 || group == 128; }
bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

template <typename T>
int orthogonalize_impl(const T* G, T* O, int64_t nf, int64_t nt, int64_t ntasks, const double* coefficients, int steps,
                       void* ws, size_t ws_bytes, cudaStream_t stream) {
    if (nf < 0 || nt < 0 || ntasks < 0) return GLMB_ERR_INVALID_VALUE;
    OrthoSteps plan;
    int st = ortho_plan_steps(coefficients, steps, &plan);
    if (st != GLMB_OK) return st;
    if (nf == 0 || nt == 0 || ntasks == 0) return GLMB_OK;
    if (G == nullptr || O == nullptr || !aligned(ws, 256)) return GLMB_ERR_INVALID_VALUE;
    if (!sizes_ok(nf, nt, ntasks)) return GLMB_ERR_TOO_LARGE;
    const size_t bytes = size_t(nf) * size_t(nt) * size_t(ntasks) * sizeof(T);
    if (G != O && overlap(G, bytes, O, bytes)) return GLMB_ERR_INVALID_VALUE;
    if ((st = device_check()) != GLMB_OK) return st;
    return ortho_run<T>(G, nullptr, O, nf, nt, ntasks, plan, nullptr, ws, ws_bytes, stream);
}

template <typename T>
int step_impl(T* M, const T* grad, float* V, int64_t nf, int64_t nt, int64_t ntasks, double lr, double mu,
              double weight_decay, double scale, uint32_t flags, const double* coefficients, int steps, void* ws,
              size_t ws_bytes, cudaStream_t stream) {
    if (nf < 0 || nt < 0 || ntasks < 0 || (flags & ~GLMM_STEP_NESTEROV) != 0) return GLMB_ERR_INVALID_VALUE;
    if (!std::isfinite(lr) || !std::isfinite(mu) || !std::isfinite(weight_decay) || !std::isfinite(scale))
        return GLMB_ERR_INVALID_VALUE;
    // what the kernels take, as floats; finite arguments can still have products that are not
    const OrthoUpdate up{float(mu), (flags & GLMM_STEP_NESTEROV) != 0, float(1.0 - lr * weight_decay),
                         float(lr * scale)};
    if (!std::isfinite(up.mu) || !std::isfinite(up.keep) || !std::isfinite(up.rate)) return GLMB_ERR_INVALID_VALUE;
    OrthoSteps plan;
    int st = ortho_plan_steps(coefficients, steps, &plan);
    if (st != GLMB_OK) return st;
    if (nf == 0 || nt == 0 || ntasks == 0) return GLMB_OK;
    if (M == nullptr || grad == nullptr || V == nullptr || !aligned(ws, 256)) return GLMB_ERR_INVALID_VALUE;
    if (!sizes_ok(nf, nt, ntasks)) return GLMB_ERR_TOO_LARGE;
    const size_t n = size_t(nf) * size_t(nt) * size_t(ntasks);
    if (overlap(M, n * sizeof(T), grad, n * sizeof(T)) || overlap(M, n * sizeof(T), V, n * sizeof(float)) ||
        overlap(grad, n * sizeof(T), V, n * sizeof(float)))
        return GLMB_ERR_INVALID_VALUE;
    if ((st = device_check()) != GLMB_OK) return st;
    return ortho_run<T>(grad, V, M, nf, nt, ntasks, plan, &up, ws, ws_bytes, stream);
}

// Whether an array lies apart from a 4-bit model's codes and scales (and those from one another).
template <typename T>
bool apart(const void* p, size_t bytes, const void* codes, const T* scales, int64_t nf, int64_t nt, int64_t ntasks,
           int group) {
    const size_t blocks = size_t(ntasks) * size_t(q4_row_blocks(nt));
    const size_t cb = blocks * size_t(q4_col_blocks(nf)) * kQ4BlockBytes,
                 sb = blocks * kQ4Rows * size_t(q4_groups(nf, group)) * sizeof(T);
    return !overlap(p, bytes, codes, cb) && !overlap(p, bytes, scales, sb) && !overlap(codes, cb, scales, sb);
}

template <typename T>
int quantize_impl(const T* M, void* codes, T* scales, int64_t nf, int64_t nt, int64_t ntasks, int group,
                  cudaStream_t stream) {
    if (nf < 0 || nt < 0 || ntasks < 0 || !group_ok(group)) return GLMB_ERR_INVALID_VALUE;
    if (nf == 0 || nt == 0 || ntasks == 0) return GLMB_OK;
    if (M == nullptr || codes == nullptr || scales == nullptr || !aligned(codes, 16)) return GLMB_ERR_INVALID_VALUE;
    if (!sizes_ok(nf, nt, ntasks)) return GLMB_ERR_TOO_LARGE;
    if (!apart(M, size_t(nf) * size_t(nt) * size_t(ntasks) * sizeof(T), codes, scales, nf, nt, ntasks, group))
        return GLMB_ERR_INVALID_VALUE;
    if (const int st = device_check(); st != GLMB_OK) return st;
    return q4_quantize<T>(M, codes, scales, nf, nt, ntasks, group, stream);
}

template <typename T>
int dequantize_impl(const void* codes, const T* scales, T* M, int64_t nf, int64_t nt, int64_t ntasks, int group,
                    cudaStream_t stream) {
    if (nf < 0 || nt < 0 || ntasks < 0 || !group_ok(group)) return GLMB_ERR_INVALID_VALUE;
    if (nf == 0 || nt == 0 || ntasks == 0) return GLMB_OK;
    if (M == nullptr || codes == nullptr || scales == nullptr || !aligned(codes, 16)) return GLMB_ERR_INVALID_VALUE;
    if (!sizes_ok(nf, nt, ntasks)) return GLMB_ERR_TOO_LARGE;
    if (!apart(M, size_t(nf) * size_t(nt) * size_t(ntasks) * sizeof(T), codes, scales, nf, nt, ntasks, group))
        return GLMB_ERR_INVALID_VALUE;
    if (const int st = device_check(); st != GLMB_OK) return st;
    return q4_dequantize<T>(codes, scales, M, nf, nt, ntasks, group, stream);
}

template <typename T>
int predict_q4_impl(const T* X, const void* codes, const T* scales, T* Yhat, int64_t nf, int64_t nt, int64_t ntasks,
                    int64_t nobs, int group, void* ws, size_t ws_bytes, cudaStream_t stream) {
    if (nf < 0 || nt < 0 || ntasks < 0 || nobs < 0 || !group_ok(group)) return GLMB_ERR_INVALID_VALUE;
    if (nt == 0 || ntasks == 0 || nobs == 0) return GLMB_OK;
    if (Yhat == nullptr || !aligned(ws, 256)) return GLMB_ERR_INVALID_VALUE;
    if (nf > 0 && (X == nullptr || codes == nullptr || scales == nullptr || !aligned(codes, 16)))
        return GLMB_ERR_INVALID_VALUE;
    if (!sizes_ok(nf, nt, ntasks) || !sizes_ok(nf, ntasks, nobs) || !sizes_ok(nt, ntasks, nobs))
        return GLMB_ERR_TOO_LARGE;
    const size_t rows = size_t(ntasks) * size_t(nobs) * sizeof(T);
    if (nf > 0 && (overlap(X, rows * size_t(nf), Yhat, rows * size_t(nt)) ||
                   !apart(Yhat, rows * size_t(nt), codes, scales, nf, nt, ntasks, group)))
        return GLMB_ERR_INVALID_VALUE;
    if (const int st = device_check(); st != GLMB_OK) return st;
    if (nf == 0) {
        set_last_path("memset");
        return int(cudaMemsetAsync(Yhat, 0, size_t(nt) * size_t(ntasks) * size_t(nobs) * sizeof(T), stream));
    }
    return q4_predict<T>(X, codes, scales, Yhat, nf, nt, ntasks, nobs, group, ws, ws_bytes, stream);
}

}  // namespace
}  // namespace glmb

extern "C" {

int64_t glmm_q4_codes_bytes(int64_t nf, int64_t nt, int64_t ntasks) {
    if (nf <= 0 || nt <= 0 || ntasks <= 0 || !glmb::sizes_ok(nf, nt, ntasks)) return 0;
    return ntasks * glmb::q4_row_blocks(nt) * glmb::q4_col_blocks(nf) * glmb::kQ4BlockBytes;
}

int64_t glmm_q4_scales_count(int64_t nf, int64_t nt, int64_t ntasks, int group) {
    if (nf <= 0 || nt <= 0 || ntasks <= 0 || !glmb::group_ok(group) || !glmb::sizes_ok(nf, nt, ntasks)) return 0;
    return ntasks * glmb::q4_row_blocks(nt) * glmb::kQ4Rows * glmb::q4_groups(nf, group);
}

#define GLMM_DEFINE(SFX, CT, NT_)                                                                                    \
    size_t glmm_orthogonal_workspace_size_##SFX(int64_t nf, int64_t nt, int64_t ntasks) {                            \
        if (nf <= 0 || nt <= 0 || ntasks <= 0 || !glmb::sizes_ok(nf, nt, ntasks)) return 0;                          \
        try {                                                                                                        \
            return glmb::ortho_workspace<NT_>(nf, nt, ntasks);                                                       \
        } catch (...) {                                                                                              \
            return 0;                                                                                                \
        }                                                                                                            \
    }                                                                                                                \
    int glmm_orthogonalize_##SFX(const CT* G, CT* O, int64_t nf, int64_t nt, int64_t ntasks,                         \
                                 const double* coefficients, int steps, void* workspace, size_t workspace_bytes,     \
                                 glmb_stream_t stream) {                                                             \
        return glmb::guarded_call([&] {                                                                              \
            return glmb::orthogonalize_impl<NT_>(reinterpret_cast<const NT_*>(G), reinterpret_cast<NT_*>(O), nf, nt, \
                                                 ntasks, coefficients, steps, workspace, workspace_bytes,            \
                                                 reinterpret_cast<cudaStream_t>(stream));                            \
        });                                                                                                          \
    }                                                                                                                \
    int glmm_orthogonal_step_##SFX(CT* M, const CT* grad, float* momentum, int64_t nf, int64_t nt, int64_t ntasks,   \
                                   double lr, double mu, double weight_decay, double scale, uint32_t flags,          \
                                   const double* coefficients, int steps, void* workspace, size_t workspace_bytes,   \
                                   glmb_stream_t stream) {                                                           \
        return glmb::guarded_call([&] {                                                                              \
            return glmb::step_impl<NT_>(reinterpret_cast<NT_*>(M), reinterpret_cast<const NT_*>(grad), momentum, nf, \
                                        nt, ntasks, lr, mu, weight_decay, scale, flags, coefficients, steps,         \
                                        workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));         \
        });                                                                                                          \
    }                                                                                                                \
    int glmm_quantize_q4_##SFX(const CT* M, void* codes, CT* scales, int64_t nf, int64_t nt, int64_t ntasks,         \
                               int group, glmb_stream_t stream) {                                                    \
        return glmb::guarded_call([&] {                                                                              \
            return glmb::quantize_impl<NT_>(reinterpret_cast<const NT_*>(M), codes, reinterpret_cast<NT_*>(scales),  \
                                            nf, nt, ntasks, group, reinterpret_cast<cudaStream_t>(stream));          \
        });                                                                                                          \
    }                                                                                                                \
    int glmm_dequantize_q4_##SFX(const void* codes, const CT* scales, CT* M, int64_t nf, int64_t nt, int64_t ntasks, \
                                 int group, glmb_stream_t stream) {                                                  \
        return glmb::guarded_call([&] {                                                                              \
            return glmb::dequantize_impl<NT_>(codes, reinterpret_cast<const NT_*>(scales),                           \
                                              reinterpret_cast<NT_*>(M), nf, nt, ntasks, group,                      \
                                              reinterpret_cast<cudaStream_t>(stream));                               \
        });                                                                                                          \
    }                                                                                                                \
    size_t glmm_predict_q4_workspace_size_##SFX(int64_t nf, int64_t nt, int64_t ntasks, int64_t nobs, int group) {   \
        if (nf <= 0 || nt <= 0 || ntasks <= 0 || nobs <= 0 || !glmb::group_ok(group) ||                              \
            !glmb::sizes_ok(nf, nt, ntasks) || !glmb::sizes_ok(nf, ntasks, nobs) ||                                  \
            !glmb::sizes_ok(nt, ntasks, nobs))                                                                       \
            return 0;                                                                                                \
        try {                                                                                                        \
            return glmb::q4_predict_workspace<NT_>(nf, nt, ntasks, nobs, group);                                     \
        } catch (...) {                                                                                              \
            return 0;                                                                                                \
        }                                                                                                            \
    }                                                                                                                \
    int glmm_predict_q4_##SFX(const CT* X, const void* codes, const CT* scales, CT* Yhat, int64_t nf, int64_t nt,    \
                              int64_t ntasks, int64_t nobs, int group, void* workspace, size_t workspace_bytes,      \
                              glmb_stream_t stream) {                                                                \
        return glmb::guarded_call([&] {                                                                              \
            return glmb::predict_q4_impl<NT_>(reinterpret_cast<const NT_*>(X), codes,                                \
                                              reinterpret_cast<const NT_*>(scales), reinterpret_cast<NT_*>(Yhat),    \
                                              nf, nt, ntasks, nobs, group, workspace, workspace_bytes,               \
                                              reinterpret_cast<cudaStream_t>(stream));                               \
        });                                                                                                          \
    }

GLMM_DEFINE(f32, float, float)
GLMM_DEFINE(f16, uint16_t, __half)
GLMM_DEFINE(bf16, uint16_t, __nv_bfloat16)

}  // extern "C"
