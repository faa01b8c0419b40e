/*
 * glm_matrix_b200.h -- C ABI of libglm_b200.so for whole-matrix operators on
 * models: orthogonalised updates (for training a model with many targets) and
 * the 4-bit form of a model with the prediction that reads it (for serving).
 *
 * The conventions are those of glm_b200.h: Tensor3D layout (X (nfeatures,
 * ntasks, nobs), M (nfeatures, ntargets, ntasks), the first index fastest),
 * device pointers, asynchronous launches on `stream` of the current device,
 * GLMB_* status codes, no C++ exception across the boundary, `workspace`
 * (256-byte aligned) of at least the size the matching *_workspace_size
 * function reports or NULL for a stream-ordered allocation.  Outputs overlap
 * no input unless an entry point says so (GLMB_ERR_INVALID_VALUE).  A workspace holds nothing between calls,
 * but two calls that may overlap on the GPU (other streams, captured graphs
 * that are replayed side by side) need one each.  The reference has no
 * counterpart of these operators.
 *
 * Types: f32, f16 (__half bits) and bf16 (bfloat16 bits).
 */
#ifndef GLM_MATRIX_B200_H
#define GLM_MATRIX_B200_H

#include "glm_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------
 * Orthogonalisation by Newton-Schulz steps.  For every task, with X the
 * task's ntargets x nfeatures matrix of G divided by its Frobenius norm (a
 * zero matrix stays zero), `steps` times
 *   X <- a X + (b A + c A A) X,   A = X X^T   (on the shorter side)
 * with (a, b, c) = coefficients[3*k ..] of step k, a host array of 3*steps
 * doubles that is read during the call; NULL stands for (3.4445, -4.7750,
 * 2.0315) in every step, which brings the singular values of X near 1 in five
 * steps.  O may be G.  Sums are float or wider, whatever the type.  Where both
 * sides are longer than 32, iterates carry 22 significant bits down to 2^-17 of
 * the largest singular value that the coefficients let them have (1 at first;
 * counted as 1e-3 where it is less) and steps of 2^-38 of it below that: the
 * entries of a feature a million times smaller than the others keep a few bits
 * of their own.  Shorter matrices are worked on in double.  A NaN or infinity in
 * a task's G makes that task's O NaN.
 * GLMB_ERR_INVALID_VALUE also when steps is outside 1..GLMM_MAX_STEPS, or
 * when the coefficients are not finite or let a singular value of X grow past
 * 16 (or |a + b s^2 + c s^4| past 1024).  GLMB_ERR_TOO_LARGE for more than
 * 65535 tasks whose matrices have over 32 rows and columns, or a side past 2^30
 * of such a matrix.
 * ---------------------------------------------------------------------- */
#define GLMM_MAX_STEPS 16

/* Update of a model by its orthogonalised momentum:
 *   V <- mu V + grad          (V: float, the model's shape)
 *   U  = grad + mu V with GLMM_STEP_NESTEROV, V otherwise
 *   M <- (1 - lr*weight_decay) M - lr*scale * O(U)
 * with O the orthogonalisation above.  M, grad and V are distinct arrays.
 * GLMB_ERR_INVALID_VALUE also when mu, 1 - lr*weight_decay or lr*scale is not
 * finite as a float. */
#define GLMM_STEP_NESTEROV 0x1u

/* The workspace serves both entry points. */
#define GLMM_DECLARE_ORTHO(SFX, T)                                                      \
    size_t glmm_orthogonal_workspace_size_##SFX(int64_t nfeatures, int64_t ntargets,    \
                                                int64_t ntasks);                        \
    int glmm_orthogonalize_##SFX(const T* G, T* O, int64_t nfeatures, int64_t ntargets, \
                                 int64_t ntasks, const double* coefficients, int steps, \
                                 void* workspace, size_t workspace_bytes,               \
                                 glmb_stream_t stream);                                 \
    int glmm_orthogonal_step_##SFX(T* M, const T* grad, float* momentum,                \
                                   int64_t nfeatures, int64_t ntargets, int64_t ntasks, \
                                   double lr, double mu, double weight_decay,           \
                                   double scale, uint32_t flags,                        \
                                   const double* coefficients, int steps,               \
                                   void* workspace, size_t workspace_bytes,             \
                                   glmb_stream_t stream);

GLMM_DECLARE_ORTHO(f32, float)
GLMM_DECLARE_ORTHO(f16, uint16_t)
GLMM_DECLARE_ORTHO(bf16, uint16_t)

/* ------------------------------------------------------------------------
 * Models in 4 bits.  Each target's features are taken in groups of `group`
 * (64 or 128; the last one may be short).  A group has a scale
 *   s = max|w| / 7   rounded to the model's type
 * and every weight a code q = w / s rounded to the nearest whole number (ties
 * to even), held within -7..7; the weight stands for q*s exactly.  A group of
 * zeros has s = 0; a group with a NaN or an infinity has s = NaN.
 *
 * `codes` (glmm_q4_codes_bytes bytes, 16-byte aligned) and `scales`
 * (glmm_q4_scales_count elements) are laid out for the kernels that read
 * them:
 *   codes  [task][target/16][feature/64][lane 0..31][word 0..3] (32-bit words):
 *          a 16 x 64 block of codes in the order in which the lanes of a warp
 *          feed them to the tensor core.  Word s of lane 4g + c holds features
 *          f = 16s + 4c .. f + 3 of targets g and g + 8, each code as q + 8 in
 *          four bits; from bit 0 up: (g, f), (g+8, f), (g, f+2), (g+8, f+2),
 *          and from bit 16 up the same of f + 1 and f + 3;
 *   scales [task][target/16][group][target%8][target/8%2].
 * Targets are filled up to a multiple of 16 and features to one of 128; what
 * fills up has code 0, and groups of nothing else s = 0.
 * ---------------------------------------------------------------------- */
int64_t glmm_q4_codes_bytes(int64_t nfeatures, int64_t ntargets, int64_t ntasks);
int64_t glmm_q4_scales_count(int64_t nfeatures, int64_t ntargets, int64_t ntasks, int group);

/* quantize: codes and scales of M.  dequantize: M = q*s, rounded to the type.
 * predict: Yhat[t, task, obs] = sum_f q[f, t, task]*s * X[f, task, obs], sums
 * in float, one rounding to the type.  A group's sum of q*X is formed before it
 * is multiplied by s, 2^-10 of it, so that no finite X takes it past float's
 * range.  Bits of a float X below 2^-133 are lost, and a float or bfloat16
 * result below 2^-116 is summed in steps of 2^-139. */
#define GLMM_DECLARE_Q4(SFX, T)                                                         \
    int glmm_quantize_q4_##SFX(const T* M, void* codes, T* scales, int64_t nfeatures,   \
                               int64_t ntargets, int64_t ntasks, int group,             \
                               glmb_stream_t stream);                                   \
    int glmm_dequantize_q4_##SFX(const void* codes, const T* scales, T* M,              \
                                 int64_t nfeatures, int64_t ntargets, int64_t ntasks,   \
                                 int group, glmb_stream_t stream);                      \
    size_t glmm_predict_q4_workspace_size_##SFX(int64_t nfeatures, int64_t ntargets,    \
                                                int64_t ntasks, int64_t nobs,           \
                                                int group);                             \
    int glmm_predict_q4_##SFX(const T* X, const void* codes, const T* scales, T* Yhat,  \
                              int64_t nfeatures, int64_t ntargets, int64_t ntasks,      \
                              int64_t nobs, int group, void* workspace,                 \
                              size_t workspace_bytes, glmb_stream_t stream);

GLMM_DECLARE_Q4(f32, float)
GLMM_DECLARE_Q4(f16, uint16_t)
GLMM_DECLARE_Q4(bf16, uint16_t)

#ifdef __cplusplus
}
#endif
#endif /* GLM_MATRIX_B200_H */
