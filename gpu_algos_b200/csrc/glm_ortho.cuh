// glm_ortho.cuh -- Newton-Schulz orthogonalisation and the model update built on it (glm_ortho.cu).
#pragma once

#include "glm_common.cuh"

namespace glmb {

// What the steps may reach, from the coefficients alone (see ortho_plan_steps).
struct OrthoStep {
    float a, b, c;
    double x_max;  // largest singular value X may have before the step
    double b_max;  // largest |a + b s + c s^2| over the eigenvalues s of A the step may meet
};

constexpr int kOrthoMaxSteps = 16;

struct OrthoSteps {
    int n = 0;
    OrthoStep step[kOrthoMaxSteps];
};

// Fills `out` from 3*steps coefficients (nullptr: the default ones); GLMB_ERR_INVALID_VALUE as documented.
int ortho_plan_steps(const double* coefficients, int steps, OrthoSteps* out);

// The update of orthogonal_step: U = grad + nesterov*mu*V after V <- mu V + grad, M <- keep*M - rate*O(U).
struct OrthoUpdate {
    float mu;
    bool nesterov;
    float keep, rate;
};

// What orthogonalises when m (the shorter side) is large: binary16 planes [task][2: hi, lo][rows][ld].
struct OrthoPlanes {
    int64_t m, n, ld_m, ld_n, ntasks;
    __half* X[2];  // m x n, before and after a step in turn
    __half* A;     // m x m
    __half* B;
    __half* C;
    float4* partial;  // ortho_partial_bytes(): sums of tiles whose K two clusters share (nullptr for none)
    int* arrived;     // ortho_arrived_bytes(), zero
};
size_t ortho_partial_bytes(int64_t m, int64_t n, int64_t ntasks);
size_t ortho_arrived_bytes();
// The power of two that X's planes carry before a step.
float ortho_x_scale(const OrthoStep& s);
// All steps from X[0] (scaled by ortho_x_scale of the first) to `out` or, with `up`, the model's update;
// *status != 0 makes the outputs NaN (glm_ortho_gemm.cu).
template <typename T>
int ortho_products(const OrthoPlanes& p, const OrthoSteps& steps, T* out, bool tall, const OrthoUpdate* up, int* status,
                   cudaStream_t stream);

// m <= kOrthoSmallRows: one launch in double (glm_ortho_small.cu).
constexpr int64_t kOrthoSmallRows = 32;
template <typename T>
int ortho_small(const T* G, float* V, T* out, int64_t m, int64_t n, bool tall, int64_t ntasks, const OrthoSteps& steps,
                const OrthoUpdate* up, cudaStream_t stream);

// The matrix to orthogonalise at element e: G itself, or the (updated) momentum's direction.
template <typename T>
__device__ __forceinline__ float ortho_direction(const T* G, const float* V, int64_t e, const OrthoUpdate& up) {
    const float g = to_arith<float>(G[e]);
    if (V == nullptr) return g;
    return up.nesterov ? fmaf(up.mu, V[e], g) : V[e];
}

template <typename T>
size_t ortho_workspace(int64_t nf, int64_t nt, int64_t ntasks);
// out = O(G); with `up`, G is the gradient, V the momentum and out the model.  out may be G (up == nullptr).
template <typename T>
int ortho_run(const T* G, float* V, T* out, int64_t nf, int64_t nt, int64_t ntasks, const OrthoSteps& steps,
              const OrthoUpdate* up, void* ws, size_t ws_bytes, cudaStream_t stream);

}  // namespace glmb
