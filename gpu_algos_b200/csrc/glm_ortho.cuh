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

template <typename T>
size_t ortho_workspace(int64_t nf, int64_t nt, int64_t ntasks);
// out = O(G); with `up`, G is the gradient, V the momentum and out the model.  out may be G (up == nullptr).
template <typename T>
int ortho_run(const T* G, float* V, T* out, int64_t nf, int64_t nt, int64_t ntasks, const OrthoSteps& steps,
              const OrthoUpdate* up, void* ws, size_t ws_bytes, cudaStream_t stream);

}  // namespace glmb
