// glm_ortho.cu -- Newton-Schulz orthogonalisation of model-shaped matrices.
//
// Per task, with X the matrix over its Frobenius norm and m <= n its sides:
//   X <- (aI + bA + cA^2) X,  A = X X^T,
// an odd polynomial of X's singular values.  Three products a step:
//   A = X X^T,  B = aI + bA + cA A,  X' = B X.
#include <algorithm>
#include <cmath>

#include "glm_ortho.cuh"

namespace glmb {

namespace {

constexpr int kThreads = 256;
constexpr int kNormBlocks = 64;  // partial sums of a task's squared norm

__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < int(blockDim.x >> 5); ++w) s += red[w];
    __syncthreads();
    return s;
}

// The matrix to orthogonalise at element e: G itself, or the momentum's direction.
template <typename T>
__device__ __forceinline__ float direction(const T* G, const float* V, int64_t e, const OrthoUpdate& up) {
    const float g = to_arith<float>(G[e]);
    if (V == nullptr) return g;
    return up.nesterov ? fmaf(up.mu, V[e], g) : V[e];
}

// part[task][block] = the block's share of |U|^2 in double; with a momentum, V <- mu V + G first.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    ortho_norm_kernel(const T* __restrict__ G, float* __restrict__ V, double* __restrict__ part, int64_t size,
                      OrthoUpdate up) {
    __shared__ double red[kThreads / 32];
    const int64_t base = int64_t(blockIdx.y) * size;
    double s = 0.0;
    for (int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x; i < size; i += int64_t(gridDim.x) * kThreads) {
        if (V != nullptr) V[base + i] = fmaf(up.mu, V[base + i], to_arith<float>(G[base + i]));
        const double u = double(direction(G, V, base + i, up));
        s += u * u;
    }
    s = block_sum(s, red);
    if (threadIdx.x == 0) part[int64_t(blockIdx.y) * gridDim.x + blockIdx.x] = s;
}

// X[task][i][j] = U / |U|, transposed when the matrix is taller than wide.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    ortho_init_kernel(const T* __restrict__ G, const float* __restrict__ V, const double* __restrict__ part,
                      float* __restrict__ X, int64_t m, int64_t n, bool tall, OrthoUpdate up) {
    double ss = 0.0;
    for (int i = 0; i < kNormBlocks; ++i) ss += part[int64_t(blockIdx.y) * kNormBlocks + i];
    const double inv = ss == 0.0 ? 0.0 : 1.0 / sqrt(ss);
    const int64_t size = m * n, base = int64_t(blockIdx.y) * size;
    for (int64_t e = int64_t(blockIdx.x) * kThreads + threadIdx.x; e < size; e += int64_t(gridDim.x) * kThreads) {
        const int64_t i = e / n, j = e % n;
        X[base + e] = float(double(direction(G, V, base + (tall ? j * m + i : e), up)) * inv);
    }
}

// D[rows x cols] = alpha * P Q (+ beta * C) (+ gamma on the diagonal), Q read as Q[c][k] when QT.
template <bool QT>
__global__ void __launch_bounds__(256)
    ortho_gemm_kernel(const float* __restrict__ P, const float* __restrict__ Q, const float* C, float* __restrict__ D,
                      int64_t rows, int64_t cols, int64_t K, int64_t p_task, int64_t q_task, int64_t d_task,
                      float alpha, float beta, float gamma) {
    __shared__ float sp[16][68], sq[16][68];
    const int64_t task = blockIdx.z, r0 = int64_t(blockIdx.y) * 64, c0 = int64_t(blockIdx.x) * 64;
    P += task * p_task;
    Q += task * q_task;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[4][4] = {};
    for (int64_t k0 = 0; k0 < K; k0 += 16) {
        for (int i = threadIdx.x; i < 1024; i += 256) {
            const int r = i >> 4, k = i & 15;
            sp[k][r] = r0 + r < rows && k0 + k < K ? P[(r0 + r) * K + k0 + k] : 0.0f;
            if (QT) sq[k][r] = c0 + r < cols && k0 + k < K ? Q[(c0 + r) * K + k0 + k] : 0.0f;
            const int c = i & 63, kk = i >> 6;
            if (!QT) sq[kk][c] = c0 + c < cols && k0 + kk < K ? Q[(k0 + kk) * cols + c0 + c] : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sp[k][ty * 4 + i], sq[k][tx * 4 + j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t r = r0 + ty * 4 + i, c = c0 + tx * 4 + j;
            if (r >= rows || c >= cols) continue;
            const int64_t e = task * d_task + r * cols + c;
            float v = alpha * acc[i][j];
            if (C != nullptr) v = fmaf(beta, C[e], v);
            if (r == c) v += gamma;
            D[e] = v;
        }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    ortho_store_kernel(const float* __restrict__ X, T* __restrict__ out, int64_t m, int64_t n, bool tall, bool update,
                       OrthoUpdate up) {
    const int64_t size = m * n, base = int64_t(blockIdx.y) * size;
    for (int64_t e = int64_t(blockIdx.x) * kThreads + threadIdx.x; e < size; e += int64_t(gridDim.x) * kThreads) {
        const int64_t o = base + (tall ? (e % n) * m + e / n : e);
        float v = X[base + e];
        if (update) v = fmaf(-up.rate, v, up.keep * to_arith<float>(out[o]));
        out[o] = from_arith<T>(v);
    }
}

}  // namespace

int ortho_plan_steps(const double* coefficients, int steps, OrthoSteps* out) {
    static const double kDefault[3] = {3.4445, -4.7750, 2.0315};
    if (steps < 1 || steps > kOrthoMaxSteps) return GLMB_ERR_INVALID_VALUE;
    out->n = steps;
    double top = 1.0;  // singular values of X before the step lie in [0, top]
    for (int k = 0; k < steps; ++k) {
        const double* q = coefficients != nullptr ? coefficients + 3 * k : kDefault;
        const double a = q[0], b = q[1], c = q[2];
        if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return GLMB_ERR_INVALID_VALUE;
        // |a + bs + cs^2| over s in [0, top^2]: at the ends or at s = -b/2c
        const double S = top * top;
        auto f = [&](double s) { return std::fabs(a + s * (b + s * c)); };
        double b_max = std::max(f(0.0), f(S));
        if (c != 0.0 && -b / (2.0 * c) > 0.0 && -b / (2.0 * c) < S) b_max = std::max(b_max, f(-b / (2.0 * c)));
        // |x f(x^2)| over x in [0, top]: at the end or where a + 3bs + 5cs^2 = 0
        double x_next = top * f(S);
        auto at = [&](double s) {
            if (s > 0.0 && s < S) x_next = std::max(x_next, std::sqrt(s) * f(s));
        };
        if (c != 0.0) {
            const double disc = 9.0 * b * b - 20.0 * a * c;
            if (disc >= 0.0) {
                at((-3.0 * b + std::sqrt(disc)) / (10.0 * c));
                at((-3.0 * b - std::sqrt(disc)) / (10.0 * c));
            }
        } else if (b != 0.0) {
            at(-a / (3.0 * b));
        }
        if (!(b_max <= 1024.0) || !(x_next <= 16.0)) return GLMB_ERR_INVALID_VALUE;
        out->step[k] = OrthoStep{float(a), float(b), float(c), top, b_max};
        // rounding may carry a singular value a little past the bound
        top = std::max(1e-3, x_next * 1.01);
    }
    return GLMB_OK;
}

template <typename T>
size_t ortho_workspace(int64_t nf, int64_t nt, int64_t ntasks) {
    const int64_t m = std::min(nf, nt), n = std::max(nf, nt);
    return round_up(size_t(ntasks) * kNormBlocks * 8, 256) +
           2 * round_up(size_t(ntasks) * m * n * 4, 256) + 2 * round_up(size_t(ntasks) * m * m * 4, 256);
}

template <typename T>
int ortho_run(const T* G, float* V, T* out, int64_t nf, int64_t nt, int64_t ntasks, const OrthoSteps& steps,
              const OrthoUpdate* update, void* ws, size_t ws_bytes, cudaStream_t stream) {
    const int64_t m = std::min(nf, nt), n = std::max(nf, nt), size = m * n;
    const bool tall = nt > nf;
    if (ntasks > 65535) return GLMB_ERR_TOO_LARGE;
    Scratch sc(ws, ws_bytes, ortho_workspace<T>(nf, nt, ntasks), stream);
    if (sc.status() != GLMB_OK) return sc.status();
    char* w = sc.as<char>();
    auto take = [&](size_t bytes) {
        char* p = w;
        w += round_up(bytes, 256);
        return p;
    };
    double* part = reinterpret_cast<double*>(take(size_t(ntasks) * kNormBlocks * 8));
    float* X = reinterpret_cast<float*>(take(size_t(ntasks) * size * 4));
    float* X2 = reinterpret_cast<float*>(take(size_t(ntasks) * size * 4));
    float* A = reinterpret_cast<float*>(take(size_t(ntasks) * m * m * 4));
    float* B = reinterpret_cast<float*>(take(size_t(ntasks) * m * m * 4));
    const OrthoUpdate up = update != nullptr ? *update : OrthoUpdate{};
    const unsigned eb = unsigned(std::min<int64_t>(1024, (size + kThreads - 1) / kThreads));
    set_last_path("ortho");
    ortho_norm_kernel<T><<<dim3(kNormBlocks, unsigned(ntasks)), kThreads, 0, stream>>>(G, V, part, size, up);
    ortho_init_kernel<T><<<dim3(eb, unsigned(ntasks)), kThreads, 0, stream>>>(G, V, part, X, m, n, tall, up);
    const unsigned mt = unsigned((m + 63) / 64), ntl = unsigned((n + 63) / 64);
    for (int k = 0; k < steps.n; ++k) {
        const OrthoStep& s = steps.step[k];
        ortho_gemm_kernel<true><<<dim3(mt, mt, unsigned(ntasks)), 256, 0, stream>>>(X, X, nullptr, A, m, m, n, size, size,
                                                                                    m * m, 1.0f, 0.0f, 0.0f);
        ortho_gemm_kernel<true><<<dim3(mt, mt, unsigned(ntasks)), 256, 0, stream>>>(A, A, A, B, m, m, m, m * m, m * m,
                                                                                    m * m, s.c, s.b, s.a);
        ortho_gemm_kernel<false><<<dim3(ntl, mt, unsigned(ntasks)), 256, 0, stream>>>(B, X, nullptr, X2, m, n, m, m * m,
                                                                                      size, size, 1.0f, 0.0f, 0.0f);
        std::swap(X, X2);
    }
    ortho_store_kernel<T><<<dim3(eb, unsigned(ntasks)), kThreads, 0, stream>>>(X, out, m, n, tall, update != nullptr, up);
    count_launch(3 + 3 * steps.n);
    return launch_status();
}

#define GLMB_INSTANTIATE_ORTHO(T)                                                                                \
    template size_t ortho_workspace<T>(int64_t, int64_t, int64_t);                                               \
    template int ortho_run<T>(const T*, float*, T*, int64_t, int64_t, int64_t, const OrthoSteps&,                \
                              const OrthoUpdate*, void*, size_t, cudaStream_t);

GLMB_INSTANTIATE_ORTHO(float)
GLMB_INSTANTIATE_ORTHO(__half)
GLMB_INSTANTIATE_ORTHO(__nv_bfloat16)

}  // namespace glmb
