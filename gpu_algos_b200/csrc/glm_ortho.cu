// glm_ortho.cu -- Newton-Schulz orthogonalisation of model-shaped matrices.
//
// Per task, with X the matrix over its Frobenius norm and m <= n its sides:
//   X <- (aI + bA + cA^2) X,  A = X X^T,
// an odd polynomial of X's singular values.  Short matrices (m <= 32) run in
// double in one launch (glm_ortho_small.cu); the others take the norm and the
// split of X into binary16 planes here, then three tensor-core products a step
// (glm_ortho_gemm.cu).
#include <algorithm>
#include <cmath>

#include "glm_ortho.cuh"

namespace glmb {

namespace {

constexpr int kThreads = 256;

// part[task][block] = the block's share of |U|^2 in double; with a momentum, V <- mu V + G first.
// One read of G (and a read and a write of V): bound by HBM.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    ortho_norm_kernel(const T* __restrict__ G, float* __restrict__ V, double* __restrict__ part,
                      int* __restrict__ status, int* __restrict__ arrived, int narrived, int64_t size, OrthoUpdate up) {
    __shared__ double red[kThreads / 32];
    pdl_allow_dependents();
    if (blockIdx.x == 0 && blockIdx.y == 0) {
        if (threadIdx.x == 0) *status = 0;
        for (int i = threadIdx.x; i < narrived; i += kThreads) arrived[i] = 0;
    }
    const int64_t base = int64_t(blockIdx.y) * size;
    const int64_t stride = int64_t(gridDim.x) * kThreads;
    double s = 0.0;
    int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
    auto one = [&](float g, float v, int64_t e) {
        float u = g;
        if (V != nullptr) {
            v = fmaf(up.mu, v, g);
            V[e] = v;
            u = up.nesterov ? fmaf(up.mu, v, g) : v;
        }
        s = fma(double(u), double(u), s);
    };
    constexpr int kAhead = 8;
    for (; i + (kAhead - 1) * stride < size; i += kAhead * stride) {
        float g[kAhead], v[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            g[j] = to_arith<float>(G[base + i + j * stride]);
            v[j] = V != nullptr ? V[base + i + j * stride] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) one(g[j], v[j], base + i + j * stride);
    }
    for (; i < size; i += stride)
        one(to_arith<float>(G[base + i]), V != nullptr ? V[base + i] : 0.0f, base + i);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int w = 0; w < kThreads / 32; ++w) t += red[w];
        part[int64_t(blockIdx.y) * gridDim.x + blockIdx.x] = t;
    }
}

// scale / |U| of a task from its blocks' shares, by the first warp; 0 for a zero matrix.
__device__ __forceinline__ double inverse_norm(const double* part, int nparts, double scale, double* shared) {
    if (threadIdx.x < 32) {
        double ss = 0.0;
        for (int i = threadIdx.x; i < nparts; i += 32) ss += part[i];
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
        if (threadIdx.x == 0) *shared = ss == 0.0 ? 0.0 : scale / sqrt(ss);
    }
    __syncthreads();
    return *shared;
}

// u * inv, in float unless inv leaves float's comfortable range (norms near its ends)
struct Scaled {
    double inv;
    float inv_f;
    bool wide;
    __device__ explicit Scaled(double v) : inv(v), inv_f(float(v)), wide(!(v == 0.0 || (v > 1e-30 && v < 1e30))) {}
    __device__ __forceinline__ float operator()(float u) const {
        return wide ? float(double(u) * inv) : u * inv_f;
    }
};

__device__ __forceinline__ void put_split2(__half* dst, int64_t plane, float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    *reinterpret_cast<__half2*>(dst) = h;
    *reinterpret_cast<__half2*>(dst + plane) = __floats2half2_rn(a - f.x, b - f.y);
}

// X = scale * U / |U| into its planes, for matrices at least as wide as tall: two neighbouring columns to a
// thread, four rows at a time.  Columns that fill up a row to ld are zero.  Bound by HBM.
// V and part are not __restrict__: this kernel starts while the one that writes them still runs, so their loads
// (after the wait) may not take the read-only path.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    ortho_split_kernel(const T* __restrict__ G, const float* V, const double* part, int nparts, __half* __restrict__ X,
                       int64_t m, int64_t n, int64_t ld, float scale, OrthoUpdate up) {
    __shared__ double shared;
    pdl_allow_dependents();
    pdl_wait_for_producer();
    const int64_t task = blockIdx.z, base = task * m * n;
    const Scaled scaled(inverse_norm(part + task * nparts, nparts, scale, &shared));
    constexpr int kRows = 4;
    const int64_t tiles_n = (ld / 2 + kThreads - 1) / kThreads, tiles = tiles_n * ((m + kRows - 1) / kRows);
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int64_t i0 = tile / tiles_n * kRows, j = (tile % tiles_n * kThreads + threadIdx.x) * 2;
        if (j >= ld) continue;
        float u[kRows][2];
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k)
                u[i][k] = i0 + i < m && j + k < n ? ortho_direction(G, V, base + (i0 + i) * n + j + k, up) : 0.0f;
#pragma unroll
        for (int i = 0; i < kRows; ++i)
            if (i0 + i < m)
                put_split2(X + (task * 2 * m + i0 + i) * ld + j, m * ld, scaled(u[i][0]), scaled(u[i][1]));
    }
}

// The same of matrices taller than wide, transposed through 64 x 64 tiles.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    ortho_split_tall_kernel(const T* __restrict__ G, const float* V, const double* part, int nparts,
                            __half* __restrict__ X, int64_t m, int64_t n, int64_t ld, float scale,
                            OrthoUpdate up) {
    __shared__ float t[64][65];
    __shared__ double shared;
    pdl_allow_dependents();
    pdl_wait_for_producer();
    const int64_t task = blockIdx.z, base = task * m * n;
    const Scaled scaled(inverse_norm(part + task * nparts, nparts, scale, &shared));
    const int64_t tiles_n = (n + 63) / 64, tiles = tiles_n * ((m + 63) / 64);
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int64_t i0 = tile / tiles_n * 64, j0 = tile % tiles_n * 64;
#pragma unroll 8
        for (int e = threadIdx.x; e < 64 * 64; e += kThreads) {
            // neighbouring threads on neighbouring elements of the matrix as it lies in memory
            const int i = e & 63, j = e >> 6;
            t[i][j] = i0 + i < m && j0 + j < n ? scaled(ortho_direction(G, V, base + (j0 + j) * m + i0 + i, up)) : 0.0f;
        }
        __syncthreads();
#pragma unroll 4
        for (int e = threadIdx.x; e < 64 * 32; e += kThreads) {
            const int i = e >> 5, j = 2 * (e & 31);
            if (i0 + i < m && j0 + j < ld) put_split2(X + (task * 2 * m + i0 + i) * ld + j0 + j, m * ld, t[i][j], t[i][j + 1]);
        }
        __syncthreads();
    }
}

// Blocks a task's norm is shared by: enough for the memory system (eight to each of a B200's 148 SMs over all
// tasks), 4096 elements each at the least.  The number sets the workspace's layout, so it depends on the sizes
// alone and not on the device that is current when a caller asks.
constexpr int64_t kNormBlocks = 8 * 148;
int64_t norm_blocks(int64_t size, int64_t ntasks) {
    const int64_t most = std::max<int64_t>(1, kNormBlocks / std::max<int64_t>(1, ntasks));
    return std::max<int64_t>(1, std::min(most, (size + 4095) / 4096));
}

int64_t padded(int64_t cols) { return (cols + 7) / 8 * 8; }

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
    if (m <= kOrthoSmallRows) return 0;
    return 256 + round_up(ortho_partial_bytes(m, n, ntasks), 256) + round_up(ortho_arrived_bytes(), 256) + round_up(size_t(ntasks) * norm_blocks(m * n, ntasks) * 8, 256) +
           2 * round_up(size_t(ntasks) * m * padded(n) * 4, 256) + 3 * round_up(size_t(ntasks) * m * padded(m) * 4, 256);
}

template <typename T>
int ortho_run(const T* G, float* V, T* out, int64_t nf, int64_t nt, int64_t ntasks, const OrthoSteps& steps,
              const OrthoUpdate* update, void* ws, size_t ws_bytes, cudaStream_t stream) {
    const int64_t m = std::min(nf, nt), n = std::max(nf, nt), size = m * n;
    const bool tall = nt > nf;
    if (m <= kOrthoSmallRows) {
        set_last_path("ortho_small");
        return ortho_small<T>(G, V, out, m, n, tall, ntasks, steps, update, stream);
    }
    if (ntasks > 65535 || n > (int64_t(1) << 30)) return GLMB_ERR_TOO_LARGE;
    Scratch sc(ws, ws_bytes, ortho_workspace<T>(nf, nt, ntasks), stream);
    if (sc.status() != GLMB_OK) return sc.status();
    char* w = sc.template as<char>();
    auto take = [&](size_t bytes) {
        char* p = w;
        w += round_up(bytes, 256);
        return p;
    };
    OrthoPlanes p{m, n, padded(m), padded(n), ntasks, {}, nullptr, nullptr, nullptr, nullptr, nullptr};
    int* status = reinterpret_cast<int*>(take(4));
    const int64_t nb = norm_blocks(size, ntasks);
    double* part = reinterpret_cast<double*>(take(size_t(ntasks) * nb * 8));
    p.partial = reinterpret_cast<float4*>(take(ortho_partial_bytes(m, n, ntasks)));
    p.arrived = reinterpret_cast<int*>(take(ortho_arrived_bytes()));
    for (__half*& x : p.X) x = reinterpret_cast<__half*>(take(size_t(ntasks) * m * p.ld_n * 4));
    p.A = reinterpret_cast<__half*>(take(size_t(ntasks) * m * p.ld_m * 4));
    p.B = reinterpret_cast<__half*>(take(size_t(ntasks) * m * p.ld_m * 4));
    p.C = reinterpret_cast<__half*>(take(size_t(ntasks) * m * p.ld_m * 4));
    const OrthoUpdate up = update != nullptr ? *update : OrthoUpdate{};
    set_last_path("ortho_tensor");
    ortho_norm_kernel<T><<<dim3(unsigned(nb), unsigned(ntasks)), kThreads, 0, stream>>>(
        G, V, part, status, p.arrived, int(ortho_arrived_bytes() / sizeof(int)), size, up);
    count_launch();
    int st = launch_status();
    if (st != GLMB_OK) return st;
    const int64_t tiles = tall ? (n + 63) / 64 * ((m + 63) / 64)
                               : (p.ld_n / 2 + kThreads - 1) / kThreads * ((m + 3) / 4);
    const int64_t most = std::max<int64_t>(1, 8 * int64_t(sm_count()) / ntasks);
    const cudaError_t e =
        pdl_launch(tall ? ortho_split_tall_kernel<T> : ortho_split_kernel<T>,
                   dim3(unsigned(std::min(tiles, most)), 1, unsigned(ntasks)), dim3(kThreads), 0, stream, G,
                   static_cast<const float*>(V), static_cast<const double*>(part), int(nb), p.X[0], m, n, p.ld_n,
                   ortho_x_scale(steps.step[0]), up);
    count_launch();
    if (e != cudaSuccess) return int(e);
    return ortho_products<T>(p, steps, out, tall, update, status, stream);
}

#define GLMB_INSTANTIATE_ORTHO(T)                                                                                \
    template size_t ortho_workspace<T>(int64_t, int64_t, int64_t);                                               \
    template int ortho_run<T>(const T*, float*, T*, int64_t, int64_t, int64_t, const OrthoSteps&,                \
                              const OrthoUpdate*, void*, size_t, cudaStream_t);

GLMB_INSTANTIATE_ORTHO(float)
GLMB_INSTANTIATE_ORTHO(__half)
GLMB_INSTANTIATE_ORTHO(__nv_bfloat16)

}  // namespace glmb
