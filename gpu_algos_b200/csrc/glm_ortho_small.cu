// glm_ortho_small.cu -- Newton-Schulz steps of short matrices (m <= 32 rows) in
// one launch.
//
// With so few rows the steps need not touch X between the first product and
// the last: X_k = P_k X_0 with P_k and A_k = X_k X_k^T polynomials of A_0, so
//   Q = aI + bA + cA^2,   P <- Q P,   A <- Q A Q
// run on m x m matrices alone.  That form forms small singular values from
// differences of squares, which float cannot carry (a value of 1e-3 beside 1
// would drown), so everything here is double -- whose products the FP64
// tensor pipe (mma.m8n8k4) makes at this size as fast as the launch itself.
// The squared norm is A_0's trace, so X is read once.
//
// A cluster of up to eight CTAs works on one task's matrix: each holds a
// slice of columns in shared memory, forms its share of the first product,
// sums the shares of all in rank order over distributed shared memory, runs
// the m x m chain (every CTA its own copy) and multiplies its slice by P.
//
// 64 tasks of 16 x 256 in float: about 6 us on the GPU (8.5 us a call from
// Python), 162 us as three product kernels a step; bound by the chain's 14
// dependent products of a few hundred clocks and the cluster's two meetings.
// m <= 32: beyond, the chain (17 products of m^3 in double on one SM) would take
// longer than the tensor cores' launches.
#include <algorithm>

#include "glm_ortho.cuh"
#include "glm_tc.cuh"

namespace glmb {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kChunk = 128;          // columns of X staged together
constexpr int kChunkLd = kChunk + 4;  // floats; four banks on from row to row
constexpr int kHeld = 8;             // chunks of a slice kept between the products

// d += a b on 8 x 8 tiles: lane l gives a(l/4, l%4) and b(l%4, l/4), holds d(l/4, 2(l%4) + {0, 1})
__device__ __forceinline__ void mma_f64(double (&d)[2], double a, double b) {
    asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0,%1}, {%2}, {%3}, {%0,%1};"
                 : "+d"(d[0]), "+d"(d[1])
                 : "d"(a), "d"(b));
}

template <int MT>
struct SmallSmem {
    static constexpr int kM = 8 * MT, kLd = kM + 4;
    double share[kM][kLd];            // this CTA's share of X X^T, read by its peers
    double part[kWarps][kM][kLd];     // warps' shares, then the chain's matrices
    double inv;
};

// D = L R for symmetric R (and so rows of R are its columns), tiles first, first + kWarps, ... to this warp.
template <int MT, typename F>
__device__ __forceinline__ void multiply(const double (*L)[8 * MT + 4], const double (*R)[8 * MT + 4], int first, F&& put) {
    const int lane = threadIdx.x & 31, row = lane >> 2, k = lane & 3;
    for (int t = first; t < MT * MT; t += kWarps) {
        const int ti = t / MT, tj = t % MT;
        double d[2] = {0.0, 0.0}, e[2] = {0.0, 0.0};
#pragma unroll
        for (int s = 0; s < 2 * MT; s += 2) {
            mma_f64(d, L[8 * ti + row][4 * s + k], R[8 * tj + row][4 * s + k]);
            mma_f64(e, L[8 * ti + row][4 * s + 4 + k], R[8 * tj + row][4 * s + 4 + k]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) put(8 * ti + row, 8 * tj + 2 * k + j, d[j] + e[j]);
    }
}

template <typename T, int MT>
__global__ void __launch_bounds__(kThreads)
    ortho_small_kernel(const T* G, float* V, T* out, int m, int64_t n, bool tall, int64_t slice, bool held,
                       const OrthoSteps steps, bool update, OrthoUpdate up) {
    using Smem = SmallSmem<MT>;
    constexpr int kM = Smem::kM;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    float* us = reinterpret_cast<float*>(smem_raw + sizeof(Smem));  // chunks of [kM][kChunkLd]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row = lane >> 2, kk = lane & 3;
    const uint32_t rank = blockIdx.x;  // gridDim.x CTAs are one cluster
    const int64_t base = int64_t(blockIdx.y) * m * n;
    const int64_t j0 = min(n, int64_t(rank) * slice), j1 = min(n, j0 + slice);

    // Stages U's columns [c0, c0 + kChunk) (zero past j1 and past m); `first`: the momentum is updated on the way.
    auto stage = [&](float* dst, int64_t c0, bool first) {
        const int cols = int(min(int64_t(kChunk), j1 - c0));
        const int total = m * cols;
        if (cols < kChunk || m < kM) {
            for (int i = tid; i < kM * kChunk; i += kThreads) {
                const int r = i / kChunk, c = i % kChunk;
                if (r >= m || c >= cols) dst[r * kChunkLd + c] = 0.0f;
            }
        }
#pragma unroll 8
        for (int i = tid; i < total; i += kThreads) {
            // neighbouring threads on neighbouring elements of the matrix as it lies in memory
            const int r = tall ? i % m : i / cols, c = tall ? i / m : i % cols;
            const int64_t e = base + (tall ? c0 * m + i : r * n + c0 + c);
            if (first && V != nullptr) {
                const float g = to_arith<float>(G[e]), v = fmaf(up.mu, V[e], g);
                V[e] = v;
                dst[r * kChunkLd + c] = up.nesterov ? fmaf(up.mu, v, g) : v;
            } else {
                dst[r * kChunkLd + c] = ortho_direction(G, V, e, up);
            }
        }
    };

    // ---- this CTA's share of U U^T: tiles on and above the diagonal, K shared over the warps ----
    double acc[MT * (MT + 1) / 2][2] = {};
    auto gram = [&](const float* src) {
        for (int s = warp; s < kChunk / 4; s += kWarps) {
            double f[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) f[t] = double(src[(8 * t + row) * kChunkLd + 4 * s + kk]);
#pragma unroll
            for (int tj = 0; tj < MT; ++tj)
#pragma unroll
                for (int ti = 0; ti <= tj; ++ti) mma_f64(acc[tj * (tj + 1) / 2 + ti], f[ti], f[tj]);
        }
    };
    if (held) {
        int b = 0;
        for (int64_t c0 = j0; c0 < j1; c0 += kChunk, ++b) stage(us + b * kM * kChunkLd, c0, true);
        __syncthreads();
        b = 0;
        for (int64_t c0 = j0; c0 < j1; c0 += kChunk, ++b) gram(us + b * kM * kChunkLd);
    } else {
        for (int64_t c0 = j0; c0 < j1; c0 += kChunk) {
            stage(us, c0, true);
            __syncthreads();
            gram(us);
            __syncthreads();
        }
    }
#pragma unroll
    for (int tj = 0; tj < MT; ++tj)
#pragma unroll
        for (int ti = 0; ti <= tj; ++ti)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                sm.part[warp][8 * ti + row][8 * tj + 2 * kk + j] = acc[tj * (tj + 1) / 2 + ti][j];
    __syncthreads();
    for (int i = tid; i < kM * kM; i += kThreads) {
        const int r = i / kM, c = i % kM;
        const bool upper = r / 8 <= c / 8;
        double s = 0.0;
        for (int w = 0; w < kWarps; ++w) s += upper ? sm.part[w][r][c] : sm.part[w][c][r];
        sm.share[r][c] = s;
    }
    __syncthreads();
    cluster_sync();
    double(*A)[Smem::kLd] = sm.part[0], (*Q)[Smem::kLd] = sm.part[1], (*S)[Smem::kLd] = sm.part[2];
    double(*Pa)[Smem::kLd] = sm.part[3], (*Pb)[Smem::kLd] = sm.part[4];
    for (int i = tid; i < kM * kM; i += kThreads) {
        const int r = i / kM, c = i % kM;
        double s = 0.0;
        for (uint32_t p = 0; p < gridDim.x; ++p) s += ld_cluster_f64(&sm.share[r][c], p);
        A[r][c] = s;
    }
    __syncthreads();
    cluster_sync();  // the peers have read this CTA's share
    double ss = 0.0;
    for (int r = 0; r < m; ++r) ss += A[r][r];
    const double inv2 = ss == 0.0 ? 0.0 : 1.0 / ss;
    __syncthreads();
    for (int i = tid; i < kM * kM; i += kThreads) A[i / kM][i % kM] *= inv2;
    __syncthreads();

    // ---- the m x m chain ----
    for (int k = 0; k < steps.n; ++k) {
        const double a = steps.step[k].a, b = steps.step[k].b, c = steps.step[k].c;
        multiply<MT>(A, A, warp, [&](int r, int cc, double v) {
            const double q = fma(c, v, b * A[r][cc]) + (r == cc ? a : 0.0);
            Q[r][cc] = q;
            if (k == 0) Pa[r][cc] = q;
        });
        __syncthreads();
        const bool last = k + 1 == steps.n;
        if (k > 0) multiply<MT>(Q, Pa, warp, [&](int r, int cc, double v) { Pb[r][cc] = v; });
        if (!last) multiply<MT>(A, Q, (warp + kWarps / 2) % kWarps, [&](int r, int cc, double v) { S[r][cc] = v; });
        __syncthreads();
        if (k > 0) {
            double(*t)[Smem::kLd] = Pa;
            Pa = Pb;
            Pb = t;
        }
        if (!last) {
            multiply<MT>(S, Q, warp, [&](int r, int cc, double v) { A[r][cc] = v; });
            __syncthreads();
        }
    }

    // ---- out = P U / |U| ----
    const double inv = ss == 0.0 ? 0.0 : 1.0 / sqrt(ss);
    double p[MT][2 * MT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int s = 0; s < 2 * MT; ++s) p[t][s] = Pa[8 * t + row][4 * s + kk] * inv;
    int b = 0;
    for (int64_t c0 = j0; c0 < j1; c0 += kChunk, ++b) {
        const float* src = us + (held ? b * kM * kChunkLd : 0);
        if (!held) {
            stage(us, c0, false);
            __syncthreads();
        }
        for (int cb = 8 * warp; cb < kChunk; cb += 8 * kWarps) {
            if (c0 + cb >= j1) break;
            double d[MT][2] = {};
#pragma unroll
            for (int s = 0; s < 2 * MT; ++s) {
                const double x = double(src[(4 * s + kk) * kChunkLd + cb + row]);
#pragma unroll
                for (int t = 0; t < MT; ++t) mma_f64(d[t], p[t][s], x);
            }
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int r = 8 * t + row;
                    const int64_t col = c0 + cb + 2 * kk + j;
                    if (r >= m || col >= j1) continue;
                    const int64_t e = base + (tall ? col * m + r : r * n + col);
                    float v = float(d[t][j]);
                    if (update) v = fmaf(-up.rate, v, up.keep * to_arith<float>(out[e]));
                    out[e] = from_arith<T>(v);
                }
        }
        if (!held) __syncthreads();
    }
}

template <typename T, int MT>
cudaError_t launch_small(const T* G, float* V, T* out, int64_t m, int64_t n, bool tall, int64_t ntasks,
                         const OrthoSteps& steps, const OrthoUpdate* update, cudaStream_t stream) {
    const int64_t chunks = (n + kChunk - 1) / kChunk;
    // CTAs to a task: as many as there are chunks, up to eight, while tasks alone leave SMs idle
    int cluster = 1;
    while (cluster < 8 && 2 * cluster <= chunks && 2 * cluster * ntasks <= 2 * int64_t(sm_count())) cluster *= 2;
    const int64_t per = (chunks + cluster - 1) / cluster;
    const bool held = per <= kHeld;
    const size_t chunk_bytes = size_t(8 * MT) * kChunkLd * 4;
    const size_t most = sizeof(SmallSmem<MT>) + kHeld * chunk_bytes;
    const size_t smem = sizeof(SmallSmem<MT>) + size_t(held ? per : 1) * chunk_bytes;
    static std::atomic<uint64_t> attr{0};
    auto kernel = ortho_small_kernel<T, MT>;
    cudaError_t e = set_smem_limit_once(attr, kernel, most);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(cluster), unsigned(ntasks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = unsigned(cluster);
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    count_launch();
    return cudaLaunchKernelEx(&cfg, kernel, G, V, out, int(m), n, tall, per * kChunk, held, steps, update != nullptr,
                              update != nullptr ? *update : OrthoUpdate{});
}

}  // namespace

template <typename T>
int ortho_small(const T* G, float* V, T* out, int64_t m, int64_t n, bool tall, int64_t ntasks, const OrthoSteps& steps,
                const OrthoUpdate* up, cudaStream_t stream) {
    // gridDim.y carries the tasks of one launch
    constexpr int64_t kMost = 65535;
    for (int64_t t = 0; t < ntasks; t += kMost) {
        const int64_t now = std::min(kMost, ntasks - t), at = t * m * n;
        float* v = V != nullptr ? V + at : nullptr;
        cudaError_t e;
        if (m <= 8) e = launch_small<T, 1>(G + at, v, out + at, m, n, tall, now, steps, up, stream);
        else if (m <= 16) e = launch_small<T, 2>(G + at, v, out + at, m, n, tall, now, steps, up, stream);
        else e = launch_small<T, 4>(G + at, v, out + at, m, n, tall, now, steps, up, stream);
        if (e != cudaSuccess) return int(e);
    }
    return launch_status();
}

template int ortho_small<float>(const float*, float*, float*, int64_t, int64_t, bool, int64_t, const OrthoSteps&,
                                const OrthoUpdate*, cudaStream_t);
template int ortho_small<__half>(const __half*, float*, __half*, int64_t, int64_t, bool, int64_t, const OrthoSteps&,
                                 const OrthoUpdate*, cudaStream_t);
template int ortho_small<__nv_bfloat16>(const __nv_bfloat16*, float*, __nv_bfloat16*, int64_t, int64_t, bool, int64_t,
                                        const OrthoSteps&, const OrthoUpdate*, cudaStream_t);

}  // namespace glmb
