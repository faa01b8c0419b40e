// glm_q4.cu -- models in 4 bits with group scales: quantise, dequantise, predict.
//
// A weight stands for q*s with q a whole number of -7..7 and s the scale of
// its target's group of features; codes are kept as q + 8 in blocks of 16
// targets x 64 features whose 32 x 16 bytes are the operand registers of four
// 16 x 16 tensor-core fragments, one 16-byte load per lane (the layout is
// written out in glm_matrix_b200.h).
#include <algorithm>

#include "glm_q4.cuh"

namespace glmb {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / kWarp;

inline unsigned warp_grid(int64_t warps) {
    return unsigned(std::max<int64_t>(1, std::min<int64_t>(int64_t(sm_count()) * 32, (warps + kWarps - 1) / kWarps)));
}

// Sixteen consecutive features f0.. of one row (nullptr: a row past the last
// target) as floats, zero past nf.  `vec`: rows start on 16 bytes and nf is a
// whole number of 16-byte pieces, so a piece is inside or outside as a whole.
template <typename T>
__device__ __forceinline__ void load16(const T* row, int64_t f0, int64_t nf, bool vec, float (&v)[16]) {
    constexpr int kPer = 16 / sizeof(T);
    if (vec) {
#pragma unroll
        for (int i = 0; i < 16; i += kPer) {
            T t[kPer] = {};
            if (row != nullptr && f0 + i < nf) VecLoad<T, kPer>::load(row + f0 + i, t);
#pragma unroll
            for (int j = 0; j < kPer; ++j) v[i + j] = to_arith<float>(t[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = row != nullptr && f0 + i < nf ? to_arith<float>(row[f0 + i]) : 0.0f;
    }
}

// w / s rounded to the nearest whole number, ties to even, within -7..7, for
// |w| <= 7.5 s or so and s > 0.  The float product w * (1/s) can be off by an
// ulp and land on the wrong side of a border, so the remainder w - r*s decides:
// it is exact in float (w and r*s are multiples of ulp(s)/2 when r != 0 and
// the remainder is about s/2 at most).
__device__ __forceinline__ int nearest_code(float w, float s, float inv) {
    float r = fminf(fmaxf(rintf(w * inv), -7.0f), 7.0f);
    const float d = fmaf(-r, s, w), half = 0.5f * s;
    const bool odd = (int(r) & 1) != 0;
    if (fabsf(d) > half || (fabsf(d) == half && odd)) r += d > 0.0f ? 1.0f : -1.0f;
    return int(fminf(fmaxf(r, -7.0f), 7.0f));
}

// One warp per (task, 16 targets, group): lane 4g + c takes features 16c..16c+15
// of each 64-feature block of targets g and g + 8, so the group's largest
// magnitude is a maximum over the four lanes of a target.  One pass, bound by
// HBM: the weights in, codes and scales out.
template <typename T, int GROUP>
__global__ void __launch_bounds__(kThreads)
    q4_quantize_kernel(const T* __restrict__ M, uint4* __restrict__ codes, T* __restrict__ scales, int64_t nf,
                       int64_t nt, int64_t nrb, int64_t ncb, int64_t ngroups, int64_t total, bool vec) {
    constexpr int kBlocks = GROUP / kQ4Cols;
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    for (int64_t w = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5); w < total; w += int64_t(gridDim.x) * kWarps) {
        const int64_t group = w % ngroups, rb = w / ngroups % nrb, task = w / ngroups / nrb;
        float v[2][kBlocks][16];
        float s[2], inv[2], up[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t t = rb * kQ4Rows + g + 8 * h;
            const T* row = t < nt ? M + (task * nt + t) * nf : nullptr;
            float top = 0.0f;
            bool bad = false;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                load16(row, group * GROUP + b * kQ4Cols + 16 * c, nf, vec, v[h][b]);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    top = fmaxf(top, fabsf(v[h][b][i]));
                    bad |= !(fabsf(v[h][b][i]) <= 3.402823466e38f);
                }
            }
#pragma unroll
            for (int off = 1; off < 4; off <<= 1) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                bad |= __shfl_xor_sync(0xffffffffu, int(bad), off) != 0;
            }
            const T st = from_arith<T>(bad ? __int_as_float(0x7fc00000) : __fdiv_rn(top, 7.0f));
            if (c == 0) scales[((task * nrb + rb) * ngroups + group) * kQ4Rows + g + 8 * h] = st;
            const float sf = to_arith<float>(st);
            // scales near the bottom of float's range are lifted with their weights, which changes no ratio
            up[h] = sf < 0x1p-100f ? 0x1p60f : 1.0f;
            s[h] = bad ? 0.0f : sf * up[h];
            inv[h] = s[h] > 0.0f ? __frcp_rn(s[h]) : 0.0f;
        }
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            const int64_t cb = group * kBlocks + b;
            if (cb >= ncb) break;
            uint32_t word[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                word[k] = 0;
#pragma unroll
                for (int p = 0; p < 8; ++p) {
                    // p: pair 0..3 = (g, f), (g+8, f), (g, f+2), (g+8, f+2); 4..7 the same of f + 1
                    const int h = p & 1, i = 4 * k + (p & 2) + (p >> 2);
                    const int q = s[h] > 0.0f ? nearest_code(v[h][b][i] * up[h], s[h], inv[h]) : 0;
                    word[k] |= uint32_t(q + 8) << (4 * (p & 3) + 16 * (p >> 2));
                }
            }
            codes[((task * nrb + rb) * ncb + cb) * 32 + lane] = make_uint4(word[0], word[1], word[2], word[3]);
        }
    }
}

// The code (q) of pair p (0..3), first or second element, of a word.
__device__ __forceinline__ int code_of(uint32_t word, int p, int second) {
    return int((word >> (4 * p + 16 * second)) & 15u) - 8;
}

// One warp per block of codes: M = q*s (exact in float), rounded to T.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    q4_dequantize_kernel(const uint4* __restrict__ codes, const T* __restrict__ scales, T* __restrict__ M, int64_t nf,
                         int64_t nt, int64_t nrb, int64_t ncb, int64_t ngroups, int group, int64_t total, bool vec) {
    constexpr int kPer = 16 / sizeof(T);
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    for (int64_t w = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5); w < total; w += int64_t(gridDim.x) * kWarps) {
        const int64_t cb = w % ncb, rb = w / ncb % nrb, task = w / ncb / nrb;
        const uint4 block = codes[w * 32 + lane];
        const uint32_t word[4] = {block.x, block.y, block.z, block.w};
        const int64_t f0 = cb * kQ4Cols + 16 * c;
        const T* sc = scales + ((task * nrb + rb) * ngroups + cb * kQ4Cols / group) * kQ4Rows;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t t = rb * kQ4Rows + g + 8 * h;
            if (t >= nt) continue;
            const float s = to_arith<float>(sc[g + 8 * h]);
            T* row = M + (task * nt + t) * nf + f0;
            alignas(16) T out[16];
#pragma unroll
            for (int i = 0; i < 16; ++i)
                out[i] = from_arith<T>(float(code_of(word[i >> 2], (i & 2) + h, i & 1)) * s);
            if (vec) {
#pragma unroll
                for (int i = 0; i < 16; i += kPer)
                    if (f0 + i < nf) *reinterpret_cast<uint4*>(row + i) = *reinterpret_cast<const uint4*>(out + i);
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (f0 + i < nf) row[i] = out[i];
            }
        }
    }
}

// One warp per (task, 16 targets, observation).
template <typename T>
__global__ void __launch_bounds__(kThreads)
    q4_predict_kernel(const T* __restrict__ X, const uint4* __restrict__ codes, const T* __restrict__ scales,
                      T* __restrict__ Yhat, int64_t nf, int64_t nt, int64_t ntasks, int64_t nrb, int64_t ncb,
                      int64_t ngroups, int group, int64_t total, bool vec) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    for (int64_t w = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5); w < total; w += int64_t(gridDim.x) * kWarps) {
        const int64_t rb = w % nrb, task = w / nrb % ntasks, obs = w / nrb / ntasks;
        const T* x = X + (obs * ntasks + task) * nf;
        float acc[2] = {0.0f, 0.0f};
        for (int64_t cb = 0; cb < ncb; ++cb) {
            const uint4 block = codes[((task * nrb + rb) * ncb + cb) * 32 + lane];
            const uint32_t word[4] = {block.x, block.y, block.z, block.w};
            float v[16];
            load16(x, cb * kQ4Cols + 16 * c, nf, vec, v);
            const T* sc = scales + ((task * nrb + rb) * ngroups + cb * kQ4Cols / group) * kQ4Rows;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float d = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) d = fmaf(float(code_of(word[i >> 2], (i & 2) + h, i & 1)), v[i], d);
                acc[h] = fmaf(d, to_arith<float>(sc[g + 8 * h]), acc[h]);
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            acc[h] += __shfl_xor_sync(0xffffffffu, acc[h], 1);
            acc[h] += __shfl_xor_sync(0xffffffffu, acc[h], 2);
            const int64_t t = rb * kQ4Rows + g + 8 * h;
            if (c == 0 && t < nt) Yhat[(obs * ntasks + task) * nt + t] = from_arith<T>(acc[h]);
        }
    }
}

template <typename T>
bool whole_vectors(const T* p, int64_t nf) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && nf % int64_t(16 / sizeof(T)) == 0;
}

}  // namespace

template <typename T>
int q4_quantize(const T* M, void* codes, T* scales, int64_t nf, int64_t nt, int64_t ntasks, int group,
                cudaStream_t stream) {
    const int64_t nrb = q4_row_blocks(nt), ncb = q4_col_blocks(nf), ng = q4_groups(nf, group);
    const int64_t total = ntasks * nrb * ng;
    auto kernel = group == 64 ? q4_quantize_kernel<T, 64> : q4_quantize_kernel<T, 128>;
    kernel<<<warp_grid(total), kThreads, 0, stream>>>(M, static_cast<uint4*>(codes), scales, nf, nt, nrb, ncb, ng,
                                                      total, whole_vectors(M, nf));
    count_launch();
    return launch_status();
}

template <typename T>
int q4_dequantize(const void* codes, const T* scales, T* M, int64_t nf, int64_t nt, int64_t ntasks, int group,
                  cudaStream_t stream) {
    const int64_t nrb = q4_row_blocks(nt), ncb = q4_col_blocks(nf), ng = q4_groups(nf, group);
    const int64_t total = ntasks * nrb * ncb;
    q4_dequantize_kernel<T><<<warp_grid(total), kThreads, 0, stream>>>(
        static_cast<const uint4*>(codes), scales, M, nf, nt, nrb, ncb, ng, group, total, whole_vectors(M, nf));
    count_launch();
    return launch_status();
}

template <typename T>
size_t q4_predict_workspace(int64_t, int64_t, int64_t, int64_t, int) {
    return 0;
}

template <typename T>
int q4_predict(const T* X, const void* codes, const T* scales, T* Yhat, int64_t nf, int64_t nt, int64_t ntasks,
               int64_t nobs, int group, void*, size_t, cudaStream_t stream) {
    const int64_t nrb = q4_row_blocks(nt), ncb = q4_col_blocks(nf), ng = q4_groups(nf, group);
    const int64_t total = ntasks * nrb * nobs;
    q4_predict_kernel<T><<<warp_grid(total), kThreads, 0, stream>>>(X, static_cast<const uint4*>(codes), scales, Yhat,
                                                                    nf, nt, ntasks, nrb, ncb, ng, group, total,
                                                                    whole_vectors(X, nf));
    count_launch();
    return launch_status();
}

#define GLMB_INSTANTIATE_Q4(T)                                                                                \
    template int q4_quantize<T>(const T*, void*, T*, int64_t, int64_t, int64_t, int, cudaStream_t);          \
    template int q4_dequantize<T>(const void*, const T*, T*, int64_t, int64_t, int64_t, int, cudaStream_t);  \
    template size_t q4_predict_workspace<T>(int64_t, int64_t, int64_t, int64_t, int);                        \
    template int q4_predict<T>(const T*, const void*, const T*, T*, int64_t, int64_t, int64_t, int64_t, int, \
                               void*, size_t, cudaStream_t);

GLMB_INSTANTIATE_Q4(float)
GLMB_INSTANTIATE_Q4(__half)
GLMB_INSTANTIATE_Q4(__nv_bfloat16)

}  // namespace glmb
