// glm_q4.cu -- models in 4 bits with group scales: quantise, dequantise, predict.
//
// A weight stands for q*s with q a whole number of -7..7 and s the scale of
// its target's group of features; codes are kept as q + 8 in blocks of 16
// targets x 64 features whose 32 x 16 bytes are the operand registers of four
// 16 x 16 tensor-core fragments, one 16-byte load per lane (the layout is
// written out in glm_matrix_b200.h).
#include <algorithm>

#include "glm_q4.cuh"
#include "glm_tc.cuh"

namespace glmb {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / kWarp;

inline unsigned warp_grid(int64_t warps) {
    return unsigned(std::max<int64_t>(1, std::min<int64_t>(int64_t(sm_count()) * 32, (warps + kWarps - 1) / kWarps)));
}

// ---- rows of sixteen features -------------------------------------------------
//
// Lane 4g + c of a warp works on features 16c..16c+15 of a 64-feature block of
// rows g and g + 8.  Where rows start on 16 bytes (`vec`) it moves its sixteen
// as 16-byte pieces; elsewhere the warp moves each row's 64 features side by
// side and passes them through shared memory.

constexpr int kTileLd = kQ4Cols + 8;  // elements of T between the rows of a staged block

template <typename T>
struct RowTile {
    alignas(16) T at[kQ4Rows][kTileLd];
};

// v = features f0 + 16c.. of rows row0 + g and row0 + g + 8 (zero past nf and past `rows`) of M[.][nf].
template <typename T>
__device__ __forceinline__ void load_rows(const T* M, int64_t row0, int rows, int64_t f0, int64_t nf, bool vec,
                                          RowTile<T>& tile, float (&v)[2][16]) {
    constexpr int kPer = 16 / sizeof(T);
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    if (vec) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 16; i += kPer) {
                T t[kPer] = {};
                if (g + 8 * h < rows && f0 + 16 * c + i < nf)
                    VecLoad<T, kPer>::load(M + (row0 + g + 8 * h) * nf + f0 + 16 * c + i, t);
#pragma unroll
                for (int j = 0; j < kPer; ++j) v[h][i + j] = to_arith<float>(t[j]);
            }
    } else {
        __syncwarp();
#pragma unroll 4
        for (int r = 0; r < kQ4Rows; ++r)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int64_t f = f0 + lane + 32 * i;
                tile.at[r][lane + 32 * i] = r < rows && f < nf ? M[(row0 + r) * nf + f] : from_arith<T>(0.0f);
            }
        __syncwarp();
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 16; i += kPer) {
                alignas(16) T t[kPer];
                *reinterpret_cast<uint4*>(t) = *reinterpret_cast<const uint4*>(&tile.at[g + 8 * h][16 * c + i]);
#pragma unroll
                for (int j = 0; j < kPer; ++j) v[h][i + j] = to_arith<float>(t[j]);
            }
    }
}

__device__ __forceinline__ float max_abs_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
    return r;
}

// q + 8 with q = w / s rounded to the nearest whole number, ties to even, for |w / s| < 7.5 and s > 0.  The
// float product w * (1/s) can be off by an ulp and land on the wrong side of a border, so the remainder
// d = w - q*s decides: it is exact in float (w and q*s are multiples of ulp(s)/2 when q != 0, and |d| is s/2
// or so).  `half` is s/2 and `below` the next float towards zero, the limits for even and for odd q.
__device__ __forceinline__ uint32_t nearest_code(float w, float s, float inv, float half, float below) {
    constexpr float kOne = 12582912.0f;  // 1.5 * 2^23: adding it rounds to a whole number, found in the low bits
    const float m = fmaf(w, inv, kOne);
    const float d = fmaf(kOne - m, s, w);
    const int bits = __float_as_int(m);
    const int step = (__float_as_int(d) >> 31) | 1;
    return uint32_t(bits + 8 + (fabsf(d) > ((bits & 1) != 0 ? below : half) ? step : 0)) & 15u;
}

// One warp per (task, 16 targets, group).  A group's largest magnitude is a maximum over the four lanes of
// a target.  One pass: the weights in, codes and scales out.
template <typename T, int GROUP>
__global__ void __launch_bounds__(kThreads)
    q4_quantize_kernel(const T* __restrict__ M, uint4* __restrict__ codes, T* __restrict__ scales, int64_t nf,
                       int64_t nt, int64_t nrb, int64_t ncb, int64_t ngroups, int64_t total, bool vec) {
    constexpr int kBlocks = GROUP / kQ4Cols;
    __shared__ RowTile<T> tiles[kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    for (int64_t w = int64_t(blockIdx.x) * kWarps + warp; w < total; w += int64_t(gridDim.x) * kWarps) {
        const int64_t group = w % ngroups, rb = w / ngroups % nrb, task = w / ngroups / nrb;
        const int rows = int(min(int64_t(kQ4Rows), nt - rb * kQ4Rows));
        float v[kBlocks][2][16];
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
            load_rows(M, task * nt + rb * kQ4Rows, rows, group * GROUP + b * kQ4Cols, nf, vec, tiles[warp], v[b]);
        float s[2], inv[2];
        T st[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float top = 0.0f;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) top = max_abs_nan(top, v[b][h][i]);
#pragma unroll
            for (int off = 1; off < 4; off <<= 1) top = max_abs_nan(top, __shfl_xor_sync(0xffffffffu, top, off));
            const bool finite = top <= 3.402823466e38f;
            st[h] = from_arith<T>(finite ? __fdiv_rn(top, 7.0f) : __int_as_float(0x7fc00000));
            s[h] = finite ? to_arith<float>(st[h]) : 0.0f;
            if (s[h] < 0x1p-100f || top > 7.25f * s[h]) {
                // Rare: a group of zeros or with a NaN (every code is 0); a scale near the bottom of float's
                // range, lifted with its weights, which changes no ratio; one rounded so far down, among the
                // subnormals of T, that weights reach past 7.
                const float up = s[h] < 0x1p-100f ? 0x1p60f : 1.0f;
                const float most = 7.0f * (s[h] * up);
#pragma unroll
                for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        v[b][h][i] = s[h] > 0.0f ? fminf(fmaxf(v[b][h][i] * up, -most), most) : 0.0f;
                s[h] = s[h] > 0.0f ? s[h] * up : 1.0f;
            }
            inv[h] = __frcp_rn(s[h]);
        }
        if (c == 0) {
            T* dst = scales + ((task * nrb + rb) * ngroups + group) * kQ4Rows + 2 * g;
            dst[0] = st[0];
            dst[1] = st[1];
        }
        const float half[2] = {0.5f * s[0], 0.5f * s[1]};
        const float below[2] = {__int_as_float(__float_as_int(half[0]) - 1), __int_as_float(__float_as_int(half[1]) - 1)};
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
                    word[k] |= nearest_code(v[b][h][i], s[h], inv[h], half[h], below[h]) << (4 * (p & 3) + 16 * (p >> 2));
                }
            }
            codes[((task * nrb + rb) * ncb + cb) * 32 + lane] = make_uint4(word[0], word[1], word[2], word[3]);
        }
    }
}

// The 16-bit type the tensor core multiplies in, and how many terms an X takes.
template <typename T>
struct Split16 {
    using Type = T;
    static constexpr int kTerms = 1;
};
template <>
struct Split16<float> {
    using Type = __nv_bfloat16;
    static constexpr int kTerms = 3;
};

// The four pairs of a word of codes (u = q + 8) as 16-bit floats q: the code is put under the leading bit of
// a power of two (1024 + u or, four bits up, 1024 + 16u in binary16; 128 + u in bfloat16) and the offset taken
// off again, exactly.
template <typename H>
__device__ __forceinline__ void code_pairs(uint32_t w, uint32_t (&r)[4]) {
    if constexpr (std::is_same_v<H, __half>) {
        const __half2 off = __float2half2_rn(-1032.0f), sixteenth = __float2half2_rn(0.0625f),
                      off16 = __float2half2_rn(-72.0f);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t lo = ((w >> (8 * i)) & 0x000f000fu) | 0x64006400u, hi = ((w >> (8 * i)) & 0x00f000f0u) | 0x64006400u;
            const __half2 a = __hadd2(*reinterpret_cast<__half2*>(&lo), off);
            const __half2 b = __hfma2(*reinterpret_cast<__half2*>(&hi), sixteenth, off16);
            r[2 * i] = *reinterpret_cast<const uint32_t*>(&a);
            r[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&b);
        }
    } else {
        const __nv_bfloat162 off = __float2bfloat162_rn(-136.0f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t v = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
            const __nv_bfloat162 a = __hadd2(*reinterpret_cast<__nv_bfloat162*>(&v), off);
            r[i] = *reinterpret_cast<const uint32_t*>(&a);
        }
    }
}

// A pair of codes times a scale, rounded to T, as the 32-bit words of two elements of T (one for 16-bit types).
template <typename T>
__device__ __forceinline__ void scaled_pair(uint32_t pair, T s, uint32_t* dst) {
    if constexpr (std::is_same_v<T, float>) {
        dst[0] = __float_as_uint(__uint_as_float(pair << 16) * s);
        dst[1] = __float_as_uint(__uint_as_float(pair & 0xffff0000u) * s);
    } else if constexpr (std::is_same_v<T, __half>) {
        const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&pair), __half2half2(s));
        dst[0] = *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&pair), __bfloat162bfloat162(s));
        dst[0] = *reinterpret_cast<const uint32_t*>(&v);
    }
}

// One warp per block of codes: M = q*s, rounded to T.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    q4_dequantize_kernel(const uint4* __restrict__ codes, const T* __restrict__ scales, T* __restrict__ M, int64_t nf,
                         int64_t nt, int64_t nrb, int64_t ncb, int64_t ngroups, int group_log2, int64_t total, bool vec) {
    using H = typename Split16<T>::Type;
    constexpr int kWords = 16 * sizeof(T) / 4;  // of a lane's sixteen features of one row
    __shared__ RowTile<T> tiles[kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    for (int64_t w = int64_t(blockIdx.x) * kWarps + warp; w < total; w += int64_t(gridDim.x) * kWarps) {
        const int64_t cb = w % ncb, rb = w / ncb % nrb, task = w / ncb / nrb;
        const uint4 block = codes[w * 32 + lane];
        const T* sc = scales + ((task * nrb + rb) * ngroups + ((cb * kQ4Cols) >> group_log2)) * kQ4Rows + 2 * g;
        const T s[2] = {sc[0], sc[1]};
        const uint32_t word[4] = {block.x, block.y, block.z, block.w};
        uint32_t out[2][kWords];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint32_t pair[4];
            code_pairs<H>(word[k], pair);
#pragma unroll
            for (int p = 0; p < 4; ++p) scaled_pair<T>(pair[p], s[p & 1], &out[p & 1][(2 * k + (p >> 1)) * kWords / 8]);
        }
        const int rows = int(min(int64_t(kQ4Rows), nt - rb * kQ4Rows));
        const int64_t row0 = task * nt + rb * kQ4Rows, f0 = cb * kQ4Cols;
        if (vec) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (g + 8 * h >= rows) continue;
                T* dst = M + (row0 + g + 8 * h) * nf + f0 + 16 * c;
#pragma unroll
                for (int i = 0; i < kWords; i += 4)
                    if (f0 + 16 * c + i * int(4 / sizeof(T)) < nf)
                        *reinterpret_cast<uint4*>(reinterpret_cast<uint32_t*>(dst) + i) =
                            make_uint4(out[h][i], out[h][i + 1], out[h][i + 2], out[h][i + 3]);
            }
        } else {
            RowTile<T>& tile = tiles[warp];
            __syncwarp();
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < kWords; i += 4)
                    *reinterpret_cast<uint4*>(reinterpret_cast<uint32_t*>(&tile.at[g + 8 * h][16 * c]) + i) =
                        make_uint4(out[h][i], out[h][i + 1], out[h][i + 2], out[h][i + 3]);
            __syncwarp();
#pragma unroll 4
            for (int r = 0; r < kQ4Rows; ++r)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int64_t f = f0 + lane + 32 * i;
                    if (r < rows && f < nf) M[(row0 + r) * nf + f] = tile.at[r][lane + 32 * i];
                }
        }
    }
}

// ---- a few observations: the stream of the codes ------------------------------
//
// Bound by HBM: half a byte a weight, so with 1 to 32 observations the codes
// are nearly all that moves.  A warp takes a block of 16 targets x 64 features
// per step: one 16-byte load per lane is the block's four tensor-core
// fragments (mma.m16n8k16, weights as the 16-row operand), made into whole
// numbers of X's 16-bit type in registers, so a fragment costs the same for
// one observation as for eight; products of 16-bit values are exact and sums
// float.  A block's sums are scaled and added to the warp's totals.  float
// observations are three bfloat16 terms (8 bits each, together all 24), each
// with its own products.
//
// A CTA holds its observations' features in shared memory (in the order of
// memory: lane 4g + c reads features 16c.. of observation g, which is what the
// codes' order was chosen for); its eight warps share out row blocks and, where
// a model has fewer than eight, features.  The features may also be shared by
// the CTAs of a cluster, whose partial sums meet in distributed shared memory
// in a fixed order.

constexpr int kStreamChunk = 1024;  // features staged together
constexpr int kStreamAhead = 4;     // blocks of codes in flight per warp

template <typename H>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same_v<H, __half>)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x as a sum of terms of the tensor core's type (one for a 16-bit x, three for a float)
template <typename T>
__device__ __forceinline__ void split_terms(T x, typename Split16<T>::Type (&t)[Split16<T>::kTerms]) {
    if constexpr (std::is_same_v<T, float>) {
        // a NaN or an infinity stays in the first term alone
        t[0] = __float2bfloat16_rn(x);
        const float r1 = x - __bfloat162float(t[0]);
        const bool finite = fabsf(__bfloat162float(t[0])) <= 3.402823466e38f;
        t[1] = __float2bfloat16_rn(finite ? r1 : 0.0f);
        t[2] = __float2bfloat16_rn(finite ? r1 - __bfloat162float(t[1]) : 0.0f);
    } else {
        t[0] = x;
    }
}

template <typename T>
struct alignas(2 * sizeof(T)) Pair {
    T first, second;
};

struct StreamArgs {
    int64_t nf, nt, ntasks, nobs;
    int64_t nrb, ncb, ngroups;
    int64_t row_groups;   // CTAs (clusters) a task's row blocks take
    int64_t per_rank;     // 64-feature blocks to a CTA of the cluster (even)
    int group_log2;
    int ranks;            // CTAs of a cluster, each with its share of the features
    int rows_log2;        // log2 of the row blocks a CTA takes; 8 >> rows_log2 warps share each one's features
    bool vec;
};

template <typename T, int NT>
__global__ void __launch_bounds__(kThreads)
    q4_stream_kernel(const T* __restrict__ X, const uint4* __restrict__ codes, const T* __restrict__ scales,
                     T* __restrict__ Yhat, const StreamArgs a) {
    using H = typename Split16<T>::Type;
    constexpr int kTerms = Split16<T>::kTerms;
    constexpr int kObs = 8 * NT;
    constexpr int kRowBytes = kStreamChunk * 2 + 16;  // 16 past a multiple of 128: eight lanes' reads meet no bank twice
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const uint32_t rank = cluster_rank();
    const int ranks = a.ranks;  // CTAs of a cluster
    const int64_t unit = blockIdx.x / unsigned(ranks);
    const int64_t rg = unit % a.row_groups, task = unit / a.row_groups % a.ntasks;
    const int64_t obs0 = unit / a.row_groups / a.ntasks * kObs;
    const int obs_here = int(min(int64_t(kObs), a.nobs - obs0));
    const int rows = 1 << a.rows_log2, wk = warp >> a.rows_log2, wks = kWarps >> a.rows_log2;
    const int64_t rb = rg * rows + (warp & (rows - 1));
    const bool live = rb < a.nrb;
    const int64_t cb_begin = int64_t(rank) * a.per_rank, cb_end = min(a.ncb, cb_begin + a.per_rank);
    const uint4* my_codes = codes + ((task * a.nrb + (live ? rb : 0)) * a.ncb) * 32 + lane;
    const T* my_scales = scales + (task * a.nrb + (live ? rb : 0)) * a.ngroups * kQ4Rows + 2 * g;
    const int group_shift = a.group_log2 - 6;

    float total[NT][4] = {};
    for (int64_t chunk = cb_begin; chunk < cb_end; chunk += kStreamChunk / kQ4Cols) {
        const int blocks = int(min(int64_t(kStreamChunk / kQ4Cols), cb_end - chunk));
        // (blocks come in pairs of 128 features: a warp's j-th is block wk2 + (j/2) * stride + j%2)
        const int wk2 = 2 * wk, stride = 2 * wks;
        const uint4* cp = my_codes + chunk * 32;
        const T* sp = my_scales + ((chunk * kQ4Cols) >> a.group_log2) * kQ4Rows;
        const int limit = live ? blocks : 0;
        uint4 w[kStreamAhead];
        Pair<T> s[kStreamAhead];
        auto fetch = [&](int b, uint4& cw, Pair<T>& cs) {
            if (b < limit) {
                asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                             : "=r"(cw.x), "=r"(cw.y), "=r"(cw.z), "=r"(cw.w)
                             : "l"(cp + b * 32));
                cs = *reinterpret_cast<const Pair<T>*>(sp + (b >> group_shift) * kQ4Rows);
            }
        };
#pragma unroll
        for (int j = 0; j < kStreamAhead; ++j) fetch(wk2 + (j >> 1) * stride + (j & 1), w[j], s[j]);

        if (chunk != cb_begin) __syncthreads();  // the chunk before has been read
        {
            constexpr int kPer = 16 / sizeof(T);
            const int64_t f0 = chunk * kQ4Cols;
            const int feats = blocks * kQ4Cols;
            for (int i = tid; i < obs_here * (feats / kPer); i += kThreads) {
                const int o = i / (feats / kPer), f = i % (feats / kPer) * kPer;
                const T* src = X + ((obs0 + o) * a.ntasks + task) * a.nf + f0 + f;
                T v[kPer] = {};
                if (a.vec) {
                    if (f0 + f < a.nf) VecLoad<T, kPer>::load(src, v);
                } else {
#pragma unroll
                    for (int e = 0; e < kPer; ++e)
                        if (f0 + f + e < a.nf) v[e] = src[e];
                }
                H t[kTerms][kPer];
#pragma unroll
                for (int e = 0; e < kPer; ++e) {
                    H one[kTerms];
                    split_terms<T>(v[e], one);
#pragma unroll
                    for (int q = 0; q < kTerms; ++q) t[q][e] = one[q];
                }
#pragma unroll
                for (int q = 0; q < kTerms; ++q) {
                    unsigned char* dst = smem_raw + (q * kObs + o) * kRowBytes + f * 2;
                    if constexpr (kPer == 8) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(t[q]);
                    else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(t[q]);
                }
            }
        }
        __syncthreads();

        for (int b0 = wk2; b0 < limit; b0 += kStreamAhead / 2 * stride) {
#pragma unroll
            for (int jj = 0; jj < kStreamAhead; ++jj) {
                const int b = b0 + (jj >> 1) * stride + (jj & 1);
                if (b >= limit) continue;
                const uint4 cw = w[jj];
                const float s0 = to_arith<float>(s[jj].first), s1 = to_arith<float>(s[jj].second);
                fetch(b + kStreamAhead / 2 * stride, w[jj], s[jj]);
                const uint32_t word[4] = {cw.x, cw.y, cw.z, cw.w};
                uint32_t frag[4][4];
#pragma unroll
                for (int k = 0; k < 4; ++k) code_pairs<H>(word[k], frag[k]);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    // observations past the last one read another's row; their columns are not stored
                    const int o = min(8 * n + g, obs_here - 1);
                    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int q = kTerms - 1; q >= 0; --q) {
                        const uint4* x = reinterpret_cast<const uint4*>(smem_raw + (q * kObs + o) * kRowBytes +
                                                                        (b * kQ4Cols + 16 * c) * 2);
                        const uint4 x0 = x[0], x1 = x[1];
                        mma_16816<H>(acc, frag[0], x0.x, x0.y);
                        mma_16816<H>(acc, frag[1], x0.z, x0.w);
                        mma_16816<H>(acc, frag[2], x1.x, x1.y);
                        mma_16816<H>(acc, frag[3], x1.z, x1.w);
                    }
                    total[n][0] = fmaf(s0, acc[0], total[n][0]);
                    total[n][1] = fmaf(s0, acc[1], total[n][1]);
                    total[n][2] = fmaf(s1, acc[2], total[n][2]);
                    total[n][3] = fmaf(s1, acc[3], total[n][3]);
                }
            }
        }
    }

    // ---- the warps' and the cluster's partial sums ----
    __syncthreads();
    constexpr int kPartLd = kQ4Rows + 1;
    float* part = reinterpret_cast<float*>(smem_raw);  // [warp][obs][16 targets]
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            part[(warp * kObs + 8 * n + 2 * c + (i & 1)) * kPartLd + g + 8 * (i >> 1)] = total[n][i];
    __syncthreads();
    if (ranks > 1) cluster_sync();
    const int outputs = rows * kQ4Rows * obs_here;
    const int begin = outputs * int(rank) / ranks, end = outputs * (int(rank) + 1) / ranks;
    for (int i = begin + tid; i < end; i += kThreads) {
        const int o = i / (rows * kQ4Rows), t = i % (rows * kQ4Rows);
        const int64_t target = rg * rows * kQ4Rows + t;
        float v = 0.0f;
        for (int r = 0; r < ranks; ++r)
            for (int k = 0; k < wks; ++k) {
                const float* at = part + ((k * rows + t / kQ4Rows) * kObs + o) * kPartLd + t % kQ4Rows;
                v += ranks > 1 ? ld_cluster_f32(at, r) : *at;
            }
        if (target < a.nt) Yhat[((obs0 + o) * a.ntasks + task) * a.nt + target] = from_arith<T>(v);
    }
    if (ranks > 1) cluster_sync_relaxed();  // the peers have read this CTA's sums
}

template <typename T, int NT>
int stream_launch(const T* X, const void* codes, const T* scales, T* Yhat, const StreamArgs& a,
                  cudaStream_t stream) {
    const size_t smem = std::max(size_t(Split16<T>::kTerms) * 8 * NT * (kStreamChunk * 2 + 16),
                                 size_t(kWarps) * 8 * NT * (kQ4Rows + 1) * 4);
    static std::atomic<uint64_t> attr{0};
    auto kernel = q4_stream_kernel<T, NT>;
    cudaError_t e = set_smem_limit_once(attr, kernel, smem);
    if (e != cudaSuccess) return int(e);
    cudaLaunchConfig_t cfg = {};
    const int64_t units = a.row_groups * a.ntasks * ((a.nobs + 8 * NT - 1) / (8 * NT));
    if (units > (int64_t(1) << 31) / a.ranks - 1) return GLMB_ERR_TOO_LARGE;
    cfg.gridDim = dim3(unsigned(units * a.ranks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = unsigned(a.ranks);
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    count_launch();
    e = cudaLaunchKernelEx(&cfg, kernel, X, static_cast<const uint4*>(codes), scales, Yhat, a);
    return e != cudaSuccess ? int(e) : launch_status();
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
        static_cast<const uint4*>(codes), scales, M, nf, nt, nrb, ncb, ng, group == 64 ? 6 : 7, total, whole_vectors(M, nf));
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
    StreamArgs a{nf, nt, ntasks, nobs, nrb, ncb, ng, 0, 0, group == 64 ? 6 : 7, 1, 0, whole_vectors(X, nf)};
    while (a.rows_log2 < 3 && (int64_t(1) << a.rows_log2) < nrb) ++a.rows_log2;
    a.row_groups = (nrb + (int64_t(1) << a.rows_log2) - 1) >> a.rows_log2;
    // CTAs that share a row group's features: until every SM has four CTAs, while each keeps 128 features a warp
    const int64_t least = 2 * (kWarps >> a.rows_log2);
    while (a.ranks < 8 && a.row_groups * ntasks * a.ranks * 2 <= 4 * int64_t(sm_count()) &&
           ncb >= 2 * a.ranks * least)
        a.ranks *= 2;
    a.per_rank = ((ncb + a.ranks - 1) / a.ranks + 1) / 2 * 2;
    set_last_path("q4_stream");
    if (nobs <= 8) return stream_launch<T, 1>(X, codes, scales, Yhat, a, stream);
    if (nobs <= 16) return stream_launch<T, 2>(X, codes, scales, Yhat, a, stream);
    return stream_launch<T, 4>(X, codes, scales, Yhat, a, stream);
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
