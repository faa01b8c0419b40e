// glm_q4.cu -- models in 4 bits with group scales: quantise, dequantise, predict.
//
// A weight stands for q*s with q a whole number of -7..7 and s the scale of
// its target's group of features; codes are kept as q + 8 in blocks of 16
// targets x 64 features whose 32 x 16 bytes are the operand registers of four
// 16 x 16 tensor-core fragments, one 16-byte load per lane (the layout is
// written out in glm_matrix_b200.h).
#include <algorithm>

#include "glm_q4_device.cuh"
#include "glm_tc.cuh"

namespace glmb {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / kWarp;

inline unsigned warp_grid(int64_t warps) {
    return unsigned(std::max<int64_t>(1, std::min<int64_t>(int64_t(sm_count()) * 32, (warps + kWarps - 1) / kWarps)));
}

// ---- a lane's sixteen features of a row ---------------------------------------
//
// Lane 4g + c of a warp works on features 16k + 4c .. + 3, k = 0..3, of a
// 64-feature block of rows g and g + 8.  Where rows start on, and are made of,
// whole pieces of four (`vec`) it moves them as such; elsewhere the warp moves
// each row's 64 features side by side and passes them through shared memory.

constexpr int kTileLd = kQ4Cols + 8;  // elements of T between the rows of a staged block

template <typename T>
struct RowTile {
    alignas(16) T at[kQ4Rows][kTileLd];
};

// v[h][4k + j] = feature f0 + 16k + 4c + j of row row0 + g + 8h (zero past nf and past `rows`) of M[.][nf].
template <typename T>
__device__ __forceinline__ void load_rows(const T* M, int64_t row0, int rows, int64_t f0, int64_t nf, bool vec,
                                          RowTile<T>& tile, float (&v)[2][16]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    if (vec) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                T t[4] = {};
                if (g + 8 * h < rows && f0 + 16 * k + 4 * c < nf)
                    VecLoad<T, 4>::load(M + (row0 + g + 8 * h) * nf + f0 + 16 * k + 4 * c, t);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[h][4 * k + j] = to_arith<float>(t[j]);
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
            for (int i = 0; i < 16; ++i)
                v[h][i] = to_arith<float>(tile.at[g + 8 * h][16 * (i >> 2) + 4 * c + (i & 3)]);
    }
}

__device__ __forceinline__ float max_abs_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
    return r;
}

// w / s rounded to the nearest whole number q, ties to even, for |w / s| < 7.5 and s > 0: returned as the bits
// of the float kOne + q, whose low bits are q's.
constexpr float kOne = 12582912.0f;  // 1.5 * 2^23: adding it rounds to a whole number
template <typename T>
__device__ __forceinline__ uint32_t nearest_code(float w, float s, float inv, float half, float below) {
    if constexpr (std::is_same_v<T, float>) {
        // The float quotient can be off by an ulp and land on the wrong side of a border, so the remainder
        // d = w - q*s decides: it is exact in float (w and q*s are multiples of ulp(s)/2 when q != 0, and |d|
        // is s/2 or so).  `half` is s/2 and `below` the next float towards zero, the limits for even and odd q.
        const float m = fmaf(w, inv, kOne);
        const float d = fmaf(kOne - m, s, w);
        const int bits = __float_as_int(m);
        const int step = (__float_as_int(d) >> 31) | 1;
        return uint32_t(bits + (fabsf(d) > ((bits & 1) != 0 ? below : half) ? step : 0));
    } else {
        // One correction by the fused remainder (a Newton step on the quotient, as P. Markstein published it in
        // 1990) makes it the float nearest to w / s, which is w / s itself on a border; of 16-bit w and s (11 bits
        // at most) any other quotient is 2^-12 of it or more away from one.
        const float t = w * inv;
        return __float_as_uint(fmaf(fmaf(-t, s, w), inv, t) + kOne);
    }
}

// One warp per (task, 16 targets, group).  A group's largest magnitude is a maximum over the four lanes of
// a target.  One pass: the weights in, codes and scales out.  16384 x 4096 bfloat16 in groups of 128: 57 us, 2.9
// TB/s of the 6.5 that a copy reaches; bound by latency (two CTAs to an SM, for the 64 weights of a lane).  Held
// as 16-bit values with three CTAs to an SM, or with the next group's loads ahead, it took 64 and 85 us.
template <typename T, int GROUP>
__global__ void __launch_bounds__(kThreads, 2)
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
                // the sum of (q + 8) 2^shift, modulo 2^32, from the bits of kOne + q
                word[k] = 0x11111111u * (8u - __float_as_uint(kOne));
#pragma unroll
                for (int p = 0; p < 8; ++p) {
                    // p: pair 0..3 = (g, f), (g+8, f), (g, f+2), (g+8, f+2); 4..7 the same of f + 1
                    const int h = p & 1, i = 4 * k + (p & 2) + (p >> 2);
                    word[k] += nearest_code<T>(v[b][h][i], s[h], inv[h], half[h], below[h])
                               << (4 * (p & 3) + 16 * (p >> 2));
                }
            }
            codes[((task * nrb + rb) * ncb + cb) * 32 + lane] = make_uint4(word[0], word[1], word[2], word[3]);
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

// Four elements of T from the words that hold them.
template <typename T>
__device__ __forceinline__ void store_piece(T* dst, const uint32_t* w) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
}

// One warp per block of codes: M = q*s, rounded to T.  16384 x 4096 bfloat16: 31 us, 5.5 TB/s.
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
                T* dst = M + (row0 + g + 8 * h) * nf + f0 + 4 * c;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (f0 + 16 * k + 4 * c < nf) store_piece(dst + 16 * k, &out[h][k * kWords / 4]);
            }
        } else {
            RowTile<T>& tile = tiles[warp];
            __syncwarp();
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int k = 0; k < 4; ++k) store_piece(&tile.at[g + 8 * h][16 * k + 4 * c], &out[h][k * kWords / 4]);
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
// Bound by HBM: half a byte a weight, so with 1 to 16 observations the codes
// are nearly all that moves.  A warp takes a block of 16 targets x 64 features
// per step: one 16-byte load per lane is the block's four tensor-core
// fragments (mma.m16n8k16, weights as the 16-row operand), made into whole
// numbers of X's 16-bit type in registers, so a fragment costs the same for
// one observation as for eight (two fragments' columns for nine to sixteen); products of 16-bit values are exact and sums
// float.  A block's sums are scaled and added to the warp's totals.  float
// observations are three bfloat16 terms (8 bits each, together all 24), each
// with its own products.
//
// One CTA to an SM, with 1/148 of a model's row blocks each (to the nearest
// whole one) and its observations' features and scales in shared memory; the
// row blocks' codes, laid end to end, are cut into equal runs for its warps,
// so that no warp is left without work whatever the sizes.  A warp's sums for
// a row block go to a slot of its own, and a row block's slots are added up
// in the order of the warps.  Models with fewer row blocks than SMs share the
// features out over the CTAs of a cluster as well.
//
// 16384 x 4096 in groups of 128, bfloat16: 12.1 us for one observation (5.3 us
// of codes and scales at HBM's copy rate), 16.2 for 8, 21.9 for 16.  Not the
// instructions bound it -- about 110 per 128 features of a row block are 3 us of
// each scheduler's issue slots, of which 41 % are used -- but latency at both
// ends: each warp requests its first four pairs of blocks, of some 14 in all,
// then X and the scales are staged behind a barrier before the first is used,
// and the slots are summed once the last warp is through.
// A warp to a row block, its features shared over a cluster of four CTAs, took
// 18 us: two waves of CTAs, and its index arithmetic as long as its work.

constexpr int kStreamWarps = 16, kStreamThreads = kStreamWarps * 32;
constexpr int kStreamAhead = 4;   // pairs of blocks (128 features) in flight per warp
constexpr int kStreamRows = 16;   // row blocks a CTA works on together
constexpr int kSlots = kStreamRows / kStreamWarps + 3;  // row blocks one warp's run can touch
constexpr int kSlotLd = kQ4Rows + 1;

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

struct StreamArgs {
    int64_t nf, nt, ntasks;
    int64_t task0;      // of blockIdx.y == 0
    int nobs;           // at most 8 NT
    int nrb, ncb, ngroups;
    int rows;           // row blocks of a CTA
    int per_rank;       // 64-feature blocks to a CTA of the cluster (even)
    int chunk;          // blocks whose features are staged together (even)
    int group_shift;    // log2 of the blocks a group takes
    int ranks_log2;     // CTAs of a cluster, each with its share of the features
    bool vec;
};

// Where things lie in shared memory: features [term][obs], scales [row block][group], sums [warp][slot].
template <typename T, int NT>
struct StreamLayout {
    static constexpr int kTerms = Split16<T>::kTerms;
    static constexpr int kSlotFloats = 8 * NT * kSlotLd;
    int row_bytes, scales_ld;   // of one observation's features; scales of one row block (at most)
    int scales_at, slots_at, bytes;
    // 32 past a multiple of 128: the rows that sixteen lanes read together meet no bank twice
    __host__ __device__ StreamLayout(int chunk, int obs, int rows, int group_shift)
        : row_bytes(chunk * (kQ4Cols * 2) + 32), scales_ld((chunk >> group_shift) * kQ4Rows) {
        scales_at = kTerms * obs * row_bytes;
        slots_at = (scales_at + rows * scales_ld * int(sizeof(T)) + 15) / 16 * 16;
        bytes = slots_at + kStreamWarps * kSlots * kSlotFloats * 4;
    }
};

// NT: fragments of eight observations.  GROUPS: groups in 128 features.  FLAT: the CTA takes all of its row blocks' features at once, so that the
// codes of its row blocks lie end to end.
template <typename T, int NT, int GROUPS, bool FLAT>
__global__ void __launch_bounds__(kStreamThreads, 1)
    q4_stream_kernel(const T* __restrict__ X, const uint4* __restrict__ codes, const T* __restrict__ scales,
                     T* __restrict__ Yhat, StreamArgs a) {
    using H = typename Split16<T>::Type;
    constexpr int kTerms = Split16<T>::kTerms, kSlotFloats = StreamLayout<T, NT>::kSlotFloats;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const int rank = int(blockIdx.x) & ((1 << a.ranks_log2) - 1), ranks = 1 << a.ranks_log2;
    const int64_t task = a.task0 + blockIdx.y;
    const int obs_here = a.nobs;
    const int rb_begin = (int(blockIdx.x) >> a.ranks_log2) * a.rows, rb_end = min(a.nrb, rb_begin + a.rows);
    const int cb_begin = rank * a.per_rank, cb_end = min(a.ncb, cb_begin + a.per_rank);
    const StreamLayout<T, NT> at(a.chunk, obs_here, min(a.rows, kStreamRows), a.group_shift);
    T* const sm_scales = reinterpret_cast<T*>(smem_raw + at.scales_at);
    float* const slots = reinterpret_cast<float*>(smem_raw + at.slots_at);

    for (int rb0 = rb_begin; rb0 < rb_end; rb0 += kStreamRows) {
        const int rows = min(kStreamRows, rb_end - rb0);
        // the first row block this warp's runs can touch, whatever the chunk's length
        const int first_row = max(0, warp * rows / kStreamWarps - 1);
        float* const my_slots = slots + warp * kSlots * kSlotFloats;
        for (int i = lane; i < kSlots * kSlotFloats; i += 32) my_slots[i] = 0.0f;
        for (int chunk = cb_begin; chunk < cb_end; chunk += a.chunk) {
            const int blocks = min(a.chunk, cb_end - chunk);
            // this warp's run of the row blocks' codes laid end to end, in pairs of blocks
            const int pairs = blocks / 2;
            const int run0 = rows * pairs * warp / kStreamWarps, run1 = rows * pairs * (warp + 1) / kStreamWarps;
            int row = run0 / pairs, left_in_row = pairs - (run0 - row * pairs);
            const int col0 = pairs - left_in_row;
            const uint4* ahead = codes + ((task * a.nrb + rb0 + row) * a.ncb + chunk + 2 * col0) * 32 + lane;
            int ahead_left = run1 - run0, ahead_in_row = left_in_row;
            const int64_t skip = int64_t(a.ncb - blocks) * 32;
            uint4 w[kStreamAhead][2];
            auto fetch = [&](uint4 (&cw)[2]) {
                if (ahead_left > 0) {
                    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(cw[0].x), "=r"(cw[0].y), "=r"(cw[0].z), "=r"(cw[0].w)
                                 : "l"(ahead));
                    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(cw[1].x), "=r"(cw[1].y), "=r"(cw[1].z), "=r"(cw[1].w)
                                 : "l"(ahead + 32));
                }
                --ahead_left;
                ahead += 64;
                if (!FLAT && --ahead_in_row == 0) {
                    ahead_in_row = pairs;
                    ahead += skip;
                }
            };
#pragma unroll
            for (int j = 0; j < kStreamAhead; ++j) fetch(w[j]);

            if (chunk != cb_begin || rb0 != rb_begin) __syncthreads();  // what was staged has been read
            const int per_row = pairs * GROUPS * kQ4Rows;  // scales of a row block, row block after row block
            for (int i = tid; i < rows * per_row; i += kStreamThreads) {
                const int r = i / per_row, e = i - r * per_row;
                sm_scales[i] = scales[((task * a.nrb + rb0 + r) * a.ngroups + chunk / 2 * GROUPS) * kQ4Rows + e];
            }
            if (rb0 == rb_begin || a.chunk < a.per_rank) {
                constexpr int kPer = 16 / sizeof(T);
                const int64_t f0 = int64_t(chunk) * kQ4Cols;
                const int in = int(min(int64_t(blocks) * kQ4Cols, a.nf - f0));  // features of X; zero up to the block's end
                const int per_obs = blocks * (kQ4Cols / kPer);
#pragma unroll 2
                for (int i = tid; i < obs_here * per_obs; i += kStreamThreads) {
                    const int o = i / per_obs, f = (i - o * per_obs) * kPer;
                    const T* src = X + (o * a.ntasks + task) * a.nf + f0 + f;
                    T v[kPer] = {};
                    if (a.vec) {
                        if (f < in) VecLoad<T, kPer>::load(src, v);
                    } else {
#pragma unroll
                        for (int e = 0; e < kPer; ++e)
                            if (f + e < in) v[e] = src[e];
                    }
                    alignas(16) H t[kTerms][kPer];
#pragma unroll
                    for (int e = 0; e < kPer; ++e) {
                        H one[kTerms];
                        split_terms<T>(v[e], one);
#pragma unroll
                        for (int q = 0; q < kTerms; ++q) t[q][e] = one[q];
                    }
#pragma unroll
                    for (int q = 0; q < kTerms; ++q) {
                        unsigned char* dst = smem_raw + (q * obs_here + o) * at.row_bytes + f * 2;
                        if constexpr (kPer == 8) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(t[q]);
                        else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(t[q]);
                    }
                }
            }
            __syncthreads();

            // observations past the last one read another's row; their columns are not stored
            const unsigned char* x[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) x[n] = smem_raw + min(8 * n + g, obs_here - 1) * at.row_bytes + 8 * c;
            int col = col0 * (kQ4Cols * 4);  // bytes
            const T* sc = sm_scales + run0 * (GROUPS * kQ4Rows) + 2 * g;
            const int term_bytes = obs_here * at.row_bytes;
            float total[NT][4] = {};
            auto flush = [&] {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float* slot = my_slots + (row - first_row) * kSlotFloats + (8 * n + 2 * c) * kSlotLd + g;
                    slot[0] += total[n][0];
                    slot[kSlotLd] += total[n][1];
                    slot[8] += total[n][2];
                    slot[kSlotLd + 8] += total[n][3];
                }
            };
            auto add = [&](const float (&acc)[NT][4], const T* at_scale) {
                const Pair<T> s = *reinterpret_cast<const Pair<T>*>(at_scale);
                const float s0 = to_arith<float>(s.first), s1 = to_arith<float>(s.second);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    total[n][0] = fmaf(s0, acc[n][0], total[n][0]);
                    total[n][1] = fmaf(s0, acc[n][1], total[n][1]);
                    total[n][2] = fmaf(s1, acc[n][2], total[n][2]);
                    total[n][3] = fmaf(s1, acc[n][3], total[n][3]);
                }
            };
            for (int left = run1 - run0; left > 0; left -= kStreamAhead) {
#pragma unroll
                for (int j = 0; j < kStreamAhead; ++j) {
                    if (j >= left) break;
                    uint32_t frag[2][4][4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        code_pairs<H, kCodeDown<H>>(w[j][h].x, frag[h][0]);
                        code_pairs<H, kCodeDown<H>>(w[j][h].y, frag[h][1]);
                        code_pairs<H, kCodeDown<H>>(w[j][h].z, frag[h][2]);
                        code_pairs<H, kCodeDown<H>>(w[j][h].w, frag[h][3]);
                    }
                    fetch(w[j]);
                    float acc[NT][4] = {};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int q = kTerms - 1; q >= 0; --q)
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    const uint2 xv = *reinterpret_cast<const uint2*>(
                                        x[n] + col + q * term_bytes + h * (kQ4Cols * 2) + 32 * k);
                                    mma_16816<H>(acc[n], frag[h][k], xv.x, xv.y);
                                }
                        if (GROUPS == 2) {
                            add(acc, sc + h * kQ4Rows);
#pragma unroll
                            for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.0f;
                        }
                    }
                    if (GROUPS == 1) add(acc, sc);
                    col += kQ4Cols * 4;
                    sc += GROUPS * kQ4Rows;
                    if (--left_in_row == 0) {
                        flush();
#pragma unroll
                        for (int n = 0; n < NT; ++n) total[n][0] = total[n][1] = total[n][2] = total[n][3] = 0.0f;
                        left_in_row = pairs;
                        col = 0;
                        ++row;
                    }
                }
            }
            if (left_in_row < pairs && run1 > run0) flush();
        }

        __syncthreads();
        if (ranks > 1) cluster_sync();
        const int outputs = rows * kQ4Rows;
        for (int i = rank * kStreamThreads + tid; i < outputs * obs_here; i += ranks * kStreamThreads) {
            const int o = i / outputs, t = i - o * outputs, r = t / kQ4Rows;
            const int64_t target = int64_t(rb0) * kQ4Rows + t;
            float v = 0.0f;
            for (int p = 0; p < ranks; ++p)
                for (int k = 0; k < kStreamWarps; ++k) {
                    const int slot = r - max(0, k * rows / kStreamWarps - 1);
                    if (slot < 0) break;
                    if (slot >= kSlots) continue;
                    const float* from = slots + (k * kSlots + slot) * kSlotFloats + o * kSlotLd + t % kQ4Rows;
                    v += ranks > 1 ? ld_cluster_f32(from, p) : *from;
                }
            if (target < a.nt) Yhat[(o * a.ntasks + task) * a.nt + target] = from_arith<T>(v * kCodeUp<H>);
        }
        if (ranks > 1) cluster_sync_relaxed();  // the peers have read this CTA's sums
        else if (rb0 + kStreamRows < rb_end) __syncthreads();
    }
}

template <typename T, int NT>
int stream_predict(const T* X, const void* codes, const T* scales, T* Yhat, StreamArgs a, cudaStream_t stream) {
    constexpr size_t kRoom = size_t(224) * 1024;
    const int obs = a.nobs;
    const int64_t sms = sm_count();
    // CTAs for a task's row blocks, one to an SM
    const int64_t ctas = std::max<int64_t>(1, sms / std::min(sms, a.ntasks));
    a.rows = int((a.nrb + ctas - 1) / ctas);
    const int64_t groups = (a.nrb + a.rows - 1) / a.rows;
    // CTAs of a cluster: while they find SMs and each warp two blocks of codes
    while (a.ranks_log2 < 3 && ((groups * a.ntasks) << (a.ranks_log2 + 1)) <= sms &&
           int64_t(a.ncb) * a.rows >= (2 * kStreamWarps) << (a.ranks_log2 + 1))
        ++a.ranks_log2;
    const int ranks = 1 << a.ranks_log2, rows = std::min(a.rows, kStreamRows);
    a.per_rank = ((a.ncb + ranks - 1) / ranks + 1) / 2 * 2;
    // the longest run of features that leaves room for the scales and sums
    a.chunk = a.per_rank;
    while (size_t(StreamLayout<T, NT>(a.chunk, obs, rows, a.group_shift).bytes) > kRoom) a.chunk = (a.chunk / 2 + 1) / 2 * 2;
    const bool flat = a.chunk >= a.ncb;
    static std::atomic<uint64_t> attr[4];
    void (*const kernels[4])(const T*, const uint4*, const T*, T*, StreamArgs) = {
        q4_stream_kernel<T, NT, 1, false>, q4_stream_kernel<T, NT, 1, true>, q4_stream_kernel<T, NT, 2, false>,
        q4_stream_kernel<T, NT, 2, true>};
    const int which = (a.group_shift == 0 ? 2 : 0) + (flat ? 1 : 0);
    const auto kernel = kernels[which];
    cudaError_t e = set_smem_limit_once(attr[which], kernel, kRoom);
    if (e != cudaSuccess) return int(e);
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kStreamThreads);
    cfg.dynamicSmemBytes = size_t(StreamLayout<T, NT>(a.chunk, obs, rows, a.group_shift).bytes);
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = unsigned(ranks);
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    for (a.task0 = 0; a.task0 < a.ntasks; a.task0 += 65535) {
        cfg.gridDim = dim3(unsigned(groups << a.ranks_log2), unsigned(std::min<int64_t>(65535, a.ntasks - a.task0)));
        count_launch();
        e = cudaLaunchKernelEx(&cfg, kernel, X, static_cast<const uint4*>(codes), scales, Yhat, StreamArgs(a));
        if (e != cudaSuccess) return int(e);
    }
    return launch_status();
}

// Whether rows of nf elements from p on start on, and are made of, whole pieces of `bytes`.
template <typename T>
bool whole_pieces(const T* p, int64_t nf, size_t bytes) {
    return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0 && nf % int64_t(bytes / sizeof(T)) == 0;
}

}  // namespace

template <typename T>
int q4_quantize(const T* M, void* codes, T* scales, int64_t nf, int64_t nt, int64_t ntasks, int group,
                cudaStream_t stream) {
    const int64_t nrb = q4_row_blocks(nt), ncb = q4_col_blocks(nf), ng = q4_groups(nf, group);
    const int64_t total = ntasks * nrb * ng;
    auto kernel = group == 64 ? q4_quantize_kernel<T, 64> : q4_quantize_kernel<T, 128>;
    kernel<<<warp_grid(total), kThreads, 0, stream>>>(M, static_cast<uint4*>(codes), scales, nf, nt, nrb, ncb, ng,
                                                      total, whole_pieces(M, nf, 4 * sizeof(T)));
    count_launch();
    return launch_status();
}

template <typename T>
int q4_dequantize(const void* codes, const T* scales, T* M, int64_t nf, int64_t nt, int64_t ntasks, int group,
                  cudaStream_t stream) {
    const int64_t nrb = q4_row_blocks(nt), ncb = q4_col_blocks(nf), ng = q4_groups(nf, group);
    const int64_t total = ntasks * nrb * ncb;
    q4_dequantize_kernel<T><<<warp_grid(total), kThreads, 0, stream>>>(
        static_cast<const uint4*>(codes), scales, M, nf, nt, nrb, ncb, ng, group == 64 ? 6 : 7, total, whole_pieces(M, nf, 4 * sizeof(T)));
    count_launch();
    return launch_status();
}

// Up to this many observations go through the stream kernel.  Stream and tile on either side of the limit, in us:
// bfloat16 at 16 and 17 observations 21.8 and 20.5 on 16384 x 4096, 12.8 and 13.7 on 4096 x 4096, 6.0 and 8.4 on
// 1000 x 777, 4.7 and 5.2 on 64 models of 16 x 256, 11.8 and 20.7 on 300 of them.  float, whose three terms take
// three times the products, was measured on both sides at 16384 x 4096 alone, 32 and 26.3 at 9 observations.
template <typename T>
constexpr int64_t kStreamMost = sizeof(T) == 2 ? 16 : 8;

template <typename T>
size_t q4_predict_workspace(int64_t nf, int64_t nt, int64_t ntasks, int64_t nobs, int group) {
    return nobs <= kStreamMost<T> ? 0 : q4_tile_workspace<T>(nf, ntasks, nobs);
}

template <typename T>
int q4_predict(const T* X, const void* codes, const T* scales, T* Yhat, int64_t nf, int64_t nt, int64_t ntasks,
               int64_t nobs, int group, void* ws, size_t ws_bytes, cudaStream_t stream) {
    const int64_t nrb = q4_row_blocks(nt), ncb = q4_col_blocks(nf), ng = q4_groups(nf, group);
    if (nrb > (1 << 27) || ncb > (1 << 20)) return GLMB_ERR_TOO_LARGE;
    if (nobs > kStreamMost<T>) {
        set_last_path("q4_tile");
        return q4_tile_predict<T>(X, codes, scales, Yhat, nf, nt, ntasks, nobs, group, whole_pieces(X, nf, 16), ws,
                                  ws_bytes, stream);
    }
    StreamArgs a{nf, nt, ntasks, 0, int(nobs), int(nrb), int(ncb), int(ng), 0, 0, 0, group == 64 ? 0 : 1, 0,
                 whole_pieces(X, nf, 16)};
    set_last_path("q4_stream");
    if constexpr (kStreamMost<T> > 8)
        if (nobs > 8) return stream_predict<T, 2>(X, codes, scales, Yhat, a, stream);
    return stream_predict<T, 1>(X, codes, scales, Yhat, a, stream);
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
