// glm_ortho_gemm.cu -- the three products of a Newton-Schulz step on the
// 5th-generation tensor cores:
//   A = X X^T (and C = bI + cA),   B = aI + A C,   X' = B X      (X: m x n, m <= n).
//
// Operands are pairs of binary16 values, hi = the value rounded to nearest and
// lo = the rest rounded to nearest, after a scaling by a power of two that the
// host derives from the bound on X's singular values (glm_ortho.cuh): 22
// significant bits where the low value is normal (down to 2^-17 of the bound),
// an error of 2^-25 of the scaled unit (2^-39 of the bound) below.  A
// product takes three MMAs (hi*lo + lo*hi + hi*hi; the dropped lo*lo is 2^-22
// of the product), at twice the rate of tf32 and half its bytes.  Normalised
// iterates make this possible: nothing in X, A or B can leave binary16's range.
//
// The tensor core cuts towards zero where it accumulates, so each 64-deep
// block of K is accumulated from zero in one of two TMEM buffers (small
// corrections first) and eight warps add it into float registers, rounding to
// nearest, while the tensor core fills the other buffer.
//
// A and B are symmetric: only the tiles on and above the diagonal are
// computed, and the epilogue writes each tile and its mirror image.
//
// Two tile shapes.  PAIR: 256 x 256 on a CTA pair (cta_group::2), each CTA
// staging its 128 rows of the left operand and 128 of the 256 columns of the
// right one -- 64 KB for 1536 clocks of MMA, where a 128 x 128 tile of one CTA
// brings in the same bytes for half the work.  Single: 128 x 128 on one CTA,
// for products with too few large tiles.  Either may split K over the CTAs
// (pairs) of a cluster: every CTA leaves its partial tile in its shared
// memory and adds its peers' to its share of the rows, from the next rank on
// and around.  Where clusters would not all fit the GPU at once, two of them
// may halve a tile's K and meet in global memory instead (the 36 tiles of a
// 2048-row X X^T are 72 pairs of 74; as 36 clusters of 4 they were two waves).
//
// What bounds it.  Large products: the tensor pipe -- the main loop takes 1543
// clocks a block of the 1536 of its MMAs, at the clock the power limit leaves
// (1.4 to 1.5 GHz); a tile's start and epilogue are another 20 thousand clocks,
// and the waves' ends.  4096 x 4096, five steps: 3.9 ms, 1.05 PFLOP/s of MMAs
// done; 2048 x 8192 with its momentum and update: 1.78 ms.  Small products: the
// way through a kernel -- 1.3 us to the first tile, 1.1 for the cluster's meeting,
// 2.5 for the epilogue, 2.2 until the next kernel goes on: 256 x 4096 takes 134
// us for 17 kernels.
#include <algorithm>
#include <cmath>

#include "glm_ortho.cuh"
#include "glm_tc.cuh"

namespace glmb {

namespace {

constexpr int kBM = 128;  // rows of D per CTA
constexpr int kBK = 64;   // K per stage: 128 bytes of binary16, one swizzle row
constexpr int kStages = 3;
constexpr int kPlaneBytes = 128 * kBK * 2;  // 128 rows (or columns) of one plane: 16 KB
constexpr int kStageBytes = 4 * kPlaneBytes;  // left hi, lo, right hi, lo
constexpr int kMaxSplits = 16;  // CTAs of a cluster
constexpr int64_t kMaxHalved = 74;  // CTAs of tiles that may be halved: beyond, whole tiles fill the SMs
constexpr int kDrainWarp0 = 4, kDrainWarps = 8, kDrainThreads = kDrainWarps * 32;
constexpr int kThreads = (kDrainWarp0 + kDrainWarps) * 32;
// 384 threads launch with 168 registers each; the control warpgroup gives its share to the two that drain
constexpr uint32_t kRegsControl = 72, kRegsDrain = 208;
static_assert(128 * kRegsControl + 256 * kRegsDrain <= kThreads * 168, "register split exceeds the launch");

struct GemmSmem {
    alignas(1024) unsigned char stage[kStages][kStageBytes];  // later the float tile
    unsigned long long full[kStages];
    unsigned long long ready[kStages];  // (even CTA of a pair) the odd CTA's copies have landed
    unsigned long long empty[kStages];  // the stage's MMAs have retired: free for the next copies, sums to be drained
    unsigned long long acce[2];
    unsigned long long done;
    uint32_t tmem_base;
    int failed;
    int turn;
};

// D (f32) from binary16 A and B; K-major A, B K- or MN-major.
constexpr uint32_t instr_desc_f16(int M, int N, bool b_mn_major) {
    return (1u << 4) | (uint32_t(b_mn_major) << 16) | (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}

constexpr uint32_t kLayoutSW128 = 2;

template <bool PAIR>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
}

// One arrival on `bar` (in both CTAs of a pair, `mask` their cluster ranks) once the MMAs issued so far retire.
template <bool PAIR>
__device__ __forceinline__ void commit(unsigned long long* bar, uint16_t mask) {
    if constexpr (PAIR)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                saddr(bar)),
            "h"(mask)
            : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(saddr(bar))
                     : "memory");
}

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w,
                                            unsigned long long* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
            "r"(saddr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(saddr(bar))
        : "memory");
}

__device__ __forceinline__ void drain_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kDrainThreads) : "memory"); }

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// v ~ hi + lo of two values
__device__ __forceinline__ void split_half2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = pack_half2(a - f.x, b - f.y);
}

// Four (eight) values at `hi` and their low parts a plane on.
__device__ __forceinline__ void store_split4(__half* hi, int64_t plane, float4 v) {
    uint2 h, l;
    split_half2(v.x, v.y, h.x, l.x);
    split_half2(v.z, v.w, h.y, l.y);
    *reinterpret_cast<uint2*>(hi) = h;
    *reinterpret_cast<uint2*>(hi + plane) = l;
}
__device__ __forceinline__ void store_split8(__half* hi, int64_t plane, const float (&v)[8]) {
    uint4 h, l;
    split_half2(v[0], v[1], h.x, l.x);
    split_half2(v[2], v[3], h.y, l.y);
    split_half2(v[4], v[5], h.z, l.z);
    split_half2(v[6], v[7], h.w, l.w);
    *reinterpret_cast<uint4*>(hi) = h;
    *reinterpret_cast<uint4*>(hi + plane) = l;
}

// Four elements of a row, or as many as are left of it; `whole`: one access.
template <typename T>
__device__ __forceinline__ float4 load4(const T* p, int64_t left, bool whole) {
    alignas(16) T t[4] = {};
    if (whole) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(t) = *reinterpret_cast<const uint4*>(p);
        else *reinterpret_cast<uint2*>(t) = *reinterpret_cast<const uint2*>(p);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left) t[i] = p[i];
    }
    return make_float4(to_arith<float>(t[0]), to_arith<float>(t[1]), to_arith<float>(t[2]), to_arith<float>(t[3]));
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int64_t left, bool whole, float4 v) {
    alignas(16) T t[4] = {from_arith<T>(v.x), from_arith<T>(v.y), from_arith<T>(v.z), from_arith<T>(v.w)};
    if (whole) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(t);
        else *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(t);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left) p[i] = t[i];
    }
}

// kGram: D = A = X X^T and D2 = C = bI + cA;  kPoly: D = B = aI + A C;  kApply: D = B X;  kLast: out from B X.
enum : int { kGram, kPoly, kApply, kLast };

struct GemmArgs {
    int64_t m, n;       // rows and columns of D
    int32_t tiles_m, tiles_n;  // tiles of D (kGram, kPoly: tiles_m of them on a side)
    int32_t units;      // tiles a task has
    int32_t nkb;        // 64-deep blocks of K
    int32_t splits;     // CTAs (pairs) of a cluster, each with its share of K
    int32_t halves;     // 2: two clusters work on a tile, each with half of K (splits is 1 then)
    float4* partial;    // halves == 2: sums of the half that is done first, [tile, CTA of the pair][column / 4][thread]
    int* arrived;       // [tile, CTA of the pair], zero between launches
    float scale;        // of the accumulated sum
    float scale2;       // kGram: of D on its way to D2
    float diag;         // on the diagonal of D2 (kGram) or D (kPoly)
    __half* D;          // planes [task][2][m][ld]
    __half* D2;
    int64_t ld;
    void* out;          // kLast
    bool tall, update;
    bool whole;         // rows of `out` are whole pieces of four elements
    float keep, rate;
    int* status;
};

template <bool PAIR, int KIND, typename T>
__global__ void __launch_bounds__(kThreads, 1)
    ortho_gemm_kernel(const __grid_constant__ CUtensorMap map_left, const __grid_constant__ CUtensorMap map_right,
                      const GemmArgs a) {
    constexpr int kBN = PAIR ? 256 : 128;   // columns of a tile
    constexpr int kBT = PAIR ? 256 : 128;   // rows of a tile (of both CTAs)
    constexpr int kCols = kBN / 2;          // columns a drain thread sums
    constexpr uint32_t kTmemCols = 2 * kBN;
    constexpr int kTileLd = kBN + 4;        // floats; four banks on from row to row
    static_assert(kBM * kTileLd * 4 <= kStages * kStageBytes);
    constexpr bool kSym = KIND == kGram || KIND == kPoly;

    extern __shared__ __align__(1024) unsigned char smem_raw[];
    GemmSmem& sm = *reinterpret_cast<GemmSmem*>(
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023)));
    const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31;
    const uint32_t rank = cluster_rank();
    const uint32_t half = PAIR ? (rank & 1) : 0;          // which CTA of the pair
    const uint32_t part = PAIR ? (rank >> 1) : rank;      // which share of K
    const uint32_t lead = PAIR ? (rank & ~1u) : rank;     // the CTA that issues the MMAs
    const int csize = a.splits * (PAIR ? 2 : 1);

    const int64_t cluster = blockIdx.x / csize / a.halves;
    const int share_of = a.halves == 1 ? int(part) : int(blockIdx.x / csize % 2), shares = a.splits * a.halves;
    const int64_t task = cluster / a.units;
    const int u = int(cluster % a.units);
    int ti, tj;
    if constexpr (kSym) {
        // u counts the tiles (ti <= tj) column by column: u = tj (tj + 1) / 2 + ti
        tj = int((sqrtf(8.0f * float(u) + 1.0f) - 1.0f) * 0.5f);
        while (tj * (tj + 1) / 2 > u) --tj;
        while ((tj + 1) * (tj + 2) / 2 <= u) ++tj;
        ti = u - tj * (tj + 1) / 2;
    } else {
        // bands of eight tile rows, walked column by column: tiles that run together share both operands
        const int band = u / (8 * a.tiles_n), first = band * 8, rows = min(8, a.tiles_m - first);
        const int in = u - band * 8 * a.tiles_n;
        ti = first + in % rows;
        tj = in / rows;
    }
    const int m0 = ti * kBT + int(half) * kBM;       // this CTA's rows of D
    const int n0 = tj * kBN;
    const int nb0 = n0 + int(half) * 128;            // the columns this CTA stages
    // this CTA's share of K
    const int kb0 = int(int64_t(a.nkb) * share_of / shares), kb1 = int(int64_t(a.nkb) * (share_of + 1) / shares);
    const int nkb = kb1 - kb0;

    if (tid == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_left) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_right) : "memory");
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.ready[s], 1);
            mbar_init(&sm.empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) mbar_init(&sm.acce[b], (PAIR ? 2 : 1) * kDrainWarps);
        mbar_init(&sm.done, 1);
        sm.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(&sm.tmem_base)),
                         "r"(kTmemCols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(&sm.tmem_base)),
                         "r"(kTmemCols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (csize > 1) cluster_sync_relaxed();  // the peers' barriers exist before anyone arrives on them
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem_base, 0);
    volatile int* failed = &sm.failed;
    float* tile = reinterpret_cast<float*>(sm.stage[0]);
    bool finish = true;  // this CTA has (its rows of) the whole sum
    pdl_allow_dependents();
    pdl_wait_for_producer();

    if (warp < kDrainWarp0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));
        if (warp == 0 && lane == 0) {
            int issued = 0;
            for (int kb = 0; kb < nkb; ++kb) {
                const int s = kb % kStages;
                if (kb >= kStages && !mbar_wait(&sm.empty[s], uint32_t((kb / kStages - 1) & 1), failed)) break;
                unsigned char* st = sm.stage[s];
                const int k = (kb0 + kb) * kBK;
                mbar_expect_tx(&sm.full[s], kStageBytes);
                tma_load_4d(st, &map_left, k, m0, 0, int(task), &sm.full[s]);
                if constexpr (kSym) {
                    tma_load_4d(st + 2 * kPlaneBytes, &map_right, k, nb0, 0, int(task), &sm.full[s]);
                } else {
                    // two atoms of 64 columns x 64 rows of X, hi and lo each
                    tma_load_4d(st + 2 * kPlaneBytes, &map_right, nb0, k, 0, int(task), &sm.full[s]);
                    tma_load_4d(st + 3 * kPlaneBytes, &map_right, nb0 + 64, k, 0, int(task), &sm.full[s]);
                }
                issued = kb + 1;
            }
            // the copies still in flight land before shared memory is used for anything else
            for (int kb = issued > kStages ? issued - kStages : 0; kb < issued; ++kb)
                mbar_wait(&sm.full[kb % kStages], uint32_t((kb / kStages) & 1), nullptr);
        } else if (warp == 1) {
            if (rank == lead) {
                constexpr uint32_t idesc = instr_desc_f16(kBT, kBN, !kSym);
                const uint16_t mask = uint16_t(PAIR ? 3u << lead : 0u);
                const uint32_t left0 = desc_address(saddr(sm.stage[0]), 16);
                const uint32_t right0 = desc_address(saddr(sm.stage[0]) + 2 * kPlaneBytes, kSym ? 16 : kPlaneBytes);
                for (int kb = 0; kb < nkb; ++kb) {
                    const int s = kb % kStages, buf = kb & 1;
                    if (kb >= 2 && !mbar_wait_warp(&sm.acce[buf], uint32_t(((kb >> 1) - 1) & 1), failed)) break;
                    if (!mbar_wait_warp(&sm.full[s], uint32_t((kb / kStages) & 1), failed)) break;
                    if (PAIR && !mbar_wait_warp(&sm.ready[s], uint32_t((kb / kStages) & 1), failed)) break;
                    tc_fence_after();
                    const uint32_t d = tmem + uint32_t(buf * kBN);
                    const bool elected = elect_one();
                    // K-major: 16 binary16 = 32 bytes on along the row; 8-row groups 1024 bytes apart.
                    // MN-major: 16 K-rows of 128 bytes on; 8-row groups 1024 bytes, 64-column atoms (hi and lo of
                    // one, then of the next) a plane apart.
                    constexpr uint32_t kRest = desc_rest(1024, kLayoutSW128);
                    const uint32_t lh = left0 + uint32_t(s) * (kStageBytes >> 4), ll = lh + (kPlaneBytes >> 4);
                    const uint32_t rh = right0 + uint32_t(s) * (kStageBytes >> 4),
                                   rl = rh + ((kSym ? kPlaneBytes : kPlaneBytes / 2) >> 4);
                    constexpr uint32_t kRight = (kSym ? 32 : 2048) >> 4;
                    if (elected) {
#pragma unroll
                        for (int k = 0; k < kBK / 16; ++k) {
                            const uint64_t r = desc_join(rh + k * kRight, kRest);
                            mma_f16<PAIR>(d, desc_join(ll + 2 * k, kRest), r, idesc, k > 0 ? 1u : 0u);
                            mma_f16<PAIR>(d, desc_join(lh + 2 * k, kRest), desc_join(rl + k * kRight, kRest), idesc, 1u);
                        }
#pragma unroll
                        for (int k = 0; k < kBK / 16; ++k)
                            mma_f16<PAIR>(d, desc_join(lh + 2 * k, kRest), desc_join(rh + k * kRight, kRest), idesc, 1u);
                        commit<PAIR>(&sm.empty[s], mask);
                    }
                    __syncwarp();
                }
                if (elect_one()) commit<PAIR>(&sm.done, mask);
                __syncwarp();
                // no CTA leaves while a draining warp's arrival is on its way to it
                for (int b = 0; b < 2 && b < nkb; ++b)
                    mbar_wait_warp(&sm.acce[b], uint32_t(((nkb - b + 1) / 2 - 1) & 1), failed);
            }
            mbar_wait_warp(&sm.done, 0, nullptr);
        } else if (PAIR && warp == 2 && lane == 0 && rank != lead) {
            // tells the even CTA that this CTA's copies of a stage have landed
            for (int kb = 0; kb < nkb; ++kb) {
                const int s = kb % kStages;
                if (!mbar_wait(&sm.full[s], uint32_t((kb / kStages) & 1), failed)) break;
                fence_proxy_async();
                mbar_arrive_rank(&sm.ready[s], lead);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsDrain));
        const int quarter = warp & 3, side = (warp - kDrainWarp0) >> 2;
        const uint32_t tbase = tmem + (uint32_t(32 * quarter) << 16) + uint32_t(side * kCols);
        float sum[kCols];
#pragma unroll
        for (int i = 0; i < kCols; ++i) sum[i] = 0.0f;
        bool ok = true;
        for (int kb = 0; kb < nkb; ++kb) {
            // (the stage cannot come round again unseen: its next MMAs wait for this block's drain)
            const int buf = kb & 1;
            if (!(ok = mbar_wait_warp(&sm.empty[kb % kStages], uint32_t((kb / kStages) & 1), failed))) break;
            tc_fence_after();
#pragma unroll
            for (int h = 0; h < kCols / 32; ++h) {
                uint32_t r[2][16];
                tmem_ld16(tbase + uint32_t(buf * kBN + 32 * h), r[0]);
                tmem_ld16(tbase + uint32_t(buf * kBN + 32 * h + 16), r[1]);
                tmem_wait_ld(r[0]);
                reg_after(r[1]);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < 16; ++i) sum[32 * h + 16 * j + i] += __uint_as_float(r[j][i]);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_rank(&sm.acce[buf], lead);
        }
        if (a.halves == 2) {
            // Both halves leave their sums in global memory; the one that is there last (nobody waits) adds the
            // other's to its own -- two summands, so the order does not matter -- and goes on alone.
            if (!ok) {
#pragma unroll
                for (int i = 0; i < kCols; ++i) sum[i] = __int_as_float(0x7fc00000);
                ok = true;
            }
            const int64_t which = cluster * (PAIR ? 2 : 1) + half;
            const int dt = threadIdx.x - kDrainWarp0 * 32;
            float4* const slot = a.partial + which * 2 * (kCols / 4) * kDrainThreads + dt;
#pragma unroll
            for (int i = 0; i < kCols; i += 4)
                slot[(share_of * (kCols / 4) + i / 4) * kDrainThreads] =
                    make_float4(sum[i], sum[i + 1], sum[i + 2], sum[i + 3]);
            __threadfence();
            drain_sync();
            if (dt == 0) sm.turn = atomicAdd(&a.arrived[which], 1);
            drain_sync();
            finish = sm.turn == 1;
            if (finish) {
                if (dt == 0) a.arrived[which] = 0;  // for the next launch
                __threadfence();
#pragma unroll
                for (int i = 0; i < kCols; i += 4) {
                    const float4 v = __ldcg(slot + ((share_of ^ 1) * (kCols / 4) + i / 4) * kDrainThreads);
                    sum[i] += v.x;
                    sum[i + 1] += v.y;
                    sum[i + 2] += v.z;
                    sum[i + 3] += v.w;
                }
            }
        }
        // every copy has landed and every MMA of this CTA's stages has retired: the stages become the tile
        if (ok && finish) {
            float* row = tile + (32 * quarter + lane) * kTileLd + side * kCols;
#pragma unroll
            for (int i = 0; i < kCols; i += 4)
                *reinterpret_cast<float4*>(row + i) = make_float4(sum[i], sum[i + 1], sum[i + 2], sum[i + 3]);
        }
    }
    __syncwarp();  // the role warps worked with one lane
    tc_fence_before();
    __syncthreads();
    if (csize > 1) cluster_sync();  // the peers' partial tiles are complete

    if (warp >= kDrainWarp0 && finish) {
        const int share = kBM / a.splits;  // rows of the tile this CTA finishes
        const int r0 = int(part) * share;
        const bool mirror = kSym && ti != tj;
        bool bad = false;
        if constexpr (KIND == kLast) {
            bad = *static_cast<volatile int*>(a.status) != 0;
            for (int p = 0; p < csize; ++p) bad |= ld_cluster_s32(&sm.failed, p) != 0;
        }
        // Four columns to a thread, every kRowsAtOnce-th row.  The loops here are kept rolled: this code runs once
        // per tile, and straight-line code costs an instruction fetch from L2 every eight instructions.
        const int dt = threadIdx.x - kDrainWarp0 * 32;
        constexpr int kRowsAtOnce = kDrainThreads * 4 / kBN;
        const int c = 4 * (dt % (kBN / 4)), col = n0 + c, rt = r0 + dt / (kBN / 4);
        // The peers' partial sums onto this CTA's own, from the next rank on and around; eight loads in flight.
        if (a.splits > 1) {
            constexpr int kTogether = 8;
            const int items_log2 = 31 - __clz(share / kRowsAtOnce), loads = (a.splits - 1) << items_log2;
            const uint32_t at = saddr(tile + rt * kTileLd + c);
#pragma unroll 1
            for (int i = 0; i < loads; i += kTogether) {
                float4 q[kTogether];
#pragma unroll
                for (int j = 0; j < kTogether; ++j)
                    if (i + j < loads) {
                        const uint32_t peer = (part + 1u + uint32_t((i + j) >> items_log2)) & uint32_t(a.splits - 1);
                        const int row = ((i + j) & ((1 << items_log2) - 1)) * kRowsAtOnce;
                        q[j] = ld_cluster_f4(mapa(at + uint32_t(row * kTileLd * 4), PAIR ? 2 * peer + half : peer));
                    }
#pragma unroll
                for (int j = 0; j < kTogether; ++j)
                    if (i + j < loads) {
                        const int row = ((i + j) & ((1 << items_log2) - 1)) * kRowsAtOnce;
                        float4* const to = reinterpret_cast<float4*>(tile + (rt + row) * kTileLd + c);
                        const float4 v = *to;
                        *to = make_float4(v.x + q[j].x, v.y + q[j].y, v.z + q[j].z, v.w + q[j].w);
                    }
            }
        }
        // the operator's own arithmetic, in place, and the output as the rows lie
        T* const out = KIND == kLast ? static_cast<T*>(a.out) + task * a.m * a.n : nullptr;
        constexpr int kUnroll = KIND == kLast ? 4 : 2;
#pragma unroll 1
        for (int rr = rt; rr < r0 + share; rr += kUnroll * kRowsAtOnce) {
            [[maybe_unused]] float4 old[kUnroll];
            if constexpr (KIND == kLast) {
                if (a.update && !a.tall) {
#pragma unroll
                    for (int j = 0; j < kUnroll; ++j) {
                        const int row = m0 + rr + j * kRowsAtOnce;
                        if (row < a.m && col < a.n) old[j] = load4(out + int64_t(row) * a.n + col, a.n - col, a.whole);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) {
                const int r = rr + j * kRowsAtOnce, row = m0 + r;
                if (r >= r0 + share) break;
                float4 v = *reinterpret_cast<const float4*>(tile + r * kTileLd + c);
                v.x = fmaf(v.x, a.scale, KIND == kPoly && row == col ? a.diag : 0.0f);
                v.y = fmaf(v.y, a.scale, KIND == kPoly && row == col + 1 ? a.diag : 0.0f);
                v.z = fmaf(v.z, a.scale, KIND == kPoly && row == col + 2 ? a.diag : 0.0f);
                v.w = fmaf(v.w, a.scale, KIND == kPoly && row == col + 3 ? a.diag : 0.0f);
                if constexpr (KIND == kLast) {
                    if (a.tall) {
                        *reinterpret_cast<float4*>(tile + r * kTileLd + c) = v;
                    } else if (row < a.m && col < a.n) {
                        if (a.update) {
                            v.x = fmaf(-a.rate, v.x, a.keep * old[j].x);
                            v.y = fmaf(-a.rate, v.y, a.keep * old[j].y);
                            v.z = fmaf(-a.rate, v.z, a.keep * old[j].z);
                            v.w = fmaf(-a.rate, v.w, a.keep * old[j].w);
                        }
                        if (bad) v.x = v.y = v.z = v.w = __int_as_float(0x7fc00000);
                        store4(out + int64_t(row) * a.n + col, a.n - col, a.whole, v);
                    }
                } else {
                    if (row < a.m && col < a.ld) {
                        const int64_t at = (task * 2 * a.m + row) * a.ld + col;
                        store_split4(a.D + at, a.m * a.ld, v);
                        if constexpr (KIND == kGram) {
                            const float4 w = make_float4(
                                fmaf(v.x, a.scale2, row == col ? a.diag : 0.0f),
                                fmaf(v.y, a.scale2, row == col + 1 ? a.diag : 0.0f),
                                fmaf(v.z, a.scale2, row == col + 2 ? a.diag : 0.0f),
                                fmaf(v.w, a.scale2, row == col + 3 ? a.diag : 0.0f));
                            store_split4(a.D2 + at, a.m * a.ld, w);
                        }
                    }
                    if (mirror) *reinterpret_cast<float4*>(tile + r * kTileLd + c) = v;
                }
            }
        }
        const bool across = KIND == kLast ? a.tall : mirror;  // the tile is needed column by column too
        if (across) drain_sync();
        if constexpr (kSym) {
            if (mirror) {
                // eight rows of one column to a thread: 16 bytes of a row of the mirror image
#pragma unroll 1
                for (int i = dt; i < kBN * (share / 8); i += kDrainThreads) {
                    const int c = i % kBN, r = r0 + i / kBN * 8;
                    const int row = n0 + c, col = m0 + r;  // of the mirror image
                    if (row >= a.m || col >= a.ld) continue;
                    float v[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] = tile[(r + k) * kTileLd + c];
                    const int64_t at = (task * 2 * a.m + row) * a.ld + col;
                    store_split8(a.D + at, a.m * a.ld, v);
                    if constexpr (KIND == kGram) {
#pragma unroll
                        for (int k = 0; k < 8; ++k) v[k] *= a.scale2;  // off the diagonal
                        store_split8(a.D2 + at, a.m * a.ld, v);
                    }
                }
            }
        }
        if constexpr (KIND == kLast) {
            if (a.tall) {
                const int share_log2 = 31 - __clz(share);
                constexpr int kAhead = 4;  // share * kBN is a multiple of 4 * kDrainThreads
#pragma unroll 1
                for (int i0 = dt; i0 < share * kBN; i0 += kAhead * kDrainThreads) {
                    float old[kAhead];
                    if (a.update) {
#pragma unroll
                        for (int j = 0; j < kAhead; ++j) {
                            const int i = i0 + j * kDrainThreads;
                            const int64_t row = m0 + r0 + (i & (share - 1)), col = n0 + (i >> share_log2);
                            old[j] = row < a.m && col < a.n ? to_arith<float>(out[col * a.m + row]) : 0.0f;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < kAhead; ++j) {
                        // neighbouring threads on neighbouring rows, which lie side by side in the output
                        const int i = i0 + j * kDrainThreads, r = r0 + (i & (share - 1)), c = i >> share_log2;
                        const int64_t row = m0 + r, col = n0 + c;
                        if (row >= a.m || col >= a.n) continue;
                        float v = tile[r * kTileLd + c];
                        if (a.update) v = fmaf(-a.rate, v, a.keep * old[j]);
                        out[col * a.m + row] = from_arith<T>(bad ? __int_as_float(0x7fc00000) : v);
                    }
                }
            }
        }
    }
    __syncwarp();  // the role warps worked with one lane
    tc_fence_before();
    __syncthreads();
    if (csize > 1) cluster_sync_relaxed();  // no read of a peer's shared memory is outstanding
    if (warp == 1) {
        tc_fence_after();
        if constexpr (PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
    if (tid == 0 && sm.failed) atomicExch(a.status, 1);
}

// Planes [task][2][rows][ld] as a 4-D map of their `cols` valid columns; box 64 columns x box_rows x both planes.
bool plane_map(CUtensorMap* map, const __half* base, int64_t cols, int64_t rows, int64_t ld, int64_t ntasks,
               int box_rows) {
    auto fn = tensor_map_encoder();
    if (fn == nullptr) return false;
    const cuuint64_t dims[4] = {cuuint64_t(cols), cuuint64_t(rows), 2, cuuint64_t(ntasks)};
    const cuuint64_t strides[3] = {cuuint64_t(ld) * 2, cuuint64_t(rows * ld) * 2, cuuint64_t(2 * rows * ld) * 2};
    const cuuint32_t box[4] = {kBK, cuuint32_t(box_rows), 2, 1}, one[4] = {1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<__half*>(base), dims, strides, box, one,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How a product is cut: the shape of its tiles and the shares of K.
struct Cut {
    bool pair;
    int splits, halves;
    int64_t tiles_m, tiles_n, units;
};

// Clusters of `csize` CTAs, one to an SM, that the device holds at once: the SMs of a GPC come in numbers that
// larger clusters do not divide (148 SMs hold 74 clusters of 2, 33 of 4, 15 of 8 and 7 of 16).
int64_t clusters_at_once(int csize) {
    static std::atomic<int> known[64][5];
    int dev = 0, log2 = 0;
    while ((1 << log2) < csize) ++log2;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return csize > 8 ? 0 : std::max(1, sm_count() / csize);
    int n = known[dev][log2].load(std::memory_order_relaxed);
    if (n == 0) {
        auto kernel = ortho_gemm_kernel<false, kGram, float>;
        static std::atomic<uint64_t> attr{0};
        const size_t smem = sizeof(GemmSmem) + 1024;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(unsigned(csize));
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = unsigned(csize);
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        if (set_smem_limit_once(attr, kernel, smem) != cudaSuccess ||
            (csize > 8 && cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) ||
            cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
            (void)cudaGetLastError();
            n = csize > 8 ? 0 : std::max(1, sm_count() / csize * 7 / 8);
        }
        known[dev][log2].store(n == 0 ? -1 : n, std::memory_order_relaxed);
    }
    return std::max(n, 0);
}

// The cut with the least estimated time, in clocks: waves of clusters over the
// SMs times (blocks of K per share + what a tile costs besides).  A pair's
// block is its 12 MMAs of 128 clocks; a single CTA's 12 MMAs of half that
// size take hardly less (1390 measured).
Cut cut_product(int64_t m, int64_t n, int64_t nkb, int64_t ntasks, bool sym) {
    Cut best{};
    double least = 0.0;
    for (const bool pair : {true, false}) {
        const int64_t bt = pair ? 256 : 128, tm = (m + bt - 1) / bt, tn = (n + bt - 1) / bt;
        const int64_t units = sym ? tm * (tm + 1) / 2 : tm * tn;
        for (int shares = 1; shares <= (pair ? kMaxSplits / 4 : kMaxSplits); shares *= 2) {
            if (shares > 1 && nkb < 2 * shares) break;
            for (int halves = 1; halves <= 2; ++halves) {
                // two halves of a tile meet in global memory: only for few tiles, whose partial sums stay small
                if (halves == 2 && (shares != 2 || units * ntasks * (pair ? 2 : 1) > kMaxHalved)) continue;
                const int splits = shares / halves;
                const int64_t at_once = clusters_at_once(splits * (pair ? 2 : 1));
                if (at_once == 0) continue;
                const int64_t waves = (units * ntasks * halves + at_once - 1) / at_once;
                const double block = pair ? 1550.0 : 1390.0;
                const double tile = 4500.0 + (pair ? 10000.0 : 5000.0) / splits + (splits > 1 ? 2500.0 : 0.0) +
                                    (halves > 1 ? (pair ? 5000.0 : 2500.0) : 0.0);
                const double t = double(waves) * (double((nkb + shares - 1) / shares) * block + tile);
                if (least == 0.0 || t < least) {
                    least = t;
                    best = Cut{pair, splits, halves, tm, tn, units};
                }
            }
        }
    }
    return best;
}

template <bool PAIR, int KIND, typename T>
cudaError_t launch_gemm(const CUtensorMap& left, const CUtensorMap& right, const GemmArgs& args, int64_t ntasks,
                        cudaStream_t stream) {
    static std::atomic<uint64_t> attr{0};
    const size_t smem = sizeof(GemmSmem) + 1024;
    auto kernel = ortho_gemm_kernel<PAIR, KIND, T>;
    cudaError_t e = set_smem_limit_once(attr, kernel, smem);
    if (e != cudaSuccess) return e;
    const int csize = args.splits * (PAIR ? 2 : 1);
    if (csize > 8) {
        static std::atomic<uint64_t> wide{0};
        int dev = 0;
        if ((e = cudaGetDevice(&dev)) != cudaSuccess) return e;
        const uint64_t bit = dev >= 0 && dev < 64 ? uint64_t(1) << dev : 0;
        if (bit == 0 || (wide.load(std::memory_order_acquire) & bit) == 0) {
            if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess) return e;
            wide.fetch_or(bit, std::memory_order_release);
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(int64_t(args.units) * ntasks * csize * args.halves));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = unsigned(csize);
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    count_launch();
    return cudaLaunchKernelEx(&cfg, kernel, left, right, args);
}

template <int KIND, typename T>
cudaError_t launch_cut(const Cut& cut, const CUtensorMap& left, const CUtensorMap& right, GemmArgs args, int64_t ntasks,
                       cudaStream_t stream) {
    args.tiles_m = int32_t(cut.tiles_m);
    args.tiles_n = int32_t(cut.tiles_n);
    args.units = int32_t(cut.units);
    args.splits = cut.splits;
    args.halves = cut.halves;
    return cut.pair ? launch_gemm<true, KIND, T>(left, right, args, ntasks, stream)
                    : launch_gemm<false, KIND, T>(left, right, args, ntasks, stream);
}

// The largest power of two that keeps `bound` times it within 2^15 (binary16 ends at 65504).
float scale_for(double bound) { return float(std::exp2(15.0 - std::ceil(std::log2(std::max(bound, 1e-3))))); }

}  // namespace

namespace {
struct Cuts {
    Cut gram, poly, apply;
    Cuts(int64_t m, int64_t n, int64_t ntasks)
        : gram(cut_product(m, m, (n + kBK - 1) / kBK, ntasks, true)),
          poly(cut_product(m, m, (m + kBK - 1) / kBK, ntasks, true)),
          apply(cut_product(m, n, (m + kBK - 1) / kBK, ntasks, false)) {}
};
}  // namespace

// What any cut of the three products may take, whatever clusters the device holds: the size a caller asked for
// while another device was current has to do.
size_t ortho_partial_bytes(int64_t m, int64_t n, int64_t ntasks) {
    const int64_t kbn = (n + kBK - 1) / kBK, kbm = (m + kBK - 1) / kBK;
    size_t most = 0;
    for (const bool pair : {true, false})
        for (int product = 0; product < 3; ++product) {
            const int64_t bt = pair ? 256 : 128, tm = (m + bt - 1) / bt, tn = (n + bt - 1) / bt;
            const int64_t ctas = (product < 2 ? tm * (tm + 1) / 2 : tm * tn) * ntasks * (pair ? 2 : 1);
            if (ctas <= kMaxHalved && (product == 0 ? kbn : kbm) >= 4)
                most = std::max(most, size_t(ctas) * 2 * 128 * (pair ? 256 : 128) * sizeof(float));
        }
    return most;
}
size_t ortho_arrived_bytes() { return size_t(kMaxHalved) * sizeof(int); }

float ortho_x_scale(const OrthoStep& s) { return scale_for(s.x_max); }

template <typename T>
int ortho_products(const OrthoPlanes& p, const OrthoSteps& steps, T* out, bool tall, const OrthoUpdate* up, int* status,
                   cudaStream_t stream) {
    const int64_t m = p.m, n = p.n;
    const int64_t kbn = (n + kBK - 1) / kBK, kbm = (m + kBK - 1) / kBK;
    const Cuts cuts(m, n, p.ntasks);
    const Cut &gram = cuts.gram, &poly = cuts.poly, &apply = cuts.apply;
    for (const Cut& c : {gram, poly, apply})
        if (c.units * p.ntasks > (int64_t(1) << 27)) return GLMB_ERR_TOO_LARGE;
    CUtensorMap x_rows[2], x_cols[2], a_rows, b_rows, c_rows;
    for (int i = 0; i < 2; ++i)
        if (!plane_map(&x_rows[i], p.X[i], n, m, p.ld_n, p.ntasks, 128) ||
            !plane_map(&x_cols[i], p.X[i], n, m, p.ld_n, p.ntasks, 64))
            return GLMB_ERR_UNSUPPORTED;
    if (!plane_map(&a_rows, p.A, m, m, p.ld_m, p.ntasks, 128) || !plane_map(&b_rows, p.B, m, m, p.ld_m, p.ntasks, 128) ||
        !plane_map(&c_rows, p.C, m, m, p.ld_m, p.ntasks, 128))
        return GLMB_ERR_UNSUPPORTED;
    for (int k = 0; k < steps.n; ++k) {
        const OrthoStep& s = steps.step[k];
        const float sx = ortho_x_scale(s), sa = scale_for(s.x_max * s.x_max), sb = scale_for(s.b_max),
                    sc = scale_for(std::fabs(s.b) + std::fabs(s.c) * s.x_max * s.x_max);
        const int cur = k & 1;
        const bool last = k + 1 == steps.n;
        GemmArgs g{};
        g.status = status;
        g.partial = p.partial;
        g.arrived = p.arrived;
        g.m = g.n = m;
        g.nkb = int32_t(kbn);
        g.scale = sa / (sx * sx);
        g.scale2 = s.c * sc / sa;
        g.diag = s.b * sc;
        g.D = p.A;
        g.D2 = p.C;
        g.ld = p.ld_m;
        cudaError_t e = launch_cut<kGram, float>(gram, x_rows[cur], x_rows[cur], g, p.ntasks, stream);
        if (e != cudaSuccess) return int(e);
        g.nkb = int32_t(kbm);
        g.scale = sb / (sa * sc);
        g.diag = s.a * sb;
        g.D = p.B;
        g.D2 = nullptr;
        if ((e = launch_cut<kPoly, float>(poly, a_rows, c_rows, g, p.ntasks, stream)) != cudaSuccess) return int(e);
        g.n = n;
        g.ld = p.ld_n;
        if (!last) {
            g.D = p.X[cur ^ 1];
            g.scale = ortho_x_scale(steps.step[k + 1]) / (sb * sx);
            e = launch_cut<kApply, float>(apply, b_rows, x_cols[cur], g, p.ntasks, stream);
        } else {
            g.D = nullptr;
            g.scale = 1.0f / (sb * sx);
            g.out = out;
            g.tall = tall;
            g.whole = n % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & (4 * sizeof(T) - 1)) == 0;
            g.update = up != nullptr;
            if (up != nullptr) {
                g.keep = up->keep;
                g.rate = up->rate;
            }
            e = launch_cut<kLast, T>(apply, b_rows, x_cols[cur], g, p.ntasks, stream);
        }
        if (e != cudaSuccess) return int(e);
    }
    return launch_status();
}

template int ortho_products<float>(const OrthoPlanes&, const OrthoSteps&, float*, bool, const OrthoUpdate*, int*,
                                   cudaStream_t);
template int ortho_products<__half>(const OrthoPlanes&, const OrthoSteps&, __half*, bool, const OrthoUpdate*, int*,
                                    cudaStream_t);
template int ortho_products<__nv_bfloat16>(const OrthoPlanes&, const OrthoSteps&, __nv_bfloat16*, bool,
                                           const OrthoUpdate*, int*, cudaStream_t);

}  // namespace glmb
