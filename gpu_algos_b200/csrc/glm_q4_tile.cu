// glm_q4_tile.cu -- prediction from 4-bit models for many observations, on the
// 5th-generation tensor cores.
//
// A CTA pair (cta_group::2) computes 256 targets x N observations (N = 32 to
// 256): the codes are the 256-row operand, made into whole numbers of X's
// 16-bit type on their way into shared memory by eight warps of each CTA, so
// the weights cross L2 and HBM as half a byte; X comes by TMA, each CTA
// staging half of the observations.  Products of 16-bit values are exact.
// Each group of features is accumulated from zero in one of two TMEM buffers
// and added, times the group's scale (one per target, which is one per thread
// of the eight draining warps), to float registers: the scale multiplies a sum
// of whole-number products and no weight is ever rounded.
// float observations are three bfloat16 terms with products of their own.
// Few tiles share the features out over two pairs of a cluster; their partial
// sums meet in distributed shared memory in rank order.
//
// What bounds it.  128 features at N = 256 are eight MMAs of 128 clocks; they
// take about 1350: making the operands (two blocks of codes by each warp, 800 to
// 1000 clocks), draining (640) and issuing the MMAs all run beside each other.
// At small N an MMA still takes its 256 rows about 85 clocks.  16384 targets x
// 4096 features, bfloat16: 20.4 us at 17 observations, 24 at 128, 231 at 2048
// while the clock is at 1965 MHz (1.19 PFLOP/s, 0.73 of cuBLAS in a burst); in
// long runs the power limit holds it to 1.6 GHz, 260 to 270 us (0.75 of cuBLAS
// sustained).  Measured and not kept: the operand
// in tensor memory instead of shared memory (it leaves room for N = 192 at
// most: 408 us against 311 then), two sets of making warps (no gain: the MMA
// warp is the longest path at small N), four pairs to a cluster (clusters of
// eight CTAs do not all fit the GPU at once: 25 us against 18 at 16 x 4096 x 4096).
#include <algorithm>

#include "glm_q4_device.cuh"
#include "glm_tc.cuh"

namespace glmb {

namespace {

constexpr int kBM = 128;  // targets per CTA
constexpr int kBK = 64;   // features of a block of codes: one 128-byte swizzle row
constexpr int kATileBytes = kBM * kBK * 2;
constexpr int kDrainWarp0 = 4, kDrainWarps = 8;
constexpr int kMakeWarp0 = kDrainWarp0 + kDrainWarps, kMakeWarps = 8;  // a row block of the tile each
constexpr int kThreads = (kMakeWarp0 + kMakeWarps) * 32;
constexpr int kMakeAhead = 4;  // blocks of codes in flight per warp (whole stages)
constexpr int kMaxSplits = 2;  // pairs of a cluster
// 640 threads launch with 96 registers each; control and making warps give to those that drain
constexpr uint32_t kRegsControl = 40, kRegsDrain = 168, kRegsMake = 48;
static_assert(128 * kRegsControl + 256 * kRegsDrain + 256 * kRegsMake <= kThreads * 96, "register split");

template <typename T, int N>
struct TileShape {
    static constexpr int kTerms = Split16<T>::kTerms;
    // blocks per stage: two, so that handing a stage over (a proxy fence and an arrival, by every warp that
    // makes operands) is paid half as often; the three terms of a float X leave room for one
    static constexpr int kSub = kTerms == 1 ? 2 : 1;
    static constexpr int kXTermBytes = N / 2 * kBK * 2;  // this CTA's observations, one term
    static constexpr int kXBytes = kTerms * kXTermBytes;
    static constexpr int kStageBytes = kSub * (kATileBytes + kXBytes);  // operands, then X, block by block
    static constexpr int kStages = std::min(8, 192 * 1024 / kStageBytes);
    static constexpr int kCols = N / 2;  // observations a draining thread sums
};

template <typename T, int N>
struct TileSmem {
    using S = TileShape<T, N>;
    alignas(1024) unsigned char stage[S::kStages][S::kStageBytes];  // later the partial sums
    unsigned long long xfull[S::kStages];  // this CTA's X has landed
    unsigned long long ready[S::kStages];  // (even CTA) X and operands of both CTAs are there
    unsigned long long empty[S::kStages];  // the stage's MMAs have retired
    unsigned long long accf;               // the first block's, where a stage holds two groups of features
    unsigned long long acce[2];
    unsigned long long done;
    uint32_t tmem_base;
    int failed;
};

template <typename H>
constexpr uint32_t instr_desc_16(int M, int N) {
    const uint32_t fmt = std::is_same_v<H, __half> ? 0u : 1u;  // binary16 or bfloat16, both operands
    return (1u << 4) | (fmt << 7) | (fmt << 10) | (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}

__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void commit_pair(unsigned long long* bar, uint16_t mask) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            saddr(bar)),
        "h"(mask)
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

// a += s x, b += s y in one instruction
__device__ __forceinline__ void fma_pair(float& a, float& b, float s, float x, float y) {
    asm("{\n\t.reg .b64 p, q, r;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %2};\n\tmov.b64 r, {%3, %4};\n\t"
        "fma.rn.f32x2 p, q, r, p;\n\tmov.b64 {%0, %1}, p;\n\t}"
        : "+f"(a), "+f"(b)
        : "f"(s), "f"(x), "f"(y));
}

struct TileArgs {
    int64_t nt, ntasks, nobs;
    int64_t nrb;
    int ncb, ngroups;
    int tiles_m, tiles_n;
    int splits;
    int group_shift;  // log2 of the 64-feature blocks a group takes
};

template <typename T, int N>
__global__ void __launch_bounds__(kThreads, 1)
    q4_tile_kernel(const __grid_constant__ CUtensorMap map_x, const uint4* __restrict__ codes,
                   const T* __restrict__ scales, T* __restrict__ Yhat, const TileArgs a) {
    using S = TileShape<T, N>;
    using H = typename Split16<T>::Type;
    constexpr int kStages = S::kStages, kCols = S::kCols, kSub = S::kSub;
    constexpr uint32_t kTmemCols = 2 * N;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    TileSmem<T, N>& sm = *reinterpret_cast<TileSmem<T, N>*>(
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023)));
    const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31;
    const uint32_t rank = cluster_rank(), half = rank & 1, part = rank >> 1, lead = rank & ~1u;
    const int csize = 2 * a.splits;
    const int64_t unit = blockIdx.x / unsigned(csize);
    const int tm = int(unit % a.tiles_m);
    const int tn = int(unit / a.tiles_m % a.tiles_n);
    const int64_t task = unit / a.tiles_m / a.tiles_n;
    const int64_t m0 = int64_t(tm) * 256 + half * kBM;  // this CTA's targets
    const int64_t n0 = int64_t(tn) * N;                 // the pair's observations
    // this pair's share of the features, in blocks; whole pairs of blocks, and so whole groups
    const int kb0 = int(int64_t(a.ncb / 2) * part / a.splits) * 2, kb1 = int(int64_t(a.ncb / 2) * (part + 1) / a.splits) * 2;
    const int nkb = kb1 - kb0;
    const int gb = 1 << a.group_shift;  // blocks accumulated together
    const int nst = nkb / kSub;

    if (tid == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&sm.xfull[s], 1);
            mbar_init(&sm.ready[s], 2 * (kMakeWarps + 1));
            mbar_init(&sm.empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) mbar_init(&sm.acce[b], 2 * kDrainWarps);
        mbar_init(&sm.accf, 1);
        mbar_init(&sm.done, 1);
        sm.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(&sm.tmem_base)),
                     "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync_relaxed();  // the peers' barriers exist before anyone arrives on them
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem_base, 0);
    volatile int* failed = &sm.failed;
    float* part_sums = reinterpret_cast<float*>(sm.stage[0]);  // [observation][target]

    if (warp < kDrainWarp0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));
        if (warp == 0 && lane == 0) {
            pdl_wait_for_producer();  // X may be the terms that the kernel before wrote
            int issued = 0;
            for (int st = 0; st < nst; ++st) {
                const int s = st % kStages;
                if (st >= kStages && !mbar_wait(&sm.empty[s], uint32_t((st / kStages - 1) & 1), failed)) break;
                mbar_expect_tx(&sm.xfull[s], kSub * S::kXBytes);
#pragma unroll
                for (int j = 0; j < kSub; ++j)
                    tma_load_4d(sm.stage[s] + kSub * kATileBytes + j * S::kXBytes, &map_x, (kb0 + st * kSub + j) * kBK,
                                int(n0 + half * (N / 2)), int(task), 0, &sm.xfull[s]);
                issued = st + 1;
            }
            // the copies still in flight land before shared memory is used for anything else
            for (int st = issued > kStages ? issued - kStages : 0; st < issued; ++st)
                mbar_wait(&sm.xfull[st % kStages], uint32_t((st / kStages) & 1), nullptr);
        } else if (warp == 1) {
            if (rank == lead) {
                constexpr uint32_t idesc = instr_desc_16<H>(256, N);
                const uint16_t mask = uint16_t(3u << lead);
                const uint32_t stage0 = desc_address(saddr(sm.stage[0]), 16);
                bool ok = true;
                for (int st = 0; st < nst && ok; ++st) {
                    const int s = st % kStages;
                    if (!(ok = mbar_wait_warp(&sm.ready[s], uint32_t((st / kStages) & 1), failed))) break;
#pragma unroll
                    for (int j = 0; j < kSub; ++j) {
                        const int kb = st * kSub + j, grp = kb >> a.group_shift, buf = grp & 1;
                        const bool first = (kb & (gb - 1)) == 0;
                        if (first && grp >= 2 &&
                            !(ok = mbar_wait_warp(&sm.acce[buf], uint32_t(((grp >> 1) - 1) & 1), failed)))
                            break;
                        tc_fence_after();
                        // K-major: 16 features = 32 bytes on along the row; 8-row groups 1024 bytes apart
                        constexpr uint32_t kRest = desc_rest(1024, 2);
                        const uint32_t w = stage0 + uint32_t(s) * (S::kStageBytes >> 4) + j * (kATileBytes >> 4);
                        const uint32_t x = stage0 + uint32_t(s) * (S::kStageBytes >> 4) +
                                           ((kSub * kATileBytes + j * S::kXBytes) >> 4);
                        const uint32_t d = tmem + uint32_t(buf * N);
                        if (elect_one()) {
#pragma unroll
                            for (int q = S::kTerms - 1; q >= 0; --q)
#pragma unroll
                                for (int k = 0; k < kBK / 16; ++k)
                                    mma_pair(d, desc_join(w + 2 * k, kRest),
                                             desc_join(x + q * (S::kXTermBytes >> 4) + 2 * k, kRest), idesc,
                                             q == S::kTerms - 1 && k == 0 ? uint32_t(!first) : 1u);
                            if (j == kSub - 1) commit_pair(&sm.empty[s], mask);
                            else if (gb == 1) commit_pair(&sm.accf, mask);
                        }
                        __syncwarp();
                    }
                }
                if (elect_one()) commit_pair(&sm.done, mask);
                __syncwarp();
                // no CTA leaves while a draining warp's arrival is on its way to it
                const int ngrp = nkb >> a.group_shift;
                for (int b = 0; b < 2 && b < ngrp; ++b)
                    mbar_wait_warp(&sm.acce[b], uint32_t(((ngrp - b + 1) / 2 - 1) & 1), failed);
            }
            mbar_wait_warp(&sm.done, 0, nullptr);
        } else if (warp == 2 && lane == 0) {
            // tells the even CTA that this CTA's copies of a stage have landed
            for (int st = 0; st < nst; ++st) {
                const int s = st % kStages;
                if (!mbar_wait(&sm.xfull[s], uint32_t((st / kStages) & 1), failed)) break;
                fence_proxy_async();
                mbar_arrive_rank(&sm.ready[s], lead);
            }
        }
    } else if (warp < kMakeWarp0) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsDrain));
        const int quarter = warp & 3, side = (warp - kDrainWarp0) >> 2;
        const uint32_t tbase = tmem + (uint32_t(32 * quarter) << 16) + uint32_t(side * kCols);
        const int64_t target = m0 + 32 * quarter + lane;
        const int64_t rb = target / kQ4Rows;
        const bool live = rb < a.nrb;
        const T* sc = scales + ((task * a.nrb + (live ? rb : 0)) * a.ngroups + (kb0 >> a.group_shift)) * kQ4Rows +
                      2 * (target % 8) + target / 8 % 2;
        float sum[kCols];
#pragma unroll
        for (int i = 0; i < kCols; ++i) sum[i] = 0.0f;
        bool ok = true;
        const int ngrp = nkb >> a.group_shift;
        T next = live ? sc[0] : from_arith<T>(0.0f);
        for (int grp = 0; grp < ngrp; ++grp) {
            const int buf = grp & 1;
            const float s = to_arith<float>(next);
            sc += kQ4Rows;
            if (live && grp + 1 < ngrp) next = *sc;
            // A group is complete with its last block's stage (which cannot come round again unseen: its next MMAs
            // wait for this group's drain) or, where two groups share a stage, with the first block.
            const int last = ((grp + 1) << a.group_shift) - 1, st = last / kSub;
            const bool whole = last % kSub == kSub - 1;
            if (!(ok = mbar_wait_warp(whole ? &sm.empty[st % kStages] : &sm.accf,
                                      uint32_t((whole ? st / kStages : grp >> 1) & 1), failed)))
                break;
            tc_fence_after();
            // the next sixteen columns load while these are added
            uint32_t r[2][16];
            tmem_ld16(tbase + uint32_t(buf * N), r[0]);
            tmem_wait_ld(r[0]);
#pragma unroll
            for (int h = 0; h < kCols / 16; ++h) {
                if (h + 1 < kCols / 16) tmem_ld16(tbase + uint32_t(buf * N + 16 * (h + 1)), r[(h + 1) & 1]);
#pragma unroll
                for (int i = 0; i < 16; i += 2)
                    fma_pair(sum[16 * h + i], sum[16 * h + i + 1], s, __uint_as_float(r[h & 1][i]),
                             __uint_as_float(r[h & 1][i + 1]));
                if (h + 1 < kCols / 16) tmem_wait_ld(r[(h + 1) & 1]);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_rank(&sm.acce[buf], lead);
        }
        if (a.splits == 1) {
            // neighbouring lanes on neighbouring targets
            if (target < a.nt) {
                const int64_t first = n0 + side * kCols, step = a.ntasks * a.nt;
                const int left = int(min(int64_t(kCols), a.nobs - first));
                T* to = Yhat + (first * a.ntasks + task) * a.nt + target;
                if (ok) {
#pragma unroll
                    for (int i = 0; i < kCols; ++i) {
                        if (i < left) *to = from_arith<T>(sum[i] * kCodeUp<H>);
                        to += step;
                    }
                } else {
                    for (int i = 0; i < left; ++i, to += step) *to = from_arith<T>(__int_as_float(0x7fc00000));
                }
            }
        } else if (ok) {
#pragma unroll
            for (int i = 0; i < kCols; ++i) part_sums[(side * kCols + i) * kBM + 32 * quarter + lane] = sum[i];
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsMake));
        // ---- a row block's codes into rows 16 r .. of the operand, block after block of features ----
        const int r = warp - kMakeWarp0, g = lane >> 2, c = lane & 3;
        const int64_t rb = m0 / kQ4Rows + r;
        const bool live = rb < a.nrb;  // rows past the last target are not stored and may hold anything
        const uint4* src = codes + ((task * a.nrb + (live ? rb : 0)) * a.ncb + kb0) * 32 + lane;
        // Word k is four features -- eight bytes -- of row g (and of row g + 8) at feature 16 k + 4 c: half of the
        // 16-byte chunk 2 k + c / 2, which the swizzle puts at that number xor g.  Lanes of odd g take the words
        // two on, so that the sixteen lanes of a store meet no bank twice.
        const uint32_t row = uint32_t((16 * r + g) * 128 + 8 * (c & 1));
        const bool odd = (g & 1) != 0;
        uint32_t at[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) at[k] = row + uint32_t(((2 * (k ^ (odd ? 2 : 0)) + (c >> 1)) ^ g) * 16);
        uint4 w[kMakeAhead];
        auto fetch = [&](int kb, uint4& cw) {
            if (live && kb < nkb)
                asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                             : "=r"(cw.x), "=r"(cw.y), "=r"(cw.z), "=r"(cw.w)
                             : "l"(src + int64_t(kb) * 32));
        };
#pragma unroll
        for (int j = 0; j < kMakeAhead; ++j) fetch(j, w[j]);
        bool ok = true;
        int s = 0;
        uint32_t phase = 1;
        constexpr int kRound = kMakeAhead / kSub;  // stages per turn of the loop
        for (int st0 = 0; st0 < nst && ok; st0 += kRound) {
#pragma unroll
            for (int i = 0; i < kRound; ++i) {
                const int st = st0 + i;
                if (st >= nst || !ok) break;
                if (st >= kStages && !(ok = mbar_wait_warp(&sm.empty[s], phase, failed))) break;
                if (live) {
#pragma unroll
                    for (int j = 0; j < kSub; ++j) {
                        unsigned char* tile = sm.stage[s] + j * kATileBytes;
                        uint4& cw = w[i * kSub + j];
                        const uint32_t word[4] = {odd ? cw.z : cw.x, odd ? cw.w : cw.y, odd ? cw.x : cw.z,
                                                  odd ? cw.y : cw.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            uint32_t p[4];
                            code_pairs<H, kCodeDown<H>>(word[k], p);
                            *reinterpret_cast<uint2*>(tile + at[k]) = make_uint2(p[0], p[2]);
                            *reinterpret_cast<uint2*>(tile + at[k] + 8 * 128) = make_uint2(p[1], p[3]);
                        }
                        fetch((st + kRound) * kSub + j, cw);
                    }
                    fence_proxy_async();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive_rank(&sm.ready[s], lead);
                if (++s == kStages) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
    }
    __syncwarp();  // the role warps worked with one lane
    tc_fence_before();
    __syncthreads();
    if (a.splits > 1) {
        cluster_sync();  // the peers' partial sums are complete
        bool bad = false;
        for (int p = 0; p < csize; ++p) bad |= ld_cluster_s32(&sm.failed, p) != 0;
        if (tid < 4 * kBM) {
            // this CTA finishes its share of the observations for its 128 targets
            const int64_t target = m0 + tid % kBM;
            for (int o = int(part) * 4 + tid / kBM; o < N; o += 4 * a.splits) {
                const int64_t obs = n0 + o;
                if (obs >= a.nobs || target >= a.nt) continue;
                float v[kMaxSplits];
#pragma unroll
                for (int p = 0; p < kMaxSplits; ++p)
                    if (p < a.splits) v[p] = ld_cluster_f32(part_sums + o * kBM + tid % kBM, 2 * p + half);
#pragma unroll
                for (int p = 1; p < kMaxSplits; ++p)
                    if (p < a.splits) v[0] += v[p];
                Yhat[(obs * a.ntasks + task) * a.nt + target] = from_arith<T>(bad ? __int_as_float(0x7fc00000) : v[0] * kCodeUp<H>);
            }
        }
    }
    __syncwarp();
    cluster_sync_relaxed();  // no arrival, MMA or read targets a CTA that has left
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

// X as terms [term][obs][task][ld] of the tensor core's type, rows filled up with zeros to ld.
template <typename T>
__global__ void __launch_bounds__(256)
    q4_terms_kernel(const T* __restrict__ X, typename Split16<T>::Type* __restrict__ out, int64_t rows, int64_t nf,
                    int64_t ld, bool vec) {
    constexpr int kTerms = Split16<T>::kTerms;
    pdl_allow_dependents();
    const int64_t pieces = ld / 8, total = rows * pieces;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
        const int64_t row = i / pieces, f = (i - row * pieces) * 8;
        constexpr int kPer = 16 / sizeof(T);
        T x[8];
        if (vec) {  // ld == nf rounded up to 8: the last piece may end at nf, on a whole 16 bytes
#pragma unroll
            for (int e = 0; e < 8; e += kPer) {
                T part[kPer] = {};
                if (f + e < nf) VecLoad<T, kPer>::load(X + row * nf + f + e, part);
#pragma unroll
                for (int j = 0; j < kPer; ++j) x[e + j] = part[j];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = f + e < nf ? X[row * nf + f + e] : from_arith<T>(0.0f);
        }
        alignas(16) typename Split16<T>::Type t[kTerms][8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            typename Split16<T>::Type one[kTerms];
            split_terms<T>(x[e], one);
#pragma unroll
            for (int q = 0; q < kTerms; ++q) t[q][e] = one[q];
        }
#pragma unroll
        for (int q = 0; q < kTerms; ++q)
            *reinterpret_cast<uint4*>(out + (q * rows + row) * ld + f) = *reinterpret_cast<const uint4*>(t[q]);
    }
}

int64_t padded(int64_t nf) { return (nf + 7) / 8 * 8; }

template <typename T, int N>
int launch_tile(const CUtensorMap& map, const void* codes, const T* scales, T* Yhat, const TileArgs& a, bool dependent,
                cudaStream_t stream) {
    const size_t smem = sizeof(TileSmem<T, N>) + 1024;
    static std::atomic<uint64_t> attr{0};
    auto kernel = q4_tile_kernel<T, N>;
    cudaError_t e = set_smem_limit_once(attr, kernel, smem);
    if (e != cudaSuccess) return int(e);
    const int64_t ctas = int64_t(a.tiles_m) * a.tiles_n * a.ntasks * 2 * a.splits;
    if (ctas > 0x7fffffff) return GLMB_ERR_TOO_LARGE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(ctas));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = unsigned(2 * a.splits);
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = dependent ? 2 : 1;
    count_launch();
    e = cudaLaunchKernelEx(&cfg, kernel, map, static_cast<const uint4*>(codes), scales, Yhat, a);
    return e != cudaSuccess ? int(e) : launch_status();
}

}  // namespace

template <typename T>
size_t q4_tile_workspace(int64_t nf, int64_t ntasks, int64_t nobs) {
    // float X, and X whose rows TMA cannot step over, are laid out anew first (also where only X's address is odd)
    return round_up(size_t(Split16<T>::kTerms) * size_t(nobs) * size_t(ntasks) * size_t(padded(nf)) * 2, 256);
}

template <typename T>
int q4_tile_predict(const T* X, const void* codes, const T* scales, T* Yhat, int64_t nf, int64_t nt, int64_t ntasks,
                    int64_t nobs, int group, bool vec, void* ws, size_t ws_bytes, cudaStream_t stream) {
    using H = typename Split16<T>::Type;
    constexpr int kTerms = Split16<T>::kTerms;
    auto fn = tensor_map_encoder();
    if (fn == nullptr) return GLMB_ERR_UNSUPPORTED;
    if (nobs > (int64_t(1) << 30) || ntasks > (int64_t(1) << 30)) return GLMB_ERR_TOO_LARGE;
    const bool lay_out = kTerms > 1 || !vec;
    const size_t need = q4_tile_workspace<T>(nf, ntasks, nobs);
    if (ws != nullptr && ws_bytes < need) return GLMB_ERR_WORKSPACE;
    Scratch sc(ws, ws_bytes, lay_out ? need : 0, stream);
    if (sc.status() != GLMB_OK) return sc.status();
    const int64_t ld = lay_out ? padded(nf) : nf, rows = nobs * ntasks;
    const H* src = reinterpret_cast<const H*>(X);
    if (lay_out) {
        H* out = sc.template as<H>();
        const int64_t blocks = std::min<int64_t>(int64_t(sm_count()) * 16, (rows * (ld / 8) + 255) / 256);
        q4_terms_kernel<T><<<unsigned(std::max<int64_t>(1, blocks)), 256, 0, stream>>>(X, out, rows, nf, ld, vec);
        count_launch();
        if (const int st = launch_status(); st != GLMB_OK) return st;
        src = out;
    }
    TileArgs a{nt, ntasks, nobs, q4_row_blocks(nt), int(q4_col_blocks(nf)), int(q4_groups(nf, group)), 0, 0, 1,
               group == 64 ? 0 : 1};
    a.tiles_m = int((nt + 255) / 256);
    // The cut with the least estimated time, in clocks: a block of features takes 2 N clocks of MMA a term and no
    // less than the 450 of making its operands; a tile 5000 besides, and its outputs.
    int best_n = 0;
    double least = 0.0;
    for (int n = 32; n <= 256; n *= 2) {
        const int64_t tiles_n = (nobs + n - 1) / n;
        for (int splits = 1; splits <= kMaxSplits; splits *= 2) {
            if (splits > 1 && a.ncb < 8 * splits) break;
            const int64_t at_once = std::max<int64_t>(1, sm_count() / (2 * splits));
            const int64_t waves = (int64_t(a.tiles_m) * tiles_n * ntasks + at_once - 1) / at_once;
            const double block = std::max(450.0, 2.2 * n * kTerms);
            const double t = double(waves) * ((a.ncb + splits - 1) / splits * block + 5000.0 + 10.0 * n +
                                              (splits > 1 ? 2500.0 + 10.0 * n / splits : 0.0));
            if (least == 0.0 || t < least) {
                least = t;
                best_n = n;
                a.tiles_n = int(tiles_n);
                a.splits = splits;
            }
        }
    }
    CUtensorMap map;
    const cuuint64_t dims[4] = {cuuint64_t(nf), cuuint64_t(nobs), cuuint64_t(ntasks), cuuint64_t(kTerms)};
    const cuuint64_t strides[3] = {cuuint64_t(ntasks * ld) * 2, cuuint64_t(ld) * 2, cuuint64_t(rows * ld) * 2};
    const cuuint32_t box[4] = {kBK, cuuint32_t(best_n / 2), 1, cuuint32_t(kTerms)}, one[4] = {1, 1, 1, 1};
    const auto type = std::is_same_v<H, __half> ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    if (fn(&map, type, 4, const_cast<H*>(src), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return GLMB_ERR_TOO_LARGE;
    switch (best_n) {
        case 32: return launch_tile<T, 32>(map, codes, scales, Yhat, a, lay_out, stream);
        case 64: return launch_tile<T, 64>(map, codes, scales, Yhat, a, lay_out, stream);
        case 128: return launch_tile<T, 128>(map, codes, scales, Yhat, a, lay_out, stream);
        default: return launch_tile<T, 256>(map, codes, scales, Yhat, a, lay_out, stream);
    }
}

#define GLMB_INSTANTIATE_Q4_TILE(T)                                                                             \
    template size_t q4_tile_workspace<T>(int64_t, int64_t, int64_t);                                            \
    template int q4_tile_predict<T>(const T*, const void*, const T*, T*, int64_t, int64_t, int64_t, int64_t, int, \
                                    bool, void*, size_t, cudaStream_t);

GLMB_INSTANTIATE_Q4_TILE(float)
GLMB_INSTANTIATE_Q4_TILE(__half)
GLMB_INSTANTIATE_Q4_TILE(__nv_bfloat16)

}  // namespace glmb
