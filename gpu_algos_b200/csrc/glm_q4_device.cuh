// glm_q4_device.cuh -- device helpers of the 4-bit kernels (glm_q4.cu, glm_q4_tile.cu).
#pragma once

#include "glm_q4.cuh"

namespace glmb {

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

// What prediction's codes are multiplied by as operands, 2^-kCodeDown: a group's sum of q x is formed before its
// scale brings it back to the result's size, and 128 products of up to 7 |x| would pass float's range for a
// bfloat16 or float x near its end.  The total is multiplied by 2^kCodeDown when it is written; powers of two
// change no bits of either (below 2^-116 a float result keeps steps of 2^-139).  binary16 has no such x.
template <typename H>
inline constexpr int kCodeDown = std::is_same_v<H, __half> ? 0 : 10;
template <typename H>
inline constexpr float kCodeUp = float(1 << kCodeDown<H>);

// The four pairs of a word of codes (u = q + 8) as 16-bit floats q 2^-DOWN, by the usual conversion of small whole
// numbers: the code is put under the leading bit of a power of two (1024 + u or, four bits up, 1024 + 16u in
// binary16, whose fraction has 10 bits; (128 + u) 2^-DOWN in bfloat16, which has 7) and the offset taken off
// again, exactly.
template <typename H, int DOWN = 0>
__device__ __forceinline__ void code_pairs(uint32_t w, uint32_t (&r)[4]) {
    if constexpr (std::is_same_v<H, __half>) {
        static_assert(DOWN == 0);
        const uint32_t w8 = w >> 8;
        uint32_t t;
        asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(t) : "r"(w));
        asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r[0]) : "r"(t), "r"(0xe408e408u));  // -1032
        asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(t) : "r"(w));
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r[1]) : "r"(t), "r"(0x2c002c00u), "r"(0xd480d480u));  // /16 - 72
        asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(t) : "r"(w8));
        asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r[2]) : "r"(t), "r"(0xe408e408u));
        asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(t) : "r"(w8));
        asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r[3]) : "r"(t), "r"(0x2c002c00u), "r"(0xd480d480u));
    } else {
        constexpr uint32_t kLess = uint32_t(DOWN) * 0x00800080u;  // of both exponents
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t t;
            asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(t) : "r"(w >> (4 * i)), "n"(0x43004300u - kLess));
            asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r[i]) : "r"(t), "r"(0xc308c308u - kLess));  // -136 2^-DOWN
        }
    }
}

// x as a sum of terms of the tensor core's type (one for a 16-bit x, three for a float)
template <typename T>
__device__ __forceinline__ void split_terms(T x, typename Split16<T>::Type (&t)[Split16<T>::kTerms]) {
    if constexpr (std::is_same_v<T, float>) {
        // a NaN or an infinity stays in the first term alone; a finite x past bfloat16's largest leaves the rest to
        // the second
        const bool finite = fabsf(x) <= 3.402823466e38f;
        const float most = __uint_as_float(0x7f7f0000u);
        t[0] = __float2bfloat16_rn(finite ? fminf(fmaxf(x, -most), most) : x);
        const float r1 = x - __bfloat162float(t[0]);
        t[1] = __float2bfloat16_rn(finite ? r1 : 0.0f);
        t[2] = __float2bfloat16_rn(finite ? r1 - __bfloat162float(t[1]) : 0.0f);
    } else {
        t[0] = x;
    }
}

// The scales of targets g and g + 8, which lie side by side.
template <typename T>
struct alignas(2 * sizeof(T)) Pair {
    T first, second;
};

}  // namespace glmb
