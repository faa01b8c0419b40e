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

// The four pairs of a word of codes (u = q + 8) as 16-bit floats q: the code is put under the leading bit of
// a power of two (1024 + u or, four bits up, 1024 + 16u in binary16; 128 + u in bfloat16) and the offset taken
// off again, exactly.
template <typename H>
__device__ __forceinline__ void code_pairs(uint32_t w, uint32_t (&r)[4]) {
    if constexpr (std::is_same_v<H, __half>) {
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
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t t;
            asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(t) : "r"(w >> (4 * i)));
            asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r[i]) : "r"(t), "r"(0xc308c308u));  // -136
        }
    }
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

// The scales of targets g and g + 8, which lie side by side.
template <typename T>
struct alignas(2 * sizeof(T)) Pair {
    T first, second;
};

}  // namespace glmb
