// Decoding of 4-bit cache words, shared by the attention kernels over that cache.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace gb {

__device__ __forceinline__ uint32_t h2u(__half2 h) { return *(uint32_t*)&h; }
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *(__half2*)&u; }

__device__ __forceinline__ float q4_to_f(float x) { return x; }
__device__ __forceinline__ float q4_to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float q4_to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void q4_put(float* p, float x) { *p = x; }
__device__ __forceinline__ void q4_put(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void q4_put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Scales that V's product cannot take: infinities, NaN and magnitudes beyond 8188, the largest that a
// write stores (8 times more has no f16).  Their sign bits mark them, in each half of a word.
__device__ __forceinline__ uint32_t bad_scales(uint32_t d) {
    return ((d & 0x7FFF7FFFu) + 0x10001000u) & 0x80008000u;
}

// (x & MASK) | 0x64006400 as the one instruction it is (written in C it came out as two)
template <uint32_t MASK>
__device__ __forceinline__ uint32_t and_or(uint32_t x) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "n"(MASK), "r"(0x64006400u));
    return r;
}
// four f16 pairs from `x`: nibbles 0, 1, 2, 3 of each half, as 1024 + n (0, 2) or 1024 + 16 n
// (1, 3).  Of one code word the pairs are its dims (0, 4), (1, 5), (2, 6), (3, 7)
__device__ __forceinline__ void nibbles(uint32_t x, uint32_t (&r)[4]) {
    const uint32_t y = x >> 8;
    r[0] = and_or<0x000F000F>(x);
    r[1] = and_or<0x00F000F0>(x);
    r[2] = and_or<0x000F000F>(y);
    r[3] = and_or<0x00F000F0>(y);
}
// the same as exact integers code - 8
__device__ __forceinline__ void codes(uint32_t x, __half2 (&v)[4]) {
    uint32_t r[4];
    nibbles(x, r);
    const __half2 o = u2h(0x64086408u), m16 = u2h(0x2C002C00u), s = u2h(0xD480D480u);
    v[0] = __hsub2(u2h(r[0]), o);          // 1024 + n - 1032
    v[1] = __hfma2(u2h(r[1]), m16, s);     // (1024 + 16 n) / 16 - 72
    v[2] = __hsub2(u2h(r[2]), o);
    v[3] = __hfma2(u2h(r[3]), m16, s);
}

}  // namespace gb
