// The 8-bit cache of keys and values: its page layout and its numbers, shared by the kernels that write and read it.
//
// A row (the head_dim numbers of one token's key or value in one KV head) is kept as e4m3 numbers c_i and one scale 2^e:
//
//   e = the smallest whole number with  max_i |x_i| <= 448 * 2^e,  kept between -60 and 40;      c_i = rn_e4m3(x_i * 2^-e)
//
// A power of two costs a floating number nothing: whatever the scale's fraction, a normal e4m3 number is off by at most 2^-4 of
// itself, and c_i * 2^e is exact in bfloat16 and in 32 bits.  The bounds on e keep weights and scales of one softmax
// within the range of 32-bit numbers however rows differ (beyond 448 * 2^40 = 4.9e14 a number saturates).  A number that is not finite is
// kept as NaN and does not count in the maximum; a row of zeros has e = -60.
//
// A page: [2][kv_heads][page_size][head_dim] bytes (keys, then values), then [2][kv_heads][page_size] scale bytes e + 127, then
// padding to a multiple of 16 bytes.  Rows and pages start on 16-byte boundaries, as head sizes are multiples of 16.
#pragma once
#include "common.cuh"

#define KV8_LOWEST (-60)
#define KV8_HIGHEST 40

__host__ __device__ __forceinline__ long long kv8_page_bytes(int nkv, int P, int hd) {
    return ((2LL * nkv * P * (hd + 1)) + 15) / 16 * 16;
}

// 2^e from the byte that holds e + 127 (1 .. 254)
__device__ __forceinline__ float kv8_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// a row's scale byte from the largest magnitude's bits (finite, non-negative): 448 = 1.75 * 2^8
__device__ __forceinline__ int kv8_scale_byte(uint32_t amax_bits) {
    const int e = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, KV8_LOWEST), KV8_HIGHEST) + 127;
}

// four e4m3 numbers of a word to 32 bits, exactly
__device__ __forceinline__ float4 kv8_unpack(uint32_t w) {
    uint32_t lo, hi;
    asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}" : "=r"(lo), "=r"(hi) : "r"(w));
    float4 f;
    asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.f32.f16 %0, a;\ncvt.f32.f16 %1, b;\n}" : "=f"(f.x), "=f"(f.y) : "r"(lo));
    asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.f32.f16 %0, a;\ncvt.f32.f16 %1, b;\n}" : "=f"(f.z), "=f"(f.w) : "r"(hi));
    return f;
}

// two numbers to e4m3, `a` in the lower byte; beyond the range: the largest
__device__ __forceinline__ uint32_t kv8_pack2(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint32_t kv8_pack4(float a, float b, float c, float d) {
    return kv8_pack2(a, b) | (kv8_pack2(c, d) << 16);
}
