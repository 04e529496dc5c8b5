// kv8.cuh - the 8-bit paged KV cache: page layout and conversions.
//
// A pool is uint8 [num_blocks][num_layers][num_kv_heads][32 * head_dim + 16]: for each
// page and kv head the K codes of its 16 tokens, [16][head_dim] bytes (e4m3), the V codes
// likewise, then the two scales (fp32: K's, V's) and 8 unused bytes. An element stands for
//     e4m3(code) * scale
// with one scale for all tokens of the page, so that a product with K takes it once per
// page and score, and one with V once per page and probability. Scales are powers of two
// from 2^-40 to 2^40: e4m3 has 4 significant bits wherever its exponent is, so a finer
// scale would add none, a page's tokens move to a larger scale without a second rounding
// (but for the smallest), and unpacked values are exact in bf16.
//
// The 16-dim pieces of a token's row are permuted by its number (kv8_piece): the decode
// reads four tokens' pieces at once, and rows lie one (or two) to a line of shared memory.
// The bulk copy that brings a page keeps the order; in plain order V's reads would hit the
// same banks four times over, K's twice.
#pragma once

#include <cuda_fp16.h>

#include "lc_common.cuh"

namespace lc {

constexpr int kKv8MinExp = -40, kKv8MaxExp = 40;  // of a scale
constexpr uint32_t kKv8Nan = 0x7f;

__host__ __device__ constexpr int kv8_half_bytes(int hd) { return kBlockSize * hd; }
__host__ __device__ constexpr int kv8_page_bytes(int hd) { return 2 * kv8_half_bytes(hd) + 16; }

// Byte offset of (physical block, layer, kv head): K there, V kv8_half_bytes on, the
// scales 2 * kv8_half_bytes on.
__host__ __device__ inline int64_t kv8_offset(int64_t phys, int layer, int kv_head,
                                              int num_layers, int num_kv_heads, int hd) {
    return ((phys * num_layers + layer) * num_kv_heads + kv_head) * kv8_page_bytes(hd);
}

// Where the 16-dim piece `piece` of a token's row lies in the row.
__host__ __device__ constexpr int kv8_piece(int hd, int token, int piece) {
    return piece ^ ((token * hd / 64) & (hd / 16 - 2));
}

// Exponent of the smallest scale that holds a magnitude with the fp32 bits `amax`
// (finite): amax <= 448 * 2^e, 448 = 1.75 * 2^8.
__device__ __forceinline__ int kv8_exponent(uint32_t amax) {
    const int e = (int)(amax >> 23) - (127 + 8) + ((amax & 0x7fffffu) > 0x600000u);
    return min(max(e, kKv8MinExp), kKv8MaxExp);
}
__device__ __forceinline__ float kv8_scale(int e) { return __int_as_float((e + 127) << 23); }
// The exponent of a scale as a page holds it, whatever the page holds.
__device__ __forceinline__ int kv8_scale_exp(uint32_t bits) {
    return min(max((int)(bits >> 23 & 0xffu) - 127, kKv8MinExp), kKv8MaxExp);
}

// Two e4m3 codes (the low 16 bits, low byte first) as an fp16 pair, exactly.
__device__ __forceinline__ uint32_t kv8_half2(uint32_t two) {
    uint32_t h;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, lo;\n\t}"
        : "=r"(h)
        : "r"(two));
    return h;
}
// Four codes as two fp16 pairs.
__device__ __forceinline__ void kv8_half4(uint32_t four, uint32_t &lo, uint32_t &hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(four));
}
// Four values as codes, to nearest even, at most 448 in magnitude; NaN stays NaN.
__device__ __forceinline__ uint32_t kv8_codes4(float a, float b, float c, float d) {
    uint32_t w;
    asm("{\n\t.reg .b16 lo, hi;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
        "mov.b32 %0, {lo, hi};\n\t}"
        : "=r"(w)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return w;
}
// Four codes of a page whose scale grows by 1 / `down`, a power of two below 1.
__device__ __forceinline__ uint32_t kv8_rescale4(uint32_t four, float down) {
    uint32_t lo, hi;
    kv8_half4(four, lo, hi);
    const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&lo));
    const float2 y = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
    return kv8_codes4(x.x * down, x.y * down, y.x * down, y.y * down);
}

}  // namespace lc
