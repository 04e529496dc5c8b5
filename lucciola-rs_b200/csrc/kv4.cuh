// kv4.cuh - the 4-bit paged KV cache: page layout and conversions.
//
// A pool is uint8 [num_blocks][num_layers][num_kv_heads][2][9 * head_dim]: for
// each page and kv head first K, then V. One half holds the codes of the 16
// tokens, [16][head_dim / 2] bytes (e2m1 values, even dim in the low nibble),
// then their scales, [16][head_dim / 16] bytes (e4m3, one per 16 dims). An
// element stands for
//     e2m1(code) * e4m3(scale) * g
// with a caller's factor g per tensor (k_scale, v_scale). K and V of a page are
// adjacent, so that one bulk copy of 18 * head_dim bytes brings both.
//
// e2m1 has 2 significant bits and e4m3 has 4, so e2m1 * e4m3 has at most 6 and
// lies in [2^-10, 2688]: the product is exact in fp16 and in bf16.
#pragma once

#include <cuda_fp16.h>

#include "lc_common.cuh"

namespace lc {

constexpr int kKv4Group = 16;  // dims per scale
constexpr uint32_t kKv4NanScale = 0x7f;

__host__ __device__ constexpr int kv4_code_bytes(int hd) { return kBlockSize * hd / 2; }
__host__ __device__ constexpr int kv4_half_bytes(int hd) {
    return kv4_code_bytes(hd) + kBlockSize * hd / kKv4Group;
}

// Byte offset of (physical block, layer, kv head): K there, V kv4_half_bytes on.
__host__ __device__ inline int64_t kv4_offset(int64_t phys, int layer, int kv_head,
                                              int num_layers, int num_kv_heads, int hd) {
    return ((phys * num_layers + layer) * num_kv_heads + kv_head) * 2 * kv4_half_bytes(hd);
}

// A caller's factor g: positive and far enough from the ends of fp32 that
// 6 g, 2688 g and a quotient by 2^-9 g stay finite.
inline bool kv4_scale_ok(float g) { return g >= 0x1p-64f && g <= 0x1p64f; }

// The eight codes of `w` (dims in nibble order) as fp16 pairs. Load `w` as a
// word: with a single byte loaded for it, nvcc 12.9 builds code that gives zeros.
__device__ __forceinline__ void e2m1x8_to_half(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
}

// Two e4m3 scales (low byte first) as an fp16 pair; a NaN scale gives NaN.
__device__ __forceinline__ uint32_t e4m3x2_to_half(uint32_t s) {
    uint32_t h;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, lo;\n\t}"
        : "=r"(h)
        : "r"(s));
    return h;
}

__device__ __forceinline__ float e4m3_to_float(uint32_t s) {
    const uint32_t h = e4m3x2_to_half(s & 0xffu);
    return __low2float(*reinterpret_cast<const __half2 *>(&h));
}

// Scale byte of a 16-dim group whose largest magnitude has the bits `amax`:
// e4m3(amax / (6 g)), nearest even, at most 448, so that the largest code (6)
// meets the largest value. A group that holds an infinity or a NaN gets a NaN
// scale, and with it NaN in all its elements: 4 bits cannot say which it was.
__device__ __forceinline__ uint32_t kv4_scale_byte(uint32_t amax, float six_g) {
    if (amax >= 0x7f800000u) return kKv4NanScale;
    uint32_t s;
    asm("{\n\t.reg .b16 t;\n\tcvt.rn.satfinite.e4m3x2.f32 t, %2, %1;\n\tmov.b32 %0, {t, t};\n\t}"
        : "=r"(s)
        : "f"(__fdiv_rn(__uint_as_float(amax), six_g)), "f"(0.f));
    return s & 0xffu;
}

// Pairs of fp32 values, each operation rounded by itself. A sum of products is
// written as fma2(product, one, product) with a `one` that the compiler cannot see
// through: nvcc 12.9 contracts mul.rn.f32x2 and add.rn.f32x2 into one rounding.
__device__ __forceinline__ uint64_t pair2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 split2(uint64_t a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// Codes of eight values (pairs) over `step` = e4m3(scale) * g: e2m1(x / step),
// nearest even; `amax` holds the bits of the group's largest magnitude. The
// quotient has to be the rounded one, not a product with a reciprocal: bf16 values
// over 4-bit scales often lie exactly between two codes, and a quotient off by one
// rounding would send them to the wrong one. A product with the rounded reciprocal
// corrected once by its exact remainder (P. Markstein, "Computation of elementary
// functions on the IBM RISC System/6000 processor", 1990) gives it in three
// operations per pair: equal to the divided value for every one of 18 million tried
// around the boundaries. It is -x / step that is computed, and the codes' signs are
// turned afterwards: a zero x then keeps its sign (the remainder is +0 for both zeros,
// and +0 times the negative reciprocal added to a zero leaves that as it is), where
// x / step would make +0 of -0. Groups whose scale is at its limit (quotients beyond 8)
// take the division.
__device__ __forceinline__ uint32_t kv4_codes(const uint64_t (&x)[4], float step, uint32_t amax) {
    float y[8];
    uint32_t signs = 0;
    if (step > 0.f && __uint_as_float(amax) <= 8.f * step) {
        const float r = __frcp_rn(step);
        const uint64_t rr = pair2(-r, -r), ss = pair2(step, step);
        signs = 0x88888888u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint64_t q = mul2(x[i], rr);  // -x / step, nearly; x + q step is what is left
            const float2 v = split2(fma2(fma2(q, ss, x[i]), rr, q));
            y[2 * i] = v.x, y[2 * i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 v = split2(x[i]);
            y[2 * i] = step > 0.f ? __fdiv_rn(v.x, step) : copysignf(0.f, v.x);
            y[2 * i + 1] = step > 0.f ? __fdiv_rn(v.y, step) : copysignf(0.f, v.y);
        }
    }
    uint32_t w;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(w)
        : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
    return w ^ signs;
}

}  // namespace lc
