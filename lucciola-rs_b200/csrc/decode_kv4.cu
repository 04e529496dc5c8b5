// decode_kv4.cu - attention of the newest tokens of each sequence over the 4-bit
// paged cache (kv4.cuh): decode_stream.cuh with its pages.
//
// Bounds. 64 sequences of 1024 .. 16384 tokens, 64/8 heads of 128: 122 us, 5.0 TB/s
// of pages (77 % of a device copy's rate); 32 of 8192, 28/4 heads: 37.5 us, 3.9 TB/s.
// There a page of 128 dims costs 309 instructions of a warp (8 columns): 54 % of the issue
// slots, the ALU pipe 47 %, the tensor pipe 22 %, its ends included. About 8 of the 37.5 us
// are ends; between them the pages come at 78 % of the copy's rate and two thirds of the
// issue slots are taken, so that no one unit binds, the warps' own chain (load, convert,
// multiply, product) with four of them per scheduler does. With 24 columns a page costs
// 390 instructions, 45 % of the issue slots and 44 % of the tensor pipe, with two warps
// per scheduler. Short work is bound by its ends, length -> table -> page before the
// first product (3.6 us) and the join after the last (2 to 4 us): one sequence of 1024
// tokens 6.7 us.
//
// Unpacking. e2m1 to fp16 is one conversion per pair, the scale one multiplication per
// pair, both exact (kv4.cuh).
//  * K: a lane's operand elements are 4 dims per step of 2 tokens. The order of
//    dims within the sum is free, so lane t of a quad takes the dims hd/4 * t ..
//    and reads them as one 16-byte (8 at hd 64) load per token.
//  * V: a lane holds hd/8 consecutive dims of 4 tokens and needs pairs of tokens
//    per dim: two tokens' words are interleaved by nibbles first, then converted.
#include "decode_stream.cuh"
#include "kv4.cuh"

namespace lc {
namespace {

// The 4-bit pages, for decode_stream.cuh.
template <int D>
struct Kv4 {
    static constexpr int kDim = D;
    static constexpr int kPage = 18 * D;  // K and V of one kv head
    template <int NT>
    static constexpr int kGroup = 2;
    static constexpr int kStages = D == 64 ? 4 : 2;  // two groups of the 128-dim pages
    static constexpr int kMinPages = 16;  // pages per CTA at least: a group for each of its warps
    // (64 sequences of 256 .. 4096 tokens, 14/2 heads of 64: 14.6 us with 32 units, 15.1 with
    // 24, 18.3 with none; 256 of 100 .. 300: 15.2, 15.3, 19.5; 32 of 8192, 28/4 heads of 128:
    // 37.5, 37.4, 38.9, and 38.1 with 36.)
    static constexpr int kEdgeUnits = 32;
    static constexpr int kAlonePages = 0;
    static constexpr bool kPageScales = false;
    static constexpr int kSteps = D / 16, kWords = D / 32;  // code words per token and lane (K)

    static __device__ __forceinline__ int64_t offset(int64_t phys, int layer, int head, int layers,
                                                     int heads) {
        return kv4_offset(phys, layer, head, layers, heads, D);
    }
    // Lane t's dims of q, eight at a time: a quarter of them in a row.
    static __device__ __forceinline__ int q_dim(int t, int k) { return t * (D / 4) + 8 * k; }

    template <int NT, int kGroup>
    static __device__ __forceinline__ void scores(const uint8_t *st, const uint2 *qs, int pi0, int t,
                                                  float (&s)[kGroup][NT][4]) {
        uint32_t wa[kGroup][kWords], wb[kGroup][kWords], sa[kGroup][2], sb[kGroup][2];
#pragma unroll
        for (int pg = 0; pg < kGroup; ++pg) {
            const uint8_t *kp = st + pg * kPage;
            if constexpr (kDim == 128) {
                const uint4 a = *reinterpret_cast<const uint4 *>(kp + pi0 * 64 + t * 16);
                const uint4 b = *reinterpret_cast<const uint4 *>(kp + (pi0 + 8) * 64 + t * 16);
                wa[pg][0] = a.x, wa[pg][1] = a.y, wa[pg][2] = a.z, wa[pg][3] = a.w;
                wb[pg][0] = b.x, wb[pg][1] = b.y, wb[pg][2] = b.z, wb[pg][3] = b.w;
                const uint8_t *sc = kp + kv4_code_bytes(kDim) + pi0 * 8 + t * 2;
                const uint32_t ha = e4m3x2_to_half(*reinterpret_cast<const uint16_t *>(sc));
                const uint32_t hb = e4m3x2_to_half(*reinterpret_cast<const uint16_t *>(sc + 64));
                sa[pg][0] = both_low(ha), sa[pg][1] = both_high(ha);
                sb[pg][0] = both_low(hb), sb[pg][1] = both_high(hb);
            } else {
                const uint2 a = *reinterpret_cast<const uint2 *>(kp + pi0 * 32 + t * 8);
                const uint2 b = *reinterpret_cast<const uint2 *>(kp + (pi0 + 8) * 32 + t * 8);
                wa[pg][0] = a.x, wa[pg][1] = a.y;
                wb[pg][0] = b.x, wb[pg][1] = b.y;
                const uint8_t *sc = kp + kv4_code_bytes(kDim) + pi0 * 4 + t;
                const uint32_t h = e4m3x2_to_half(sc[0] | sc[32] << 8);
                sa[pg][0] = both_low(h);
                sb[pg][0] = both_high(h);
            }
        }
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
            uint2 qf[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int k = 0; k < 2; ++k) qf[nt][k] = qs[(nt * kSteps + 2 * w + k) * 32];
#pragma unroll
            for (int pg = 0; pg < kGroup; ++pg) {
                uint32_t ha[4], hb[4];
                e2m1x8_to_half(wa[pg][w], ha);
                e2m1x8_to_half(wb[pg][w], hb);
                const uint32_t fa = sa[pg][w / 2], fb = sb[pg][w / 2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t a0 = hmul2(ha[2 * k], fa), a2 = hmul2(ha[2 * k + 1], fa);
                    const uint32_t a1 = hmul2(hb[2 * k], fb), a3 = hmul2(hb[2 * k + 1], fb);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        if (w + k == 0)
                            mma_f16_first(s[pg][nt], a0, a1, a2, a3, qf[nt][k].x, qf[nt][k].y);
                        else
                            mma_f16(s[pg][nt], a0, a1, a2, a3, qf[nt][k].x, qf[nt][k].y);
                }
            }
        }
    }

    // Page pg of the group at token tok0. `held`: tokens of the chunk's pages, `all`: that every
    // column sees, lim: that a column sees. (The sums of these are written out where they are
    // used: handed over ready, they cost spills.)
    template <int NT, bool kTail>
    static __device__ __forceinline__ void values(const uint8_t *st, int pg, int g, int t,
                                                  const uint32_t (&pf)[NT][2],
                                                  float (&o)[kSteps][NT][4], int tok0, int held,
                                                  int all, int drafts, const int (&lim)[NT][2]) {
        const uint8_t *vp = st + pg * kPage + kv4_half_bytes(kDim);
        const uint8_t *sc = vp + kv4_code_bytes(kDim);
        constexpr int kRowBytes = kDim / 2, kRowScales = kDim / 16;
        const int sg = g * (kDim / 8) / kKv4Group;  // scale of this lane's dims
        uint32_t s01 = sc[t * kRowScales + sg] | sc[(7 - t) * kRowScales + sg] << 8;
        uint32_t s23 = sc[(8 + t) * kRowScales + sg] | sc[(15 - t) * kRowScales + sg] << 8;
        if constexpr (kTail) {
            // tokens past the end hold anything: their scales become zero
            const int left = held - tok0 - pg * kBlockSize;
            if (t >= left) s01 &= 0xff00u;
            if (7 - t >= left) s01 &= 0x00ffu;
            if (8 + t >= left) s23 &= 0xff00u;
            if (15 - t >= left) s23 &= 0x00ffu;
            if (drafts > 1) {
                // Of the last tokens, which not every column sees, a NaN scale must
                // reach the columns that see it only, not as 0 * NaN the others.
                const int common = all - tok0 - pg * kBlockSize;
                uint32_t nan = 0;  // by token of the page
                auto drop = [&](uint32_t &sc2, int sh, int tok) {
                    if ((sc2 >> sh & 0x7fu) == kKv4NanScale && tok >= common && tok < left) {
                        sc2 &= ~(0xffu << sh);
                        nan |= 1u << tok;
                    }
                };
                drop(s01, 0, t);
                drop(s01, 8, 7 - t);
                drop(s23, 0, 8 + t);
                drop(s23, 8, 15 - t);
                nan |= __shfl_xor_sync(0xffffffffu, nan, 1);
                nan |= __shfl_xor_sync(0xffffffffu, nan, 2);
                if (nan)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            if (lim[nt][k] - tok0 - pg * kBlockSize > __ffs(nan) - 1)
#pragma unroll
                                for (int j = 0; j < kSteps; ++j)
                                    o[j][nt][k] = o[j][nt][k + 2] = NAN;
            }
        }
        const uint32_t h01 = e4m3x2_to_half(s01), h23 = e4m3x2_to_half(s23);
        uint32_t v[4][kDim / 64];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = (i & 1 ? 7 - t : t) + (i >> 1) * 8;
            if constexpr (kDim == 128) {
                const uint2 x = *reinterpret_cast<const uint2 *>(vp + row * kRowBytes + g * 8);
                v[i][0] = x.x, v[i][1] = x.y;
            } else {
                v[i][0] = *reinterpret_cast<const uint32_t *>(vp + row * kRowBytes + g * 4);
            }
        }
#pragma unroll
        for (int w = 0; w < kDim / 64; ++w) {
            constexpr uint32_t kLow = 0x0f0f0f0fu;
            uint32_t e01[4], d01[4], e23[4], d23[4];  // even and odd dims
            e2m1x8_to_half((v[0][w] & kLow) | (v[1][w] << 4 & ~kLow), e01);
            e2m1x8_to_half((v[0][w] >> 4 & kLow) | (v[1][w] & ~kLow), d01);
            e2m1x8_to_half((v[2][w] & kLow) | (v[3][w] << 4 & ~kLow), e23);
            e2m1x8_to_half((v[2][w] >> 4 & kLow) | (v[3][w] & ~kLow), d23);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t a0 = hmul2(e01[k], h01), a1 = hmul2(d01[k], h01);
                const uint32_t a2 = hmul2(e23[k], h23), a3 = hmul2(d23[k], h23);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    mma_f16(o[4 * w + k][nt], a0, a1, a2, a3, pf[nt][0], pf[nt][1]);
            }
        }
    }
};

}  // namespace
}  // namespace lc

using namespace lc;

extern "C" size_t lc_paged_decode_kv4_workspace_size(int batch, int num_q_heads, int num_kv_heads,
                                                     int head_dim, int tokens_per_seq) {
    return decode_workspace(batch, num_q_heads, num_kv_heads, head_dim, tokens_per_seq);
}

extern "C" int lc_paged_decode_kv4(void *out, int64_t out_stride, const void *q, int64_t q_stride,
                                   const void *kv_pool, int64_t num_blocks, int num_layers,
                                   int layer, int num_q_heads, int num_kv_heads, int head_dim,
                                   const int *block_tables, int table_stride,
                                   const int *context_lens, int len_offset, int batch,
                                   int tokens_per_seq, int max_context_len, float k_scale,
                                   float v_scale, float sm_scale, void *workspace,
                                   size_t workspace_bytes, int *dev_status, lc_stream_t stream) {
    if (!out || !q || !kv_pool || !block_tables || !context_lens || !kv4_scale_ok(k_scale) ||
        !kv4_scale_ok(v_scale))
        return LC_ERR_INVALID_ARGUMENT;
    DecodeParams p{};
    p.scale_log2 = std::fabs(sm_scale) * k_scale * 1.4426950408889634f;
    p.q_sign = std::signbit(sm_scale) ? 0x80008000u : 0u;
    p.v_scale = v_scale;
    return decode_stream<Kv4>(p, out, out_stride, q, q_stride, kv_pool, num_blocks, num_layers, layer,
                              num_q_heads, num_kv_heads, head_dim, block_tables, table_stride,
                              context_lens, len_offset, batch, tokens_per_seq, max_context_len,
                              workspace, workspace_bytes, dev_status, stream);
}
