// decode_kv8.cu - attention of the newest tokens of each sequence over the 8-bit
// paged cache (kv8.cuh): decode_stream.cuh with its pages.
//
// Unpacking. e4m3 to fp16 is one exact conversion per pair; the page's scales do not touch
// the elements (decode_stream.cuh: page_scales).
//  * K: lane t of a quad takes two 16-dim pieces of a token (one at hd 64), t and t + 4, as
//    16-byte loads; a word is one step of the product.
//  * V: a lane holds hd/8 consecutive dims of 4 tokens and needs pairs of tokens per dim:
//    two tokens' words are interleaved by bytes first, then converted.
//
// Bounds. 32 sequences of 8192 tokens, 28/4 heads of 128: 48.1 to 49.1 us for 269 MB, 84 % of a
// device copy's rate, and 2 of 131072: 49.9 us. Between the first page (2.7 us after the start) and
// the last product (39 to 44 us, by SM) the pages come at the copy's rate, and the warps wait
// for them: 268 instructions of a warp per page, 39 % of the issue slots, the tensor pipe 17 %.
// What is left is the two ends: the chain length -> table -> page, SMs that share the same
// bytes ending 4 us apart, the join of the last chunk and its pieces (2.5 us). With 24 columns
// (3 drafted tokens, 8 sequences of 1024 .. 32000 tokens, 64/8 heads: 68 us of which 42 are
// the copy's) two warps per scheduler have 405 instructions and 48 products per page: issue
// 41 %, tensor pipe 39 %. Short contexts are bound by a CTA's chunks, 4 us each with the join
// of eight columns (256 sequences of 100 .. 300 tokens, 28/4 heads of 128: 24.4 us).
#include "decode_stream.cuh"
#include "kv8.cuh"

namespace lc {
namespace {

// The 8-bit pages, for decode_stream.cuh.
template <int D>
struct Kv8 {
    static constexpr int kDim = D;
    static constexpr int kPage = kv8_page_bytes(D);  // K and V of one kv head
    // Two pages at a time share their reads of q and overlap their products, where a stage of
    // two fits. (32 sequences of 8192 tokens, 14/2 heads of 64: 16.3 us, 19.0 us one at a time;
    // 2 tokens each over 8 of 1024 .. 32000, 64/8 heads of 128: 57.1 us, 65.3 us.)
    template <int NT>
    static constexpr int kGroup = D == 64 || NT == 2 ? 2 : 1;
    static constexpr int kStages = 2;  // what fits beside a second CTA
    // Pages per CTA at least. (One sequence of 203 tokens: 5.6 us, 6.2 us with 8 or 12; of 1024
    // tokens, 14/2 heads of 64: 6.4 us, 7.6 us with 24.)
    static constexpr int kMinPages = 16;
    // (64 sequences of 256 .. 4096 tokens, 14/2 heads of 64: 13.2 us, 14.0 us with 20, 13.8 with
    // 60; 256 of 100 .. 300, 28/4 heads of 128: 24.4 us, 26.7 us with 8, 24.8 with 20, 25.8 with 48.
    // The other way round, 24 for 64 dims: 64 of 0 .. 4096 with their append 16.9 us, 16.0 so; 16 of 500 ..
    // 16000, 14/2 heads, 14.3 and 13.7; but 64 of 256 .. 4096, 32/8 heads, 31.1 and 33.1. 48 for
    // 128: 64 of 256 .. 4096, 28/4 heads, 31.4 us, 30.2 so; 16 of 500 .. 16000, 12/2 heads, 17.7 and 17.8.)
    static constexpr int kEdgeUnits = D == 64 ? 48 : 24;
    // (One sequence of 8192 tokens, 64/8 heads of 128: 10.2 us in 128 CTAs of 32 pages, 11.6 us in
    // 256 of 16; of 12345, 28/4 heads: 10.3 us in 132 of 24, 11.0 us in 196 of 16; of 16384, where
    // 128 have 32 each, 11.2 us, 11.1 us in 256. Heads of 64 gain where there are many: of 6917
    // tokens, 32/8 heads, 9.1 us, 10.0 us without; of 5957, 12/12 heads, 9.1 and 9.8; of 33157, 14/2
    // heads, 10.7 and 10.2; of 16581, 28/4 heads, 10.5 and 9.9.)
    static constexpr int kAlonePages = 32;
    static constexpr bool kPageScales = true;
    static constexpr int kSteps = D / 16, kWords = D / 16;  // words per token and lane (K)

    static __device__ __forceinline__ int64_t offset(int64_t phys, int layer, int head, int layers,
                                                     int heads) {
        return kv8_offset(phys, layer, head, layers, heads, D);
    }
    // Lane t's dims of q, eight at a time: its pieces in turn.
    static __device__ __forceinline__ int q_dim(int t, int k) { return k / 2 * 64 + t * 16 + k % 2 * 8; }

    // K's scale, log2 of V's and 1 / V's, from whatever the page holds.
    static __device__ __forceinline__ void page_scales(const uint8_t *page, float &ks, float &lv,
                                                       float &out_v) {
        const uint2 sc = *reinterpret_cast<const uint2 *>(page + 2 * kv8_half_bytes(D));
        ks = kv8_scale(kv8_scale_exp(sc.x));
        const int e = kv8_scale_exp(sc.y);
        lv = (float)e;
        out_v = kv8_scale(-e);
    }

    template <int NT, int kGroup>
    static __device__ __forceinline__ void scores(const uint8_t *st, const uint2 *qs, int pi0, int t,
                                                  float (&s)[kGroup][NT][4]) {
        uint32_t wa[kGroup][kWords], wb[kGroup][kWords];  // tokens pi0 and pi0 + 8
        const int at = pi0 * D + kv8_piece(D, pi0, t) * 16;
#pragma unroll
        for (int pg = 0; pg < kGroup; ++pg) {
#pragma unroll
            for (int i = 0; i < kWords; i += 4) {  // piece t + i, whose place differs in that bit
                const uint8_t *kp = st + pg * kPage + (at ^ (i * 16));
                const uint4 a = *reinterpret_cast<const uint4 *>(kp);
                const uint4 b = *reinterpret_cast<const uint4 *>(kp + 8 * D);
                wa[pg][i] = a.x, wa[pg][i + 1] = a.y, wa[pg][i + 2] = a.z, wa[pg][i + 3] = a.w;
                wb[pg][i] = b.x, wb[pg][i + 1] = b.y, wb[pg][i + 2] = b.z, wb[pg][i + 3] = b.w;
            }
        }
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
            uint2 qf[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) qf[nt] = qs[(nt * kSteps + w) * 32];
#pragma unroll
            for (int pg = 0; pg < kGroup; ++pg) {
                uint32_t a0, a1, a2, a3;
                kv8_half4(wa[pg][w], a0, a2);
                kv8_half4(wb[pg][w], a1, a3);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    if (w == 0)
                        mma_f16_first(s[pg][nt], a0, a1, a2, a3, qf[nt].x, qf[nt].y);
                    else
                        mma_f16(s[pg][nt], a0, a1, a2, a3, qf[nt].x, qf[nt].y);
            }
        }
    }

    // Bytes of a word that are NaN codes, a bit each.
    static __device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
        const uint32_t is = __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu);
        return (is & 1u) | (is >> 7 & 2u) | (is >> 14 & 4u) | (is >> 21 & 8u);
    }

    // Page pg of the group at token tok0. `held`: tokens of the chunk's pages, `all`: that every
    // column sees, lim: that a column sees.
    template <int NT, bool kTail>
    static __device__ __forceinline__ void values(const uint8_t *st, int pg, int g, int t,
                                                  const uint32_t (&pf)[NT][2],
                                                  float (&o)[kSteps][NT][4], int tok0, int held,
                                                  int all, int drafts, const int (&lim)[NT][2]) {
        constexpr int kVWords = D / 32;  // 4 dims each
        const uint8_t *vp = st + pg * kPage + kv8_half_bytes(D);
        uint32_t v[4][kVWords];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = (i & 1 ? 7 - t : t) + (i >> 1) * 8;
            if constexpr (D == 128) {
                const uint4 x =
                    *reinterpret_cast<const uint4 *>(vp + row * D + kv8_piece(D, row, g) * 16);
                v[i][0] = x.x, v[i][1] = x.y, v[i][2] = x.z, v[i][3] = x.w;
            } else {
                const uint2 x = *reinterpret_cast<const uint2 *>(
                    vp + row * D + kv8_piece(D, row, g / 2) * 16 + g % 2 * 8);
                v[i][0] = x.x, v[i][1] = x.y;
            }
        }
        if constexpr (kTail) {
            const int first = tok0 + pg * kBlockSize, left = held - first, common = all - first;
            uint32_t nan[4] = {};  // by dim
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = (i & 1 ? 7 - t : t) + (i >> 1) * 8;
                // tokens past the end hold anything: zeros
                const bool in = row < left;
#pragma unroll
                for (int w = 0; w < kVWords; ++w) v[i][w] = in ? v[i][w] : 0u;
                if (drafts > 1 && row >= common) {
                    // Of the last tokens, which not every column sees, NaN must reach the
                    // columns that see it only, not as 0 * NaN the others.
#pragma unroll
                    for (int w = 0; w < kVWords; ++w) {
                        const uint32_t is = nan_bytes(v[i][w]);
                        nan[i] |= is << 4 * w;
                        v[i][w] &= ~((is & 1u) * 0xffu | (is >> 1 & 1u) * 0xff00u |
                                     (is >> 2 & 1u) * 0xff0000u | (is >> 3 & 1u) * 0xff000000u);
                    }
                }
            }
            if (drafts > 1 && __any_sync(0xffffffffu, nan[0] | nan[1] | nan[2] | nan[3])) {
#pragma unroll 1
                for (int from = 0; from < 4; ++from) {  // lane of the quad
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t dims = __shfl_sync(0xffffffffu, nan[i], g * 4 + from);
                        const int row = (i & 1 ? 7 - from : from) + (i >> 1) * 8;
                        if (dims == 0) continue;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int k = 0; k < 2; ++k)
                                if (row < lim[nt][k] - first)
#pragma unroll
                                    for (int j = 0; j < kSteps; ++j) {
                                        if (dims >> 2 * j & 1) o[j][nt][k] = NAN;
                                        if (dims >> (2 * j + 1) & 1) o[j][nt][k + 2] = NAN;
                                    }
                    }
                }
            }
        }
#pragma unroll
        for (int w = 0; w < kVWords; ++w) {
            uint32_t a[4], b[4];  // dims 4 w ..: tokens t, 7 - t | 8 + t, 15 - t
            kv8_half4(__byte_perm(v[0][w], v[1][w], 0x5140), a[0], a[1]);
            kv8_half4(__byte_perm(v[0][w], v[1][w], 0x7362), a[2], a[3]);
            kv8_half4(__byte_perm(v[2][w], v[3][w], 0x5140), b[0], b[1]);
            kv8_half4(__byte_perm(v[2][w], v[3][w], 0x7362), b[2], b[3]);
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    mma_f16(o[2 * w + k][nt], a[2 * k], a[2 * k + 1], b[2 * k], b[2 * k + 1], pf[nt][0],
                            pf[nt][1]);
        }
    }
};

}  // namespace
}  // namespace lc

using namespace lc;

extern "C" size_t lc_paged_decode_kv8_workspace_size(int batch, int num_q_heads, int num_kv_heads,
                                                     int head_dim, int tokens_per_seq) {
    return decode_workspace(batch, num_q_heads, num_kv_heads, head_dim, tokens_per_seq);
}

extern "C" int lc_paged_decode_kv8(void *out, int64_t out_stride, const void *q, int64_t q_stride,
                                   const void *kv_pool, int64_t num_blocks, int num_layers,
                                   int layer, int num_q_heads, int num_kv_heads, int head_dim,
                                   const int *block_tables, int table_stride,
                                   const int *context_lens, int len_offset, int batch,
                                   int tokens_per_seq, int max_context_len, float sm_scale,
                                   void *workspace, size_t workspace_bytes, int *dev_status,
                                   lc_stream_t stream) {
    if (!out || !q || !kv_pool || !block_tables || !context_lens) return LC_ERR_INVALID_ARGUMENT;
    DecodeParams p{};
    p.scale_log2 = std::fabs(sm_scale) * 1.4426950408889634f;
    p.q_sign = std::signbit(sm_scale) ? 0x80008000u : 0u;
    p.v_scale = 1.f;
    return decode_stream<Kv8>(p, out, out_stride, q, q_stride, kv_pool, num_blocks, num_layers, layer,
                              num_q_heads, num_kv_heads, head_dim, block_tables, table_stride,
                              context_lens, len_offset, batch, tokens_per_seq, max_context_len,
                              workspace, workspace_bytes, dev_status, stream);
}
