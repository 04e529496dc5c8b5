// decode_kv8.cu - attention of the newest tokens of each sequence over the 8-bit
// paged cache (kv8.cuh). For query token i of T of sequence b, which holds n
// tokens with them, and query head h of kv head h / (Hq / Hkv):
//     out = softmax_t(q . k_t * sm_scale) . v_t    over t < n - (T - 1 - i)
// in one pass: a running maximum m and sum l per query row, the output rescaled
// when m rises. One warp per query row and head, its lanes over the dims.
#include <climits>
#include <cmath>

#include "kv8.cuh"
#include "lc_host.h"

namespace lc {
namespace {

struct DecodeKv8Params {
    bf16 *out;
    int64_t out_stride;
    const bf16 *q;
    int64_t q_stride;
    const uint8_t *kv_pool;
    int64_t num_blocks;
    int num_layers, layer, num_q_heads, num_kv_heads;
    const int *tables;
    int table_stride;
    const int *ctx_lens;
    int len_offset, batch, tokens;
    float sm_scale;
    int *status;
};

template <int HD>
__global__ void __launch_bounds__(128) decode_kv8_kernel(const DecodeKv8Params p) {
    constexpr int kPer = HD / 32;
    const int lane = threadIdx.x & 31;
    const int64_t task = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (task >= (int64_t)p.batch * p.tokens * p.num_q_heads) return;
    const int h = (int)(task % p.num_q_heads);
    const int64_t row = task / p.num_q_heads;
    const int b = (int)(row / p.tokens), i = (int)(row % p.tokens);
    const int kvh = h / (p.num_q_heads / p.num_kv_heads);
    long long n = (long long)__ldg(p.ctx_lens + b) + p.len_offset;
    if (n > (long long)p.table_stride * kBlockSize) {
        if (h == 0 && i == 0 && lane == 0) set_status(p.status, LC_DEV_BAD_POS);
        n = (long long)p.table_stride * kBlockSize;
    }
    const int seen = (int)max(n - (p.tokens - 1 - i), 0ll);
    float q[kPer], o[kPer], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int d = 0; d < kPer; ++d) {
        q[d] = __bfloat162float(p.q[row * p.q_stride + (int64_t)h * HD + lane * kPer + d]);
        o[d] = 0.f;
    }
    const int piece = lane * kPer / 16, in_piece = lane * kPer % 16;
    for (int t0 = 0; t0 < seen; t0 += kBlockSize) {
        const int phys = __ldg(p.tables + (int64_t)b * p.table_stride + t0 / kBlockSize);
        const bool ok = phys >= 0 && phys < p.num_blocks;
        if (!ok && lane == 0) set_status(p.status, LC_DEV_BAD_BLOCK);
        const uint8_t *page =
            p.kv_pool + kv8_offset(ok ? phys : 0, p.layer, kvh, p.num_layers, p.num_kv_heads, HD);
        const uint32_t *sc = reinterpret_cast<const uint32_t *>(page + 2 * kv8_half_bytes(HD));
        const float ks = kv8_scale(kv8_scale_exp(sc[0])), vs = kv8_scale(kv8_scale_exp(sc[1]));
        for (int t = 0; t < min(kBlockSize, seen - t0); ++t) {
            const uint8_t *at = page + t * HD + kv8_piece(HD, t, piece) * 16 + in_piece;
            float s = 0.f, v[kPer];
#pragma unroll
            for (int d = 0; d < kPer; d += 2) {
                const uint32_t k2 = ok ? kv8_half2(*reinterpret_cast<const uint16_t *>(at + d)) : 0u;
                const uint32_t v2 = ok ? kv8_half2(*reinterpret_cast<const uint16_t *>(
                                             at + kv8_half_bytes(HD) + d)) : 0u;
                const float2 k = __half22float2(*reinterpret_cast<const __half2 *>(&k2));
                const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&v2));
                s = fmaf(q[d], k.x, fmaf(q[d + 1], k.y, s));
                v[d] = x.x * vs, v[d + 1] = x.y * vs;
            }
#pragma unroll
            for (int w = 16; w; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
            s *= ks * p.sm_scale;
            const float top = fmaxf(m, s), off = top == -INFINITY ? 0.f : top;
            const float down = m == -INFINITY ? 0.f : expf(m - top), w = expf(s - off);
            m = top;
            l = fmaf(l, down, w);
#pragma unroll
            for (int d = 0; d < kPer; ++d) o[d] = fmaf(o[d], down, w * v[d]);
        }
    }
    const float r = seen == 0 ? 0.f : 1.f / l;
    bf16 *dst = p.out + row * p.out_stride + (int64_t)h * HD + lane * kPer;
#pragma unroll
    for (int d = 0; d < kPer; ++d) dst[d] = __float2bfloat16(o[d] * r);
}

}  // namespace
}  // namespace lc

using namespace lc;

extern "C" size_t lc_paged_decode_kv8_workspace_size(int batch, int num_q_heads, int num_kv_heads,
                                                     int head_dim, int tokens_per_seq) {
    if (batch <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads ||
        tokens_per_seq <= 0 || (head_dim != 64 && head_dim != 128))
        return 0;
    return 256;
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
    if (head_dim != 64 && head_dim != 128) return LC_ERR_UNSUPPORTED_HEAD_DIM;
    if (batch < 0 || tokens_per_seq <= 0 || num_layers <= 0 || layer < 0 || layer >= num_layers ||
        num_q_heads <= 0 || num_kv_heads <= 0 || num_blocks <= 0 || table_stride <= 0 ||
        max_context_len < 0 || len_offset < 0 || len_offset > 1)
        return LC_ERR_INVALID_ARGUMENT;
    if (num_q_heads % num_kv_heads) return LC_ERR_UNSUPPORTED_SHAPE;
    if (table_stride > INT_MAX / kBlockSize || num_blocks > INT_MAX ||
        (int64_t)batch * tokens_per_seq > INT_MAX / num_q_heads / head_dim)
        return LC_ERR_INVALID_ARGUMENT;
    if (q_stride < (int64_t)num_q_heads * head_dim || out_stride < (int64_t)num_q_heads * head_dim)
        return LC_ERR_INVALID_ARGUMENT;
    if (!aligned16(kv_pool) || !aligned16(q) || (q_stride & 7) || ((uintptr_t)out & 1))
        return LC_ERR_MISALIGNED;
    if (batch == 0) return LC_OK;
    if (!workspace || workspace_bytes < 256) return LC_ERR_WORKSPACE_TOO_SMALL;
    if (!aligned16(workspace)) return LC_ERR_MISALIGNED;
    DecodeKv8Params p{(bf16 *)out, out_stride, (const bf16 *)q, q_stride, (const uint8_t *)kv_pool,
                      num_blocks, num_layers, layer, num_q_heads, num_kv_heads, block_tables,
                      table_stride, context_lens, len_offset, batch, tokens_per_seq, sm_scale,
                      dev_status};
    const int64_t tasks = (int64_t)batch * tokens_per_seq * num_q_heads;
    const unsigned blocks = (unsigned)((tasks + 3) / 4);
    if (head_dim == 64)
        decode_kv8_kernel<64><<<blocks, 128, 0, as_stream(stream)>>>(p);
    else
        decode_kv8_kernel<128><<<blocks, 128, 0, as_stream(stream)>>>(p);
    return launch_status();
}
