// decode_kv4.cu - attention of the newest tokens of each sequence over the 4-bit
// paged cache (kv4.cuh). For query token i of T of sequence b, which holds n
// tokens with them, and query head h of kv head h / (Hq / Hkv):
//     out = softmax_t(q . k_t * sm_scale) . v_t    over t < n - (T - 1 - i)
#include <climits>

#include "kv4.cuh"
#include "lc_host.h"

namespace lc {
namespace {

constexpr int kSimpleWarps = 4;

struct DecodeKv4Params {
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
    float scale_log2, v_scale;
    int *status;
};

template <int HD>
__global__ void __launch_bounds__(kSimpleWarps * 32) decode_kv4_simple_kernel(DecodeKv4Params p) {
    constexpr int kDims = HD / 32;
    __shared__ float s_m[kSimpleWarps], s_l[kSimpleWarps], s_o[kSimpleWarps][HD];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = blockIdx.x, h = blockIdx.y, b = row / p.tokens;
    const int kvh = h / (p.num_q_heads / p.num_kv_heads);
    int n = p.ctx_lens[b] + p.len_offset;
    if (n > p.table_stride * kBlockSize) {
        if (lane == 0) set_status(p.status, LC_DEV_BAD_POS);
        n = p.table_stride * kBlockSize;
    }
    n -= p.tokens - 1 - row % p.tokens;
    float q[kDims], o[kDims] = {}, m = -INFINITY, l = 0.f;
    for (int i = 0; i < kDims; ++i)
        q[i] = __bfloat162float(p.q[row * p.q_stride + h * HD + lane * kDims + i]);
    for (int t = warp; t < n; t += kSimpleWarps) {
        const int phys = p.tables[(int64_t)b * p.table_stride + t / kBlockSize];
        const bool ok = phys >= 0 && phys < p.num_blocks;
        if (!ok && lane == 0) set_status(p.status, LC_DEV_BAD_BLOCK);
        const uint8_t *page = p.kv_pool + kv4_offset(ok ? phys : 0, p.layer, kvh, p.num_layers,
                                                     p.num_kv_heads, HD);
        float kv[2][kDims];
        for (int half = 0; half < 2; ++half) {
            const uint8_t *src = page + half * kv4_half_bytes(HD);
            const int d0 = lane * kDims, tt = t % kBlockSize;
            const float s = e4m3_to_float(src[kv4_code_bytes(HD) + tt * (HD / 16) + d0 / 16]);
            const uint32_t w = reinterpret_cast<const uint32_t *>(src)[(tt * (HD / 2) + d0 / 2) / 4]
                               >> (d0 / 2 % 4 * 8);
            uint32_t hh[4];
            e2m1x8_to_half(w, hh);
            for (int i = 0; i < kDims; ++i) {
                const __half2 v = *reinterpret_cast<__half2 *>(&hh[i / 2]);
                kv[half][i] = ok ? (i & 1 ? __high2float(v) : __low2float(v)) * s : 0.f;
            }
        }
        float x = 0.f;
        for (int i = 0; i < kDims; ++i) x += q[i] * kv[0][i];
        for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
        x *= p.scale_log2;
        const float m2 = fmaxf(m, x);
        const float base = m2 == -INFINITY ? 0.f : m2;
        const float f = exp2f(m - base), e = exp2f(x - base);
        l = l * f + e;
        for (int i = 0; i < kDims; ++i) o[i] = o[i] * f + e * kv[1][i];
        m = m2;
    }
    if (lane == 0) s_m[warp] = m, s_l[warp] = l;
    for (int i = 0; i < kDims; ++i) s_o[warp][lane * kDims + i] = o[i];
    __syncthreads();
    for (int d = threadIdx.x; d < HD; d += kSimpleWarps * 32) {
        float mm = -INFINITY, ll = 0.f, oo = 0.f;
        for (int w = 0; w < kSimpleWarps; ++w) mm = fmaxf(mm, s_m[w]);
        const float base = mm == -INFINITY ? 0.f : mm;
        for (int w = 0; w < kSimpleWarps; ++w) {
            const float f = exp2f(s_m[w] - base);
            ll += s_l[w] * f;
            oo += s_o[w][d] * f;
        }
        p.out[row * p.out_stride + h * HD + d] =
            __float2bfloat16(ll == 0.f ? 0.f : oo / ll * p.v_scale);
    }
}

}  // namespace
}  // namespace lc

using namespace lc;

extern "C" size_t lc_paged_decode_kv4_workspace_size(int batch, int num_q_heads, int num_kv_heads,
                                                     int head_dim, int tokens_per_seq) {
    if (batch <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads ||
        tokens_per_seq <= 0 || (head_dim != 64 && head_dim != 128))
        return 0;
    return 256;
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
    if (head_dim != 64 && head_dim != 128) return LC_ERR_UNSUPPORTED_HEAD_DIM;
    if (batch < 0 || tokens_per_seq <= 0 || num_layers <= 0 || layer < 0 || layer >= num_layers ||
        num_q_heads <= 0 || num_kv_heads <= 0 || num_blocks <= 0 || table_stride <= 0 ||
        max_context_len < 0 || len_offset < 0 || len_offset > 1)
        return LC_ERR_INVALID_ARGUMENT;
    if (num_q_heads % num_kv_heads) return LC_ERR_UNSUPPORTED_SHAPE;
    if (table_stride > INT_MAX / kBlockSize ||
        (int64_t)batch * tokens_per_seq > INT_MAX)
        return LC_ERR_INVALID_ARGUMENT;
    if (q_stride < (int64_t)num_q_heads * head_dim || out_stride < (int64_t)num_q_heads * head_dim)
        return LC_ERR_INVALID_ARGUMENT;
    if (!aligned16(kv_pool) || !aligned16(q) || (q_stride & 7) || ((uintptr_t)out & 1))
        return LC_ERR_MISALIGNED;
    if (batch == 0) return LC_OK;
    if (!workspace || workspace_bytes < lc_paged_decode_kv4_workspace_size(
                                            batch, num_q_heads, num_kv_heads, head_dim,
                                            tokens_per_seq))
        return LC_ERR_WORKSPACE_TOO_SMALL;
    if (!aligned16(workspace)) return LC_ERR_MISALIGNED;
    if (num_q_heads > 65535) return LC_ERR_UNSUPPORTED_SHAPE;
    DecodeKv4Params p{};
    p.out = (bf16 *)out;
    p.out_stride = out_stride;
    p.q = (const bf16 *)q;
    p.q_stride = q_stride;
    p.kv_pool = (const uint8_t *)kv_pool;
    p.num_blocks = num_blocks;
    p.num_layers = num_layers;
    p.layer = layer;
    p.num_q_heads = num_q_heads;
    p.num_kv_heads = num_kv_heads;
    p.tables = block_tables;
    p.table_stride = table_stride;
    p.ctx_lens = context_lens;
    p.len_offset = len_offset;
    p.batch = batch;
    p.tokens = tokens_per_seq;
    p.scale_log2 = sm_scale * k_scale * 1.4426950408889634f;
    p.v_scale = v_scale;
    p.status = dev_status;
    const dim3 grid(batch * tokens_per_seq, num_q_heads);
    if (head_dim == 64)
        decode_kv4_simple_kernel<64><<<grid, kSimpleWarps * 32, 0, as_stream(stream)>>>(p);
    else
        decode_kv4_simple_kernel<128><<<grid, kSimpleWarps * 32, 0, as_stream(stream)>>>(p);
    return launch_status();
}
