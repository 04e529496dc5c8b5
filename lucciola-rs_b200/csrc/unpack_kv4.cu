// unpack_kv4.cu - pages of the 4-bit cache as bf16 pages, so that a prompt that
// continues a cached context attends over it with lc_paged_prefill.
//
// Reads 9 hd and writes 32 hd bytes per page, head and tensor: HBM-bound on the
// writes. A warp takes one half page (K or V of one head); each lane converts
// code words 32 apart, 4 bytes in and 16 bytes out, so that a warp's accesses
// are whole lines on both sides. 4 x 2048 tokens of 4 heads of 128 (21.5 MB): 5.1 us,
// of which 2 are the launch and the two dependent reads (length and table, page).
#include "kv4.cuh"
#include "lc_host.h"

namespace lc {
namespace {

constexpr int kUnpackThreads = 256;

struct UnpackParams {
    bf16 *k_out, *v_out;
    const uint8_t *kv_pool;
    int64_t num_blocks;
    int num_layers, layer, num_kv_heads;
    const int *tables;
    int table_stride;
    const int *ctx_lens;
    int len_offset, batch, pages;  // pages per sequence in the output
    float k_scale, v_scale;
    int *status;
};

template <int HD>
__global__ void __launch_bounds__(kUnpackThreads) unpack_kv4_kernel(UnpackParams p) {
    constexpr int kWords = kv4_code_bytes(HD) / 4, kPer = kWords / 32;
    const int lane = threadIdx.x & 31;
    // task = ((b * pages + page) * heads + head) * 2 + (0: K, 1: V)
    int64_t t = (int64_t)blockIdx.x * (kUnpackThreads / 32) + (threadIdx.x >> 5);
    if (t >= (int64_t)p.batch * p.pages * p.num_kv_heads * 2) return;
    const int is_v = (int)(t & 1);
    t >>= 1;
    const int head = (int)(t % p.num_kv_heads);
    t /= p.num_kv_heads;
    const int page = (int)(t % p.pages), b = (int)(t / p.pages);
    int64_t n = (int64_t)__ldg(p.ctx_lens + b) + p.len_offset;
    if (n > (int64_t)p.pages * kBlockSize) {  // more than the output takes; a table row is no shorter
        if (page == 0 && head == 0 && !is_v && lane == 0) set_status(p.status, LC_DEV_BAD_POS);
        n = (int64_t)p.pages * kBlockSize;
    }
    const int64_t held = n - (int64_t)page * kBlockSize;  // tokens of this page
    if (held <= 0) return;
    const int phys = __ldg(p.tables + (int64_t)b * p.table_stride + page);
    const bool ok = phys >= 0 && phys < p.num_blocks;
    if (!ok && lane == 0) set_status(p.status, LC_DEV_BAD_BLOCK);
    const uint8_t *src = p.kv_pool +
                         kv4_offset(ok ? phys : 0, p.layer, head, p.num_layers, p.num_kv_heads, HD) +
                         is_v * kv4_half_bytes(HD);
    const uint8_t *scales = src + kv4_code_bytes(HD);
    const float g = is_v ? p.v_scale : p.k_scale;
    bf16 *dst = (is_v ? p.v_out : p.k_out) +
                (((int64_t)b * p.pages + page) * p.num_kv_heads + head) * kBlockSize * HD;
    uint32_t w[kPer], s[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int j = lane + 32 * i;  // code word: token j / (HD / 8)
        const bool in = ok && j / (HD / 8) < held;
        w[i] = in ? __ldg(reinterpret_cast<const uint32_t *>(src) + j) : 0u;
        s[i] = in ? __ldg(scales + j / 2) : 0u;  // two words per 16-dim group
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        uint32_t h[4], o[4];
        e2m1x8_to_half(w[i], h);
        const __half2 sc = __float2half2_rn(e4m3_to_float(s[i]));
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 v = __half22float2(__hmul2(*reinterpret_cast<__half2 *>(&h[k]), sc));
            o[k] = pack_bf16(v.x * g, v.y * g);
        }
        reinterpret_cast<uint4 *>(dst)[lane + 32 * i] = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

}  // namespace
}  // namespace lc

using namespace lc;

extern "C" size_t lc_kv4_page_bytes(int head_dim) {
    return head_dim == 64 || head_dim == 128 ? 2 * (size_t)kv4_half_bytes(head_dim) : 0;
}

extern "C" int lc_unpack_kv4(void *k_out, void *v_out, const void *kv_pool, int64_t num_blocks,
                             int num_layers, int layer, int num_kv_heads, int head_dim,
                             const int *block_tables, int table_stride, const int *context_lens,
                             int len_offset, int batch, int max_context_len, float k_scale,
                             float v_scale, int *dev_status, lc_stream_t stream) {
    if (!k_out || !v_out || !kv_pool || !block_tables || !context_lens ||
        !kv4_scale_ok(k_scale) || !kv4_scale_ok(v_scale))
        return LC_ERR_INVALID_ARGUMENT;
    if (head_dim != 64 && head_dim != 128) return LC_ERR_UNSUPPORTED_HEAD_DIM;
    if (batch < 0 || num_layers <= 0 || layer < 0 || layer >= num_layers || num_kv_heads <= 0 ||
        num_blocks <= 0 || table_stride <= 0 || max_context_len < 0 || len_offset < 0 ||
        len_offset > 1)
        return LC_ERR_INVALID_ARGUMENT;
    if (!aligned16(k_out) || !aligned16(v_out) || !aligned16(kv_pool)) return LC_ERR_MISALIGNED;
    if (batch == 0 || max_context_len == 0) return LC_OK;
    // output pages per sequence; a table row holds no more than table_stride of them
    const int pages = (int)(((int64_t)max_context_len + kBlockSize - 1) / kBlockSize);
    if (pages > table_stride) return LC_ERR_INVALID_ARGUMENT;
    UnpackParams p{(bf16 *)k_out, (bf16 *)v_out, (const uint8_t *)kv_pool, num_blocks,
                   num_layers, layer, num_kv_heads, block_tables, table_stride, context_lens,
                   len_offset, batch, pages, k_scale, v_scale, dev_status};
    const int64_t tasks = (int64_t)batch * pages * num_kv_heads * 2;
    const int64_t blocks = (tasks + kUnpackThreads / 32 - 1) / (kUnpackThreads / 32);
    if (blocks > INT32_MAX) return LC_ERR_INVALID_ARGUMENT;
    cudaStream_t s = as_stream(stream);
    if (head_dim == 64)
        unpack_kv4_kernel<64><<<(unsigned)blocks, kUnpackThreads, 0, s>>>(p);
    else
        unpack_kv4_kernel<128><<<(unsigned)blocks, kUnpackThreads, 0, s>>>(p);
    return launch_status();
}
