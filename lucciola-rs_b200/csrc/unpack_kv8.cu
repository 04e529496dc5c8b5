// unpack_kv8.cu - pages of the 8-bit cache as bf16 pages, so that a prompt that
// continues a cached context attends over it with lc_paged_prefill.
//
// Reads 16 hd and writes 32 hd bytes per page, head and tensor: HBM-bound on the writes.
// A warp takes one half page (K or V of one head), a lane eight codes 32 times eight apart, 8
// bytes in and 16 out, so that a warp's stores are whole lines (16 codes and two stores of
// every other 16 bytes: 8.0 us). 4 x 2048 tokens of 4 heads of 128 (25 MB): 5.8 us, 4.3 TB/s;
// 8 x 4096: 19.2 us, 5.2 TB/s.
#include "kv8.cuh"
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
    int *status;
};

template <int HD>
__global__ void __launch_bounds__(kUnpackThreads) unpack_kv8_kernel(UnpackParams p) {
    constexpr int kEighths = HD / 8, kPer = kBlockSize * kEighths / 32;  // eight codes at a time
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
    const uint8_t *src =
        p.kv_pool + kv8_offset(ok ? phys : 0, p.layer, head, p.num_layers, p.num_kv_heads, HD);
    const float scale = kv8_scale(kv8_scale_exp(
        __ldg(reinterpret_cast<const uint32_t *>(src + 2 * kv8_half_bytes(HD)) + is_v)));
    src += is_v * kv8_half_bytes(HD);
    bf16 *dst = (is_v ? p.v_out : p.k_out) +
                (((int64_t)b * p.pages + page) * p.num_kv_heads + head) * kBlockSize * HD;
    uint2 w[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int j = lane + 32 * i, token = j / kEighths;  // eighth j % kEighths of a token
        const int piece = kv8_piece(HD, token, j % kEighths / 2);
        w[i] = make_uint2(0, 0);
        if (ok && token < held)
            w[i] = __ldg(reinterpret_cast<const uint2 *>(src) + token * kEighths + piece * 2 + j % 2);
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const uint32_t c[2] = {w[i].x, w[i].y};
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            uint32_t lo, hi;
            kv8_half4(c[k], lo, hi);
            const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&lo));
            const float2 y = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
            o[2 * k] = pack_bf16(x.x * scale, x.y * scale);
            o[2 * k + 1] = pack_bf16(y.x * scale, y.y * scale);
        }
        reinterpret_cast<uint4 *>(dst)[lane + 32 * i] = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

}  // namespace
}  // namespace lc

using namespace lc;

extern "C" size_t lc_kv8_page_bytes(int head_dim) {
    return head_dim == 64 || head_dim == 128 ? (size_t)kv8_page_bytes(head_dim) : 0;
}

extern "C" int lc_unpack_kv8(void *k_out, void *v_out, const void *kv_pool, int64_t num_blocks,
                             int num_layers, int layer, int num_kv_heads, int head_dim,
                             const int *block_tables, int table_stride, const int *context_lens,
                             int len_offset, int batch, int max_context_len, int *dev_status,
                             lc_stream_t stream) {
    if (!k_out || !v_out || !kv_pool || !block_tables || !context_lens)
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
    const int64_t most = (int64_t)INT32_MAX * (kUnpackThreads / 32) / 2;  // half pages over 2
    if ((int64_t)batch * pages > most / num_kv_heads) return LC_ERR_INVALID_ARGUMENT;
    UnpackParams p{(bf16 *)k_out, (bf16 *)v_out, (const uint8_t *)kv_pool, num_blocks,
                   num_layers, layer, num_kv_heads, block_tables, table_stride, context_lens,
                   len_offset, batch, pages, dev_status};
    const int64_t tasks = (int64_t)batch * pages * num_kv_heads * 2;
    const unsigned blocks = (unsigned)((tasks + kUnpackThreads / 32 - 1) / (kUnpackThreads / 32));
    cudaStream_t s = as_stream(stream);
    if (head_dim == 64)
        unpack_kv8_kernel<64><<<blocks, kUnpackThreads, 0, s>>>(p);
    else
        unpack_kv8_kernel<128><<<blocks, kUnpackThreads, 0, s>>>(p);
    return launch_status();
}
