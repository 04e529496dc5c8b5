// norm_rope.cu - per-head RMS norm of queries and keys, rotate-half RoPE and the
// append of K and V, one pass over the qkv rows. K and V go to the bf16 pools
// (lc_qk_norm_rope_append) or to the 4-bit pool (lc_qk_norm_rope_append_kv4).
//
// For a head x of a row at position pos, with bias b and norm weight w (each
// optional), c = cos[pos], s = sin[pos]:
//     u = x + b
//     y = u * (1 / sqrt(mean(u^2) + eps)) * w               (q and k)
//     r[d] = y[d] c[d] - y[d + hd/2] s[d],  r[d + hd/2] = y[d] s[d] + y[d + hd/2] c[d]
// in fp32, rounded once: r of q to bf16 in q_out, r of k and u of v to bf16 or
// to 4 bits (kv4.cuh) in the pool. Every product and sum is rounded by itself
// and the squares are added in a fixed pairwise order (d with d + hd/2, then
// within 8 dims, then across the 8-dim chunks), so that the result does not
// depend on the launch shape: a last-bit difference in front of a 4-bit
// rounding would be a whole step behind it.
//
// hd/16 lanes share a head, each with 8 dims of the first half and their 8
// rotation partners: two 16-byte loads, both halves of a rotation in one
// thread, a reduction of 2 or 3 shuffles. A warp takes kIter times 32 / (hd/16)
// heads of one row and issues all their loads first; the row's cos and sin are
// read once per warp.
#include <cfloat>
#include <climits>

#include "kv4.cuh"
#include "lc_host.h"

namespace lc {
namespace {

constexpr int kNormRopeThreads = 128;

struct NormRopeParams {
    bf16 *q_out;
    int64_t q_out_stride;
    const bf16 *qkv;
    int64_t row_stride;
    int rows;
    const int *positions, *slot_map;
    const bf16 *q_bias, *k_bias, *v_bias;
    const bf16 *q_norm, *k_norm;
    float eps;
    const float *cos_t, *sin_t;
    int rope_rows;
    bf16 *k_pool, *v_pool;  // bf16 pools
    uint8_t *kv_pool;       // 4-bit pool
    float k_scale, v_scale;
    int64_t num_blocks;
    int num_layers, layer, num_q_heads, num_kv_heads;
    int groups;  // warp tasks per row
    int *status;
};

__device__ __forceinline__ void unpack8(const uint4 &u, float (&f)[8]) {
    const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __low2float(h[i]);
        f[2 * i + 1] = __high2float(h[i]);
    }
}

__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]),
                      pack_bf16(f[6], f[7]));
}

__device__ __forceinline__ uint4 ldg16(const bf16 *p) {
    return __ldg(reinterpret_cast<const uint4 *>(p));
}

__device__ __forceinline__ void load8f(const float *p, float (&f)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(p));
    const float4 b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}

// 1 / sqrt(mean of squares + eps) of a head, x1 and x2 its two 8-dim pieces in
// this lane. All lanes of the warp call it.
template <int HD>
__device__ __forceinline__ float rms_factor(const float (&x1)[8], const float (&x2)[8], float eps) {
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
        s[e] = __fadd_rn(__fmul_rn(x1[e], x1[e]), __fmul_rn(x2[e], x2[e]));
#pragma unroll
    for (int w = 4; w >= 1; w >>= 1)
#pragma unroll
        for (int e = 0; e < w; ++e) s[e] = __fadd_rn(s[e], s[e + w]);
    float t = s[0];
#pragma unroll
    for (int w = HD / 32; w >= 1; w >>= 1) t = __fadd_rn(t, __shfl_xor_sync(0xffffffffu, t, w));
    return __frcp_rn(__fsqrt_rn(__fadd_rn(__fmul_rn(t, 1.f / HD), eps)));
}

// Largest magnitude of a 16-dim group (this lane's 8 dims and its neighbour's),
// as float bits: a NaN is larger than every number.
__device__ __forceinline__ uint32_t group_amax(const float (&x)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(x[e]) & 0x7fffffffu);
    return max(m, __shfl_xor_sync(0xffffffffu, m, 1));
}

// kIter: heads a lane works on in one task.
template <int HD, bool KV4, int kIter>
__global__ void __launch_bounds__(kNormRopeThreads) norm_rope_append_kernel(NormRopeParams p) {
    constexpr int kLanes = HD / 16;         // lanes per head
    constexpr int kHeads = 32 / kLanes;     // heads per warp at a time
    constexpr int kHalf = HD / 2;
    const int lane = threadIdx.x & 31;
    const int64_t task = (int64_t)blockIdx.x * (kNormRopeThreads / 32) + (threadIdx.x >> 5);
    if (task >= (int64_t)p.rows * p.groups) return;
    const int row = (int)(task / p.groups);
    const int first = (int)(task - (int64_t)row * p.groups) * kHeads * kIter;
    const int hq = p.num_q_heads, hk = hq + p.num_kv_heads, heads = hk + p.num_kv_heads;
    const int c8 = (lane % kLanes) * 8;
    const int h0 = first + lane / kLanes;

    const bf16 *src = p.qkv + (int64_t)row * p.row_stride + c8;
    uint4 a[kIter], b[kIter];
#pragma unroll
    for (int u = 0; u < kIter; ++u) {
        const int h = h0 + u * kHeads;
        if (h < heads) {
            // plain loads: q_out may be these rows
            a[u] = *reinterpret_cast<const uint4 *>(src + (int64_t)h * HD);
            b[u] = *reinterpret_cast<const uint4 *>(src + (int64_t)h * HD + kHalf);
        } else {
            a[u] = b[u] = make_uint4(0, 0, 0, 0);
        }
    }
    const int pos = __ldg(p.positions + row), slot = __ldg(p.slot_map + row);
    if (pos < 0 || pos >= p.rope_rows) {  // -1: a padding row
        if (pos != -1 && first == 0 && lane == 0) set_status(p.status, LC_DEV_BAD_POS);
        return;
    }
    const bool stored = slot >= 0 && slot < p.num_blocks * kBlockSize;
    if (!stored && slot != -1 && first == 0 && lane == 0) set_status(p.status, LC_DEV_BAD_BLOCK);
    const int phys = slot / kBlockSize, off = slot % kBlockSize;
    float cs[8], sn[8];
    load8f(p.cos_t + (int64_t)pos * kHalf + c8, cs);
    load8f(p.sin_t + (int64_t)pos * kHalf + c8, sn);

#pragma unroll
    for (int u = 0; u < kIter; ++u) {
        const int hw = first + u * kHeads;  // the warp's first head of this turn
        if (hw >= heads) break;
        const int h = h0 + u * kHeads;
        const bool is_q = h < hq, is_v = h >= hk;
        const int hl = is_q ? h : is_v ? h - hk : h - hq;  // head within its part
        float x1[8], x2[8];
        unpack8(a[u], x1);
        unpack8(b[u], x2);
        const bf16 *bias = is_q ? p.q_bias : is_v ? p.v_bias : p.k_bias;
        if (bias && h < heads) {
            float t1[8], t2[8];
            unpack8(ldg16(bias + (int64_t)hl * HD + c8), t1);
            unpack8(ldg16(bias + (int64_t)hl * HD + c8 + kHalf), t2);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x1[e] = __fadd_rn(x1[e], t1[e]);
                x2[e] = __fadd_rn(x2[e], t2[e]);
            }
        }
        if (hw < hk) {  // warp-uniform: some head of this turn is q or k
            const float r = rms_factor<HD>(x1, x2, p.eps);
            const bf16 *w = is_q ? p.q_norm : p.k_norm;
            if (!is_v) {
                if (w) {
                    float t1[8], t2[8];
                    unpack8(ldg16(w + c8), t1);
                    unpack8(ldg16(w + c8 + kHalf), t2);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        x1[e] = __fmul_rn(__fmul_rn(x1[e], r), t1[e]);
                        x2[e] = __fmul_rn(__fmul_rn(x2[e], r), t2[e]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float y1 = x1[e], y2 = x2[e];
                    x1[e] = __fsub_rn(__fmul_rn(y1, cs[e]), __fmul_rn(y2, sn[e]));
                    x2[e] = __fadd_rn(__fmul_rn(y1, sn[e]), __fmul_rn(y2, cs[e]));
                }
            }
        }
        if (is_q) {
            bf16 *dst = p.q_out + (int64_t)row * p.q_out_stride + (int64_t)h * HD + c8;
            *reinterpret_cast<uint4 *>(dst) = pack8(x1);
            *reinterpret_cast<uint4 *>(dst + kHalf) = pack8(x2);
        }
        if (hw + kHeads <= hq) continue;  // warp-uniform: only queries in this turn
        if constexpr (KV4) {
            const float g = is_v ? p.v_scale : p.k_scale;
            const uint32_t s1 = kv4_scale_byte(group_amax(x1), 6.f * g);
            const uint32_t s2 = kv4_scale_byte(group_amax(x2), 6.f * g);
            if (is_q || h >= heads || !stored) continue;
            uint8_t *page = p.kv_pool + kv4_offset(phys, p.layer, hl, p.num_layers,
                                                   p.num_kv_heads, HD) +
                            (is_v ? kv4_half_bytes(HD) : 0);
            uint32_t *codes = reinterpret_cast<uint32_t *>(page + off * (HD / 2) + c8 / 2);
            codes[0] = kv4_codes(x1, e4m3_to_float(s1) * g);
            codes[kHalf / 8] = kv4_codes(x2, e4m3_to_float(s2) * g);
            if ((lane & 1) == 0) {
                uint8_t *sc = page + kv4_code_bytes(HD) + off * (HD / kKv4Group) + c8 / kKv4Group;
                sc[0] = (uint8_t)s1;
                sc[kHalf / kKv4Group] = (uint8_t)s2;
            }
        } else {
            if (is_q || h >= heads || !stored) continue;
            bf16 *dst = (is_v ? p.v_pool : p.k_pool) +
                        (page_row(phys, p.layer, hl, p.num_layers, p.num_kv_heads) + off) * HD + c8;
            *reinterpret_cast<uint4 *>(dst) = pack8(x1);
            *reinterpret_cast<uint4 *>(dst + kHalf) = pack8(x2);
        }
    }
}

template <int HD, bool KV4, int kIter>
int launch_iter(NormRopeParams p, cudaStream_t stream) {
    constexpr int kPer = 32 / (HD / 16) * kIter;
    p.groups = (p.num_q_heads + 2 * p.num_kv_heads + kPer - 1) / kPer;
    const int64_t blocks = ((int64_t)p.rows * p.groups + kNormRopeThreads / 32 - 1) /
                           (kNormRopeThreads / 32);
    if (blocks > INT_MAX) return LC_ERR_INVALID_ARGUMENT;
    norm_rope_append_kernel<HD, KV4, kIter>
        <<<(unsigned)blocks, kNormRopeThreads, 0, stream>>>(p);
    return launch_status();
}

template <bool KV4>
int launch(const NormRopeParams &p, int head_dim, cudaStream_t stream) {
    return head_dim == 64 ? launch_iter<64, KV4, 1>(p, stream)
                          : launch_iter<128, KV4, 1>(p, stream);
}

// The checks both entries share; fills everything but the pools.
int fill(NormRopeParams &p, void *q_out, int64_t q_out_stride, const void *qkv,
         int64_t row_stride, int num_rows, const int *positions, const int *slot_map,
         const void *q_bias, const void *k_bias, const void *v_bias, const void *q_norm,
         const void *k_norm, float eps, const float *cos_cache, const float *sin_cache,
         int rope_rows, int64_t num_blocks, int num_layers, int layer, int num_q_heads,
         int num_kv_heads, int head_dim, int *dev_status) {
    if (!q_out || !qkv || !positions || !slot_map || !cos_cache || !sin_cache)
        return LC_ERR_INVALID_ARGUMENT;
    if (head_dim != 64 && head_dim != 128) return LC_ERR_UNSUPPORTED_HEAD_DIM;
    if (num_rows < 0 || num_layers <= 0 || layer < 0 || layer >= num_layers ||
        num_q_heads <= 0 || num_kv_heads <= 0 || num_blocks <= 0 || rope_rows <= 0 ||
        !(eps >= 0.f) || eps > FLT_MAX)
        return LC_ERR_INVALID_ARGUMENT;
    if (num_blocks > INT_MAX / kBlockSize) return LC_ERR_INVALID_ARGUMENT;  // slots are int32
    if (num_q_heads % num_kv_heads) return LC_ERR_UNSUPPORTED_SHAPE;
    if (row_stride < ((int64_t)num_q_heads + 2 * (int64_t)num_kv_heads) * head_dim ||
        q_out_stride < (int64_t)num_q_heads * head_dim)
        return LC_ERR_INVALID_ARGUMENT;
    if (!aligned16(q_out) || !aligned16(qkv) || (q_out_stride & 7) || (row_stride & 7) ||
        !aligned16(q_bias) || !aligned16(k_bias) || !aligned16(v_bias) || !aligned16(q_norm) ||
        !aligned16(k_norm) || !aligned16(cos_cache) || !aligned16(sin_cache))
        return LC_ERR_MISALIGNED;
    p.q_out = (bf16 *)q_out;
    p.q_out_stride = q_out_stride;
    p.qkv = (const bf16 *)qkv;
    p.row_stride = row_stride;
    p.rows = num_rows;
    p.positions = positions;
    p.slot_map = slot_map;
    p.q_bias = (const bf16 *)q_bias;
    p.k_bias = (const bf16 *)k_bias;
    p.v_bias = (const bf16 *)v_bias;
    p.q_norm = (const bf16 *)q_norm;
    p.k_norm = (const bf16 *)k_norm;
    p.eps = eps;
    p.cos_t = cos_cache;
    p.sin_t = sin_cache;
    p.rope_rows = rope_rows;
    p.num_blocks = num_blocks;
    p.num_layers = num_layers;
    p.layer = layer;
    p.num_q_heads = num_q_heads;
    p.num_kv_heads = num_kv_heads;
    p.status = dev_status;
    return LC_OK;
}

}  // namespace
}  // namespace lc

using namespace lc;

extern "C" int lc_qk_norm_rope_append(
    void *q_out, int64_t q_out_stride, const void *qkv, int64_t row_stride, int num_rows,
    const int *positions, const int *slot_map, const void *q_bias, const void *k_bias,
    const void *v_bias, const void *q_norm, const void *k_norm, float eps,
    const float *cos_cache, const float *sin_cache, int rope_rows, void *k_pool, void *v_pool,
    int64_t num_blocks, int num_layers, int layer, int num_q_heads, int num_kv_heads,
    int head_dim, int *dev_status, lc_stream_t stream) {
    NormRopeParams p{};
    if (!k_pool || !v_pool) return LC_ERR_INVALID_ARGUMENT;
    const int rc = fill(p, q_out, q_out_stride, qkv, row_stride, num_rows, positions, slot_map,
                        q_bias, k_bias, v_bias, q_norm, k_norm, eps, cos_cache, sin_cache,
                        rope_rows, num_blocks, num_layers, layer, num_q_heads, num_kv_heads,
                        head_dim, dev_status);
    if (rc) return rc;
    if (!aligned16(k_pool) || !aligned16(v_pool)) return LC_ERR_MISALIGNED;
    if (num_rows == 0) return LC_OK;
    p.k_pool = (bf16 *)k_pool;
    p.v_pool = (bf16 *)v_pool;
    return launch<false>(p, head_dim, as_stream(stream));
}

extern "C" int lc_qk_norm_rope_append_kv4(
    void *q_out, int64_t q_out_stride, const void *qkv, int64_t row_stride, int num_rows,
    const int *positions, const int *slot_map, const void *q_bias, const void *k_bias,
    const void *v_bias, const void *q_norm, const void *k_norm, float eps,
    const float *cos_cache, const float *sin_cache, int rope_rows, void *kv_pool,
    float k_scale, float v_scale, int64_t num_blocks, int num_layers, int layer,
    int num_q_heads, int num_kv_heads, int head_dim, int *dev_status, lc_stream_t stream) {
    NormRopeParams p{};
    if (!kv_pool || !kv4_scale_ok(k_scale) || !kv4_scale_ok(v_scale))
        return LC_ERR_INVALID_ARGUMENT;
    const int rc = fill(p, q_out, q_out_stride, qkv, row_stride, num_rows, positions, slot_map,
                        q_bias, k_bias, v_bias, q_norm, k_norm, eps, cos_cache, sin_cache,
                        rope_rows, num_blocks, num_layers, layer, num_q_heads, num_kv_heads,
                        head_dim, dev_status);
    if (rc) return rc;
    if (!aligned16(kv_pool)) return LC_ERR_MISALIGNED;
    if (num_rows == 0) return LC_OK;
    p.kv_pool = (uint8_t *)kv_pool;
    p.k_scale = k_scale;
    p.v_scale = v_scale;
    return launch<true>(p, head_dim, as_stream(stream));
}
