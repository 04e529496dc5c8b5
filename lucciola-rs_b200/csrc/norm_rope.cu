// norm_rope.cu - per-head RMS norm of queries and keys, rotate-half RoPE and the
// append of K and V, one pass over the qkv rows. K and V go to the bf16 pools
// (lc_qk_norm_rope_append), to the 4-bit pool (lc_qk_norm_rope_append_kv4) or to the
// 8-bit pool (lc_qk_norm_rope_append_kv8, a kernel of its own further down).
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
// thread, a reduction of 2 or 3 shuffles. A warp takes 32 / (hd/16) heads at a time,
// in the order of the rows and across their ends (18 heads of 64 in turns of 8: 2.25
// per row, not 3; 16384 such rows 18.3 us, 20.8 us with turns that end with the row).
// The grid stays, and a warp loads its next heads before it works on these, so that a
// read's latency (the row, and the position before the cos and sin) is not paid once
// per set of warps that fits the GPU (16384 rows of 12/2 heads of 128: 29.6 us, 32.5 us
// with a warp per turn).
//
// Bounds. Those 16384 rows of 128-dim heads now take 27.9 us: 143 MB at 5.1 TB/s, 78 %
// of a device copy's rate. What is missing are issue slots (counting rows and heads on
// without a division: 29.6 us before); contracted products and sums would save 12
// instructions of a turn, which has some hundreds.
// Into the 4-bit pool (8192 rows of 28/4 heads, 33 us, 66 %) the quotients of K and V
// come on top: 69 % of the issue slots, with the packed operations at half rate. 32
// rows are launch and latency: 2.4 us.
#include <algorithm>
#include <cfloat>
#include <climits>

#include "kv4.cuh"
#include "kv8.cuh"
#include "lc_host.h"

namespace lc {
namespace {

constexpr int kNormRopeThreads = 128;
constexpr int kNormRopeCtas = 7;  // per SM: up to 72 registers

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
    float one;  // 1: see kv4.cuh
    const float *cos_t, *sin_t;
    int rope_rows;
    bf16 *k_pool, *v_pool;  // bf16 pools
    uint8_t *kv_pool;       // 4-bit or 8-bit pool
    float k_scale, v_scale;
    int64_t num_blocks;
    int num_layers, layer, num_q_heads, num_kv_heads;
    int *status;
};

// Eight bf16 values as four pairs, and back with one rounding.
__device__ __forceinline__ void unpack8(const uint4 &u, uint64_t (&f)[4]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        f[i] = pair2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
__device__ __forceinline__ uint4 pack8(const uint64_t (&f)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = split2(f[i]);
        w[i] = pack_bf16(x.x, x.y);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 ldg16(const bf16 *p) {
    return __ldg(reinterpret_cast<const uint4 *>(p));
}

__device__ __forceinline__ void load8f(const float *p, uint64_t (&f)[4]) {
    const ulonglong2 a = __ldg(reinterpret_cast<const ulonglong2 *>(p));
    const ulonglong2 b = __ldg(reinterpret_cast<const ulonglong2 *>(p) + 1);
    f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
}

// 1 / sqrt(mean of squares + eps) of a head, x1 and x2 its two 8-dim pieces in
// this lane. All lanes of the warp call it.
template <int HD>
__device__ __forceinline__ float rms_factor(const uint64_t (&x1)[4], const uint64_t (&x2)[4], float eps,
                                            uint64_t one) {
    uint64_t s[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = fma2(mul2(x1[e], x1[e]), one, mul2(x2[e], x2[e]));
    // dims e and e + 4, then e and e + 2, then the last two
    const float2 r = split2(add2(add2(s[0], s[2]), add2(s[1], s[3])));
    float t = __fadd_rn(r.x, r.y);
#pragma unroll
    for (int w = HD / 32; w >= 1; w >>= 1) t = __fadd_rn(t, __shfl_xor_sync(0xffffffffu, t, w));
    return __frcp_rn(__fsqrt_rn(__fadd_rn(__fmul_rn(t, 1.f / HD), eps)));
}

// Largest magnitude of a 16-dim group (this lane's 8 dims and its neighbour's),
// as float bits: a NaN is larger than every number.
__device__ __forceinline__ uint32_t group_amax(const uint64_t (&x)[4]) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 v = split2(x[e]);
        m = max(m, max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu));
    }
    return max(m, __shfl_xor_sync(0xffffffffu, m, 1));
}

template <int HD, bool KV4>
__global__ void __launch_bounds__(kNormRopeThreads, kNormRopeCtas)
    norm_rope_append_kernel(NormRopeParams p) {
    constexpr int kLanes = HD / 16;      // lanes per head
    constexpr int kHeads = 32 / kLanes;  // heads per warp at a time
    constexpr int kHalf = HD / 2;
    const int lane = threadIdx.x & 31;
    const int hq = p.num_q_heads, hk = hq + p.num_kv_heads, heads = hk + p.num_kv_heads;
    const int c8 = (lane % kLanes) * 8;
    const uint64_t one = pair2(p.one, p.one), minus_one = pair2(-p.one, -p.one);
    // a task: kHeads heads in turn, of one row or of several
    const uint32_t tasks = ((uint32_t)p.rows * heads + kHeads - 1) / kHeads;
    const uint32_t step = gridDim.x * (kNormRopeThreads / 32);

    struct Task {
        uint4 a, b;  // this lane's dims of both halves
        int row, h, pos, slot;
    };
    // Row and head that this lane loads next; a step of the grid moves them on without
    // a division.
    uint32_t task = blockIdx.x * (kNormRopeThreads / 32) + (threadIdx.x >> 5);
    if (task >= tasks) return;
    int row = (int)((task * kHeads + lane / kLanes) / (uint32_t)heads);
    int head = (int)(task * kHeads + lane / kLanes - (uint32_t)row * heads);
    const int step_rows = (int)(step * kHeads / (uint32_t)heads);
    const int step_heads = (int)(step * kHeads - (uint32_t)step_rows * heads);
    auto fetch = [&](Task &k) {
        k.row = row;
        k.h = head;
        row += step_rows;
        head += step_heads;
        if (head >= heads) head -= heads, ++row;
        k.a = k.b = make_uint4(0, 0, 0, 0);
        k.pos = k.slot = -1;
        if (k.row >= p.rows) return;
        // Padding rows too are loaded: waiting for the position first costs 0.2 us of a decode
        // step's 2.4 and 0.5 to 1.1 us of prompts. Plain loads: q_out may be these rows.
        const bf16 *src = p.qkv + (int64_t)k.row * p.row_stride + (int64_t)k.h * HD + c8;
        k.a = *reinterpret_cast<const uint4 *>(src);
        k.b = *reinterpret_cast<const uint4 *>(src + kHalf);
        k.pos = __ldg(p.positions + k.row);
        k.slot = __ldg(p.slot_map + k.row);
    };

    Task next;
    fetch(next);
    for (; task < tasks; task += step) {
        const Task cur = next;
        const int h = cur.h;
        const bool is_q = h < hq, is_v = h >= hk;
        const int hl = is_q ? h : is_v ? h - hk : h - hq;  // head within its part
        const bool live = cur.pos >= 0 && cur.pos < p.rope_rows;  // not: a padding row, or none
        uint64_t cs[4] = {}, sn[4] = {};
        if (live && !is_v) {
            load8f(p.cos_t + (int64_t)cur.pos * kHalf + c8, cs);
            load8f(p.sin_t + (int64_t)cur.pos * kHalf + c8, sn);
        }
        if (task + step < tasks) fetch(next);
        const bool stored = cur.slot >= 0 && cur.slot < p.num_blocks * kBlockSize;
        if (h == 0 && c8 == 0) {  // one lane per row
            if (!live && cur.pos != -1) set_status(p.status, LC_DEV_BAD_POS);
            if (live && !stored && cur.slot != -1) set_status(p.status, LC_DEV_BAD_BLOCK);
        }
        if (!__any_sync(0xffffffffu, live)) continue;
        uint64_t x1[4], x2[4];
        unpack8(cur.a, x1);
        unpack8(cur.b, x2);
        const bf16 *bias = is_q ? p.q_bias : is_v ? p.v_bias : p.k_bias;
        if (bias && live) {
            uint64_t t1[4], t2[4];
            unpack8(ldg16(bias + (int64_t)hl * HD + c8), t1);
            unpack8(ldg16(bias + (int64_t)hl * HD + c8 + kHalf), t2);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x1[e] = add2(x1[e], t1[e]);
                x2[e] = add2(x2[e], t2[e]);
            }
        }
        if (__any_sync(0xffffffffu, !is_v)) {  // some head of this turn is q or k
            const bf16 *w = is_q ? p.q_norm : p.k_norm;
            if (p.q_norm || p.k_norm) {  // for the whole warp: the sum goes across lanes
                const float r = rms_factor<HD>(x1, x2, p.eps, one);
                if (w && !is_v) {
                    const uint64_t rr = pair2(r, r);
                    uint64_t t1[4], t2[4];
                    unpack8(ldg16(w + c8), t1);
                    unpack8(ldg16(w + c8 + kHalf), t2);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x1[e] = mul2(mul2(x1[e], rr), t1[e]);
                        x2[e] = mul2(mul2(x2[e], rr), t2[e]);
                    }
                }
            }
            if (!is_v) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint64_t y1 = x1[e], y2 = x2[e];
                    x1[e] = fma2(mul2(y2, sn[e]), minus_one, mul2(y1, cs[e]));
                    x2[e] = fma2(mul2(y1, sn[e]), one, mul2(y2, cs[e]));
                }
            }
        }
        if (is_q && live) {
            bf16 *dst = p.q_out + (int64_t)cur.row * p.q_out_stride + (int64_t)h * HD + c8;
            *reinterpret_cast<uint4 *>(dst) = pack8(x1);
            *reinterpret_cast<uint4 *>(dst + kHalf) = pack8(x2);
        }
        if (__all_sync(0xffffffffu, is_q)) continue;  // only queries in this turn
        const int phys = cur.slot / kBlockSize, off = cur.slot % kBlockSize;
        if constexpr (KV4) {
            const float g = is_v ? p.v_scale : p.k_scale;
            const uint32_t m1 = group_amax(x1), m2 = group_amax(x2);
            const uint32_t s1 = kv4_scale_byte(m1, 6.f * g), s2 = kv4_scale_byte(m2, 6.f * g);
            if (is_q || !live || !stored) continue;
            uint8_t *page = p.kv_pool + kv4_offset(phys, p.layer, hl, p.num_layers,
                                                   p.num_kv_heads, HD) +
                            (is_v ? kv4_half_bytes(HD) : 0);
            uint32_t *codes = reinterpret_cast<uint32_t *>(page + off * (HD / 2) + c8 / 2);
            codes[0] = kv4_codes(x1, e4m3_to_float(s1) * g, m1);
            codes[kHalf / 8] = kv4_codes(x2, e4m3_to_float(s2) * g, m2);
            if ((lane & 1) == 0) {
                uint8_t *sc = page + kv4_code_bytes(HD) + off * (HD / kKv4Group) + c8 / kKv4Group;
                sc[0] = (uint8_t)s1;
                sc[kHalf / kKv4Group] = (uint8_t)s2;
            }
        } else {
            if (is_q || !live || !stored) continue;
            bf16 *dst = (is_v ? p.v_pool : p.k_pool) +
                        (page_row(phys, p.layer, hl, p.num_layers, p.num_kv_heads) + off) * HD + c8;
            *reinterpret_cast<uint4 *>(dst) = pack8(x1);
            *reinterpret_cast<uint4 *>(dst + kHalf) = pack8(x2);
        }
    }
}

template <int HD, bool KV4>
int launch_dim(NormRopeParams p, cudaStream_t stream) {
    constexpr int kHeads = 32 / (HD / 16), kWarps = kNormRopeThreads / 32;
    // 32-bit head numbers; more heads than that do not fit the memory
    const int64_t total = (int64_t)p.rows * (p.num_q_heads + 2 * p.num_kv_heads);
    if (total > INT_MAX) return LC_ERR_UNSUPPORTED_SHAPE;
    const int64_t tasks = (total + kHeads - 1) / kHeads;
    const int64_t blocks = std::min<int64_t>((tasks + kWarps - 1) / kWarps,
                                             (int64_t)sm_count() * kNormRopeCtas);
    norm_rope_append_kernel<HD, KV4><<<(unsigned)blocks, kNormRopeThreads, 0, stream>>>(p);
    return launch_status();
}

template <bool KV4>
int launch(const NormRopeParams &p, int head_dim, cudaStream_t stream) {
    return head_dim == 64 ? launch_dim<64, KV4>(p, stream) : launch_dim<128, KV4>(p, stream);
}

// ---------------------------------------------------------------- 8-bit pool --
// A page of a kv head has one scale for its 16 tokens, so the rows that a call adds to a
// page are one piece of work: a run, adjacent rows of one page with rising offsets. The
// warp that has the run takes K or V of one head: it goes through the rows once for their
// largest magnitude, which with the page's old scale gives the new one, and once more for
// their codes (append_run); where the scale grew the page's other tokens are moved to it.
// Run starts are found from the slots: a warp looks at `window` rows and works on the runs
// that start there.
//
// The first kv_blocks CTAs do so, the others the queries, as above.
//
// Bounds. 8192 rows of 28/4 heads of 128: 36 us for 147 MB, 62 % of a device copy's rate. 65 %
// of the issue slots are taken: 23.05 M instructions, 313 for four heads of a row, which go to
// unpacking rows and norm weights, to addresses, and to K's and V's second time (three of a
// page's four chunks are loaded and unpacked twice, K's normed and rotated twice). Contracted
// products and sums would save 12 of the 313. Rejected: cos, sin and the norm's weights kept for a row's
// queries (48.0 us with the unpacking, 43.9 so: the registers spill), 5 or 6 CTAs per SM (47.6,
// 45.9). 24 rows are launch and latency: slot -> scale beside the row, 5.7 us from a cold L2.
constexpr int kMaxWindow = 8;  // a run's 16 rows from the last of 8 end within a warp's lanes

template <int HD>
__device__ __forceinline__ void add_bias(const bf16 *bias, uint64_t (&x1)[4], uint64_t (&x2)[4]) {
    uint64_t t1[4], t2[4];
    unpack8(ldg16(bias), t1);
    unpack8(ldg16(bias + HD / 2), t2);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x1[e] = add2(x1[e], t1[e]);
        x2[e] = add2(x2[e], t2[e]);
    }
}

// Norm (w: this lane's weights, or none) and rotation of a head. All lanes of the warp call it.
template <int HD>
__device__ __forceinline__ void norm_rotate(const bf16 *w, float eps, uint64_t one,
                                            uint64_t minus_one, const uint64_t (&cs)[4],
                                            const uint64_t (&sn)[4], uint64_t (&x1)[4],
                                            uint64_t (&x2)[4]) {
    if (w) {
        const float r = rms_factor<HD>(x1, x2, eps, one);
        const uint64_t rr = pair2(r, r);
        uint64_t t1[4], t2[4];
        unpack8(ldg16(w), t1);
        unpack8(ldg16(w + HD / 2), t2);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x1[e] = mul2(mul2(x1[e], rr), t1[e]);
            x2[e] = mul2(mul2(x2[e], rr), t2[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint64_t y1 = x1[e], y2 = x2[e];
        x1[e] = fma2(mul2(y2, sn[e]), minus_one, mul2(y1, cs[e]));
        x2[e] = fma2(mul2(y1, sn[e]), one, mul2(y2, cs[e]));
    }
}

// Largest finite magnitude of eight values as float bits; `odd`: some are not finite.
__device__ __forceinline__ uint32_t finite_amax(const uint64_t (&x)[4], bool &odd) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 v = split2(x[e]);
        const uint32_t a = __float_as_uint(v.x) & 0x7fffffffu, b = __float_as_uint(v.y) & 0x7fffffffu;
        if (a >= 0x7f800000u || b >= 0x7f800000u) odd = true;
        m = max(m, max(a < 0x7f800000u ? a : 0u, b < 0x7f800000u ? b : 0u));
    }
    return m;
}

// Codes of eight values at the scale 1 / `inv`, a power of two; what is not finite is NaN.
__device__ __forceinline__ uint2 kv8_codes(const uint64_t (&x)[4], float inv, bool odd) {
    float y[8];
    const uint64_t ii = pair2(inv, inv);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 v = split2(mul2(x[e], ii));
        y[2 * e] = v.x, y[2 * e + 1] = v.y;
    }
    uint2 c = make_uint2(kv8_codes4(y[0], y[1], y[2], y[3]), kv8_codes4(y[4], y[5], y[6], y[7]));
    if (odd) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (!(fabsf(y[e]) <= FLT_MAX)) (e < 4 ? c.x : c.y) |= kKv8Nan << e % 4 * 8;
    }
    return c;
}

// The rows [r0, r0 + n) of one page, K or V (is_v) of head hl. Lane i of `pos` and `slot`
// holds row r0 - first + i's; all of the run's slots are valid, a row without a place in the
// RoPE tables (pos -1) is left out. The rows come kHeads at a time (a
// chunk) and twice where they are more: once for their largest magnitude, once for their
// codes, the last chunk, whose values are still there, first. Kept in registers, a page's
// values take 64 of them and leave the GPU a third of the warps (8192 rows of 28/4 heads of
// 128: 69 us).
template <int HD>
__device__ __forceinline__ void append_run(const NormRopeParams &p, int r0, int first, int n,
                                           int pos, int slot, bool is_v, int hl) {
    constexpr int kLanes = HD / 16, kHeads = 32 / kLanes, kHalf = HD / 2;
    const int lane = threadIdx.x & 31, c8 = lane % kLanes * 8, grp = lane / kLanes;
    const uint64_t one = pair2(p.one, p.one), minus_one = pair2(-p.one, -p.one);
    const uint32_t live = __ballot_sync(0xffffffffu, pos >= 0) >> first & ((1u << n) - 1);  // by row
    if (live == 0) return;
    const int slot0 = __shfl_sync(0xffffffffu, slot, first + __ffs(live) - 1);
    uint8_t *page = p.kv_pool + kv8_offset(slot0 / kBlockSize, p.layer, hl, p.num_layers,
                                           p.num_kv_heads, HD);
    uint32_t *scale = reinterpret_cast<uint32_t *>(page + 2 * kv8_half_bytes(HD)) + is_v;
    const bool fresh = slot0 % kBlockSize == 0;
    const uint32_t old = fresh ? 0u : *scale;
    page += is_v * kv8_half_bytes(HD);
    const bf16 *src = p.qkv + (int64_t)(r0 + grp) * p.row_stride +
                      (int64_t)(p.num_q_heads + (is_v ? p.num_kv_heads : 0) + hl) * HD + c8;
    const bf16 *bias = is_v ? p.v_bias : p.k_bias;
    if (bias) bias += (int64_t)hl * HD + c8;
    const int last = (n - 1) / kHeads;
    uint4 a, b;
    auto fetch = [&](int c) {
        a = b = make_uint4(0, 0, 0, 0);
        const int i = c * kHeads + grp;
        if (!(live >> i & 1)) return;
        a = *reinterpret_cast<const uint4 *>(src + (int64_t)c * kHeads * p.row_stride);
        b = *reinterpret_cast<const uint4 *>(src + (int64_t)c * kHeads * p.row_stride + kHalf);
    };
    uint64_t x1[4], x2[4];
    // Values of chunk c, whose row is in a and b; then next's row is on its way.
    auto values = [&](int c, int next) {
        const int i = c * kHeads + grp;
        const bool in = live >> i & 1;
        const int row_pos = __shfl_sync(0xffffffffu, pos, min(first + i, 31));
        uint64_t cs[4] = {}, sn[4] = {};
        if (!is_v && in) {
            load8f(p.cos_t + (int64_t)row_pos * kHalf + c8, cs);
            load8f(p.sin_t + (int64_t)row_pos * kHalf + c8, sn);
        }
        unpack8(a, x1);
        unpack8(b, x2);
        if (next >= 0) fetch(next);
        if (bias && in) add_bias<HD>(bias, x1, x2);
        if (!is_v)
            norm_rotate<HD>(p.k_norm ? p.k_norm + c8 : nullptr, p.eps, one, minus_one, cs, sn, x1, x2);
    };
    bool odd = false;
    uint32_t amax = 0;
    fetch(0);
#pragma unroll 1
    for (int c = 0; c <= last; ++c) {
        values(c, c < last ? c + 1 : c - 1);
        amax = max(amax, max(finite_amax(x1, odd), finite_amax(x2, odd)));
    }
    int e = kv8_exponent(__reduce_max_sync(0xffffffffu, amax));
    const int was = kv8_scale_exp(old);
    if (!fresh && was >= e) {
        e = was;
    } else if (!fresh) {  // the other tokens move to the larger scale
        const bool in_run = lane >= first && lane < first + n && pos >= 0;
        const uint32_t run = __reduce_or_sync(0xffffffffu, in_run ? 1u << slot % kBlockSize : 0u);
        const float down = kv8_scale(was - e);
        for (int v = lane; v < HD; v += 32) {  // 16-byte pieces
            if (run >> (v / (HD / 16)) & 1) continue;
            uint4 *at = reinterpret_cast<uint4 *>(page) + v;
            uint4 w = *at;
            w.x = kv8_rescale4(w.x, down), w.y = kv8_rescale4(w.y, down);
            w.z = kv8_rescale4(w.z, down), w.w = kv8_rescale4(w.w, down);
            *at = w;
        }
    }
    if (lane == 0) *scale = __float_as_uint(kv8_scale(e));
    const float inv = kv8_scale(-e);
#pragma unroll 1
    for (int c = last; c >= 0; --c) {
        if (c < last) values(c, c - 1);
        const int i = c * kHeads + grp;
        const int off = __shfl_sync(0xffffffffu, slot, min(first + i, 31)) % kBlockSize;
        if (!(live >> i & 1)) continue;
        uint8_t *to = page + off * HD + c8 % 16;
        *reinterpret_cast<uint2 *>(to + kv8_piece(HD, off, c8 / 16) * 16) = kv8_codes(x1, inv, odd);
        *reinterpret_cast<uint2 *>(to + kv8_piece(HD, off, (c8 + kHalf) / 16) * 16) =
            kv8_codes(x2, inv, odd);
    }
}

constexpr int kMaxTurns = 4;  // of a warp at the queries, with its next heads on their way

template <int HD>
__global__ void __launch_bounds__(kNormRopeThreads, kNormRopeCtas)
    norm_rope_append_kv8_kernel(NormRopeParams p, int window, int kv_blocks, int turns) {
    constexpr int kLanes = HD / 16, kHeads = 32 / kLanes, kHalf = HD / 2;
    constexpr int kWarps = kNormRopeThreads / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // A decode launched to start early waits for the rows itself. (One sequence of 1024 tokens, 14/2
    // heads of 64, append and decode in mode 2: 8.3 us, 9.3 us without; 9.4 us in mode 0.)
    griddep_launch_dependents();
    if ((int)blockIdx.x < kv_blocks) {
        const int kinds = 2 * p.num_kv_heads;
        const uint32_t task = blockIdx.x * kWarps + warp;
        const int kind = (int)(task % kinds);
        const int64_t row0 = (int64_t)(task / kinds) * window;
        if (row0 >= p.rows) return;
        const int64_t row = row0 - 1 + lane;  // lane 0: the row before the window
        int pos = -1, slot = -1;
        if (row >= 0 && row < p.rows) {
            pos = __ldg(p.positions + row);
            slot = __ldg(p.slot_map + row);
        }
        const bool valid = pos != -1 && slot >= 0 && slot < p.num_blocks * kBlockSize;
        if (pos >= p.rope_rows) pos = -1;  // left alone, but within its page's run
        const int page = valid ? slot / kBlockSize : -1;
        const int prev = __shfl_up_sync(0xffffffffu, page, 1);
        const int prev_slot = __shfl_up_sync(0xffffffffu, slot, 1);
        const bool same = lane > 0 && valid && page == prev;
        const uint32_t sames = __ballot_sync(0xffffffffu, same);
        const uint32_t rises = __ballot_sync(0xffffffffu, same && slot > prev_slot);
        uint32_t starts = __ballot_sync(0xffffffffu, valid && !same && lane >= 1 && lane <= window);
        while (starts) {
            const int first = __ffs(starts) - 1;
            starts &= starts - 1;
            const int n = __ffs(~(rises >> (first + 1)));  // 1 .. 16
            // a row of the page that does not rise: it and what follows is left out
            if (kind == 0 && lane == 0 && (sames >> (first + n) & 1))
                set_status(p.status, LC_DEV_BAD_BLOCK);
            append_run<HD>(p, (int)row0 - 1 + first, first, n, pos, slot, kind >= p.num_kv_heads,
                           kind >= p.num_kv_heads ? kind - p.num_kv_heads : kind);
        }
        return;
    }
    // ---- queries, kHeads of a row or of several at a time
    const int c8 = (lane % kLanes) * 8, hq = p.num_q_heads;
    const uint64_t one = pair2(p.one, p.one), minus_one = pair2(-p.one, -p.one);
    const uint32_t total = (uint32_t)p.rows * hq;
    struct Task {
        uint4 a, b;  // this lane's dims of both halves
        int row, h, pos;
    };
    const uint32_t base = ((blockIdx.x - kv_blocks) * kWarps + warp) * turns * kHeads;
    if (base >= total) return;
    int row = (int)((base + lane / kLanes) / (uint32_t)hq);
    int head = (int)(base + lane / kLanes - (uint32_t)row * hq);
    auto fetch = [&](Task &k) {
        k.row = row;
        k.h = head;
        head += kHeads;
        while (head >= hq) head -= hq, ++row;
        k.a = k.b = make_uint4(0, 0, 0, 0);
        k.pos = -1;
        if (k.row >= p.rows) return;
        const bf16 *src = p.qkv + (int64_t)k.row * p.row_stride + (int64_t)k.h * HD + c8;
        k.a = *reinterpret_cast<const uint4 *>(src);
        k.b = *reinterpret_cast<const uint4 *>(src + kHalf);
        k.pos = __ldg(p.positions + k.row);
    };
    Task next;
    fetch(next);
#pragma unroll 1
    for (int turn = 0; turn < turns; ++turn) {
        const Task cur = next;
        const bool live = cur.pos >= 0 && cur.pos < p.rope_rows;
        uint64_t cs[4] = {}, sn[4] = {};
        if (live) {
            load8f(p.cos_t + (int64_t)cur.pos * kHalf + c8, cs);
            load8f(p.sin_t + (int64_t)cur.pos * kHalf + c8, sn);
        }
        if (turn + 1 < turns) fetch(next);
        if (cur.row < p.rows && cur.h == 0 && c8 == 0) {  // one lane per row
            const int slot = __ldg(p.slot_map + cur.row);
            if (!live && cur.pos != -1) set_status(p.status, LC_DEV_BAD_POS);
            if (live && slot != -1 && (slot < 0 || slot >= p.num_blocks * kBlockSize))
                set_status(p.status, LC_DEV_BAD_BLOCK);
        }
        if (!__any_sync(0xffffffffu, live)) continue;
        uint64_t x1[4], x2[4];
        unpack8(cur.a, x1);
        unpack8(cur.b, x2);
        if (live && p.q_bias) add_bias<HD>(p.q_bias + (int64_t)cur.h * HD + c8, x1, x2);
        norm_rotate<HD>(p.q_norm ? p.q_norm + c8 : nullptr, p.eps, one, minus_one, cs, sn, x1, x2);
        if (!live) continue;
        bf16 *dst = p.q_out + (int64_t)cur.row * p.q_out_stride + (int64_t)cur.h * HD + c8;
        *reinterpret_cast<uint4 *>(dst) = pack8(x1);
        *reinterpret_cast<uint4 *>(dst + kHalf) = pack8(x2);
    }
}

template <int HD>
int launch_kv8(const NormRopeParams &p, cudaStream_t stream) {
    constexpr int kHeads = 32 / (HD / 16), kWarps = kNormRopeThreads / 32;
    const int64_t heads = (int64_t)p.num_q_heads + 2 * (int64_t)p.num_kv_heads;
    if (heads > INT_MAX / 2 || (int64_t)p.rows > INT_MAX / 2 / heads) return LC_ERR_UNSUPPORTED_SHAPE;
    // Rows per warp in search of runs. Decode steps have a run in every row, and one row per
    // warp is quickest while there are warps for them; prompts one in 16, and most of such
    // warps would find none.
    const int64_t warps = (int64_t)sm_count() * kNormRopeCtas * kWarps;
    int window = 1;
    while (window < kMaxWindow && (int64_t)p.rows * 2 * p.num_kv_heads > 2 * warps * window) window *= 2;
    const int64_t kv_tasks = ((int64_t)p.rows + window - 1) / window * 2 * p.num_kv_heads;
    // Turns of a warp: several where the reads of the next hide behind this one's work, not
    // where that leaves warps idle (a decode step of 24 rows of 64/8 heads: 5.8 us, 9.9 us with 8).
    int64_t q_tasks = ((int64_t)p.rows * p.num_q_heads + kHeads - 1) / kHeads;
    const int turns = (int)std::max<int64_t>(1, std::min<int64_t>(kMaxTurns, q_tasks / warps));
    q_tasks = (q_tasks + turns - 1) / turns;
    const int64_t kv_blocks = (kv_tasks + kWarps - 1) / kWarps, q_blocks = (q_tasks + kWarps - 1) / kWarps;
    norm_rope_append_kv8_kernel<HD><<<(unsigned)(kv_blocks + q_blocks), kNormRopeThreads, 0, stream>>>(
        p, window, (int)kv_blocks, turns);
    return launch_status();
}

// The checks the entries share; fills everything but the pools.
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
    p.one = 1.f;
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

extern "C" int lc_qk_norm_rope_append_kv8(
    void *q_out, int64_t q_out_stride, const void *qkv, int64_t row_stride, int num_rows,
    const int *positions, const int *slot_map, const void *q_bias, const void *k_bias,
    const void *v_bias, const void *q_norm, const void *k_norm, float eps,
    const float *cos_cache, const float *sin_cache, int rope_rows, void *kv_pool,
    int64_t num_blocks, int num_layers, int layer, int num_q_heads, int num_kv_heads,
    int head_dim, int *dev_status, lc_stream_t stream) {
    NormRopeParams p{};
    if (!kv_pool) return LC_ERR_INVALID_ARGUMENT;
    const int rc = fill(p, q_out, q_out_stride, qkv, row_stride, num_rows, positions, slot_map,
                        q_bias, k_bias, v_bias, q_norm, k_norm, eps, cos_cache, sin_cache,
                        rope_rows, num_blocks, num_layers, layer, num_q_heads, num_kv_heads,
                        head_dim, dev_status);
    if (rc) return rc;
    if (!aligned16(kv_pool)) return LC_ERR_MISALIGNED;
    if (num_rows == 0) return LC_OK;
    p.kv_pool = (uint8_t *)kv_pool;
    return head_dim == 64 ? launch_kv8<64>(p, as_stream(stream)) : launch_kv8<128>(p, as_stream(stream));
}
