// decode_stream.cuh - attention of the newest tokens of each sequence over a paged cache
// whose pages hold K and V of a kv head in one run of bytes (F: Kv4 in decode_kv4.cu, Kv8 in
// decode_kv8.cu). For query token i of T of sequence b, which holds n tokens with them, and
// query head h of kv head h / (Hq / Hkv):
//     out = softmax_t(q . k_t * sm_scale) . v_t    over t < n - (T - 1 - i)
// in one pass: a running maximum m and sum l per query row, the output rescaled
// when m rises.
//
// Split. The T * Hq/Hkv query rows of a kv head are the columns of its products,
// kCols = 8, 16 or 24 at a time; (sequence, kv head, slice of columns) is a segment.
// The pages of all segments form one stream, cut evenly over a persistent grid:
// every CTA moves the same bytes whatever the lengths are. A segment cut across
// CTAs leaves (O, m, l) pieces in the workspace; the CTA that finishes it last
// (arrival counter) joins them in the order of the stream, so the result does
// not depend on timing.
//
// Inside a CTA eight warps compute, taking groups of kGroup pages in turn, each
// from a ring of its own. A loading warp fills the rings, one lane per page of a
// group: one bulk copy brings K and V of the kv head, which lie side by side,
// and full and empty mbarriers per stage join a computing warp to its lanes. Edge
// warps, one for each 8 columns, work a chunk (a CTA's part of one segment) ahead
// and behind: they prepare the next chunk's q as mma operands in shared memory, and
// join the states (O, m, l) that the computing warps leave at a chunk's end, so the
// latency of that end (shared memory, the stores, the arrival counter, the other
// pieces) runs beside the next chunk. The computing warps touch no global memory
// until the CTA's last chunk, whose columns they join themselves, one per warp.
//
// Products, mma.sync m16n8k16 with fp16 operands and fp32 sums:
//     S^T[16 tokens x 8 columns] = K[16 x hd] . Q^T
//     O^T[hd x 8 columns]       += V^T[hd x 16] . P^T
// F::scores and F::values unpack K and V in registers, straight into the operand layout.
// q is scaled by a power of two per row, its largest element to [2^14, 2^15), so that fp16
// holds all of its bits down to 2^-31 of that one: only p is rounded (to fp16, 2^-11) on its
// way into a product, and its powers too are laid towards fp16's upper end (kLift).
// The order of dims within a score's sum is free (F::q_dim), and so is that of the tokens
// within a tile: row r of a 16-token tile is token pi(r), pi(2t) = t, pi(2t + 1) = 7 - t
// (and 8 more for r >= 8), which spreads the token rows over the banks.
#pragma once

#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <type_traits>

#include "lc_common.cuh"
#include "lc_host.h"

namespace lc {
namespace {

// p is 2^(s - m) with m kLift below the largest score when it is set, and may grow by
// 2^kLazy before O and l are rescaled: up to 2^15, so that fp16 keeps 11 bits of p down to
// 2^-21 of the largest, and its last one down to 2^-31.
constexpr float kLift = 7.f, kLazy = 8.f;
constexpr int kQTop = 14;  // exponent of a row's largest element of q

struct DecodeParams {
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
    int group;        // query heads per kv head
    int cols;         // tokens * group
    int slices;       // ceil(cols / kCols)
    int seg_per_seq;  // num_kv_heads * slices
    float scale_log2;  // |sm_scale| * log2(e), and K's factor where the pool has one
    uint32_t q_sign;   // sign of sm_scale, on both halves of an fp16 pair
    float v_scale;     // V's factor, or 1
    int pdl_mode;
    int seg_ctas;   // CTAs of the grid per segment, when there is one sequence
    int seg_alone;  // as many as have an SM each, if an SM takes several
    int *ws_cnt;    // [CTAs][kCols] arrivals, at the CTA of a segment's first piece
    int *ws_group;  // [2][CTAs][kCols] arrivals of a group, at the CTA of its first piece
    float2 *ws_ml;  // [pieces][kCols] m, l
    float *ws_o;    // [pieces][kCols][hd]
    int *status;
};

template <class F, int NT>
struct Cfg {
    static constexpr int HD = F::kDim;
    static constexpr int kGroup = F::template kGroup<NT>;  // pages of one warp at a time
    static constexpr int kCols = 8 * NT;
    // Two warps per scheduler, or four (two CTAs) where O takes few registers: 8 NT for
    // each 32 dims. Ten of 168 registers do not help two tiles (8 sequences of 1024 ..
    // 32768 tokens, 64/8 heads of 128: 61 us, 59 us with eight): two schedulers have three
    // then. Beside them one warp that loads and one per tile for the chunks' ends.
    static constexpr int kWarps = 8;
    static constexpr int kCtasPerSm = NT == 1 ? 2 : 1;
    static constexpr int kEdges = NT;
    static constexpr int kLoadWarp = kWarps, kEdgeWarp = kWarps + 1;
    static constexpr int kThreads = (kWarps + 1 + kEdges) * 32;
    // Three tiles of 128 dims take 210 registers: the four side warps hand theirs over.
    // (The case above with 24 columns: 69 us, 86 us with six warps of 238.) 0: as launched.
    static constexpr int kRegs = NT == 3 && HD == 128 ? 216 : 0, kSideRegs = kRegs ? 72 : 24;
    static_assert(kRegs == 0 || (kEdges == 3 && kWarps * kRegs + 4 * kSideRegs <=
                                                    12 * (65536 / kThreads / 8 * 8)));
    static constexpr int kPage = F::kPage;  // K and V of one kv head
    static constexpr int kStage = kGroup * kPage;
    static constexpr int kRow = HD + 4;  // floats between columns of a warp's state
    static constexpr int kStates = kWarps * kCols * kRow * 4;
    static constexpr int kQ = kCols * HD * 2;  // a chunk's q, fp16 operands
    // Stages per warp: the format's choice beside a second CTA, else what there is room for.
    static constexpr int kStages =
        NT == 1 ? F::kStages : (224 * 1024 - kStates - 2 * kQ) / (kWarps * kStage);
    static_assert(kStages >= 2 && kGroup * kWarps <= 32);
    static constexpr int kRing = kWarps * kStages * kStage;
    static constexpr int kSmem = kRing + kStates + 2 * kQ;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<__half2 *>(&a), *reinterpret_cast<__half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}

// Both halves of `a` replaced by its low or its high one.
__device__ __forceinline__ uint32_t both_low(uint32_t a) {
    const __half2 r = __low2half2(*reinterpret_cast<__half2 *>(&a));
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t both_high(uint32_t a) {
    const __half2 r = __high2half2(*reinterpret_cast<__half2 *>(&a));
    return *reinterpret_cast<const uint32_t *>(&r);
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same without a sum to add to.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes,
                                          uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
        ::"r"(dst), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ bool test_wait(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 q, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

__device__ __forceinline__ int tokens_of(const DecodeParams &p, int b, bool report) {
    const long long n = (long long)__ldg(p.ctx_lens + b) + p.len_offset;
    const int cap = p.table_stride * kBlockSize;
    if (n > cap) {
        if (report) set_status(p.status, LC_DEV_BAD_POS);
        return cap;
    }
    return n < 0 ? 0 : (int)n;
}
__device__ __forceinline__ int pages_of(int tokens) {
    return (tokens + kBlockSize - 1) / kBlockSize;
}

// Units of one segment in the stream: its pages and, before them, F::kEdgeUnits without a
// page, about what a chunk's two ends cost in page times; without them a CTA whose pages
// lie in many short segments takes longer than the others. A single sequence fills no CTA
// with several segments and has none.
template <class F>
__device__ __forceinline__ int edge_units(const DecodeParams &p) {
    return p.batch > 1 ? F::kEdgeUnits : 0;
}
template <class F>
__device__ __forceinline__ int units_of(const DecodeParams &p, int tokens) {
    return tokens > 0 ? pages_of(tokens) + edge_units<F>(p) : 0;
}

// CTAs that share the stream, of the grid's. `pages`: those of a segment when there is
// one sequence.
template <class F>
__device__ __forceinline__ int ctas_of(const DecodeParams &p, int total, int pages) {
    // One sequence: as many CTAs for each segment, so that none of them joins two in
    // turn, and no more than the rounds of groups ask for that the fullest one works
    // through. (4-bit pages, 28/4 heads of 128, 12345 tokens: 196 CTAs of 16 pages 11.3 us, 296 of 10
    // or 11 14.3 us; 32768 tokens: 256 of 32 14.3 us, 296 of 28 14.7 us.) From the fifth
    // round on a full grid does as well or better (100000 tokens, 64/8 heads: 32.4 us, 33.3
    // us in rounds).
    if (p.batch == 1 && p.seg_ctas > 0) {
        // Before SMs get a second one, CTAs take up to F::kAlonePages.
        if constexpr (F::kAlonePages > 0) {
#pragma unroll
            for (int n = F::kMinPages; n <= F::kAlonePages; n += 8)
                if (pages <= n * p.seg_alone)
                    return max(1, (int)((unsigned)(pages + n - 1) / (unsigned)n) * p.seg_per_seq);
        }
        int each = p.seg_ctas;
        for (int r = 1; r <= 4; ++r) {
            if (pages > F::kMinPages * r * p.seg_ctas) continue;
            each = r == 1 ? (pages + F::kMinPages - 1) / F::kMinPages
                          : (int)((unsigned)(pages + F::kMinPages * r - 1) / (unsigned)(F::kMinPages * r));
            break;
        }
        return max(1, each * p.seg_per_seq);
    }
    return max(1, min((int)gridDim.x, (total + F::kMinPages - 1) / F::kMinPages));
}

// The stream over `ctas` CTAs: CTA c takes the units from total * c / ctas on.
struct Cut {
    int total, ctas;
    // In 32 bits where the products fit: a 64-bit division costs a good part of a
    // microsecond before the first load.
    __device__ __forceinline__ int start(int cta) const {
        if (total < (1 << 22)) return (int)((unsigned)total * (unsigned)cta / (unsigned)ctas);
        return (int)((long long)total * cta / ctas);
    }
    __device__ __forceinline__ int owner(int unit) const {
        if (total < (1 << 22))
            return (int)((((unsigned)unit + 1u) * (unsigned)ctas - 1u) / (unsigned)total);
        return (int)((((long long)unit + 1) * ctas - 1) / total);
    }
};

// Where a walk over a CTA's range of the stream stands: the chunk, pages
// [p0, p0 + take) of segment seg of sequence b, which holds n tokens and starts
// at unit seg_at.
template <class F>
struct Walk {
    int b, seg, p0, take, n;
    int seg_at;
    int unit;  // next unit of the stream

    __device__ __forceinline__ void start(const DecodeParams &p, int first, int b0, int before_b0) {
        b = b0;
        n = tokens_of(p, b, false);
        const int units = units_of<F>(p, n);  // not zero
        // by steps: there are few segments, and the first load waits for this
        seg = 0, seg_at = before_b0;
        if (p.seg_per_seq <= 8) {
            for (; first >= seg_at + units; ++seg) seg_at += units;
        } else {
            seg = (first - before_b0) / units;
            seg_at += seg * units;
        }
        unit = first;
        p0 = take = 0;
    }
    // Moves to the next chunk of [.., end); false when there is none.
    __device__ __forceinline__ bool next(const DecodeParams &p, int end) {
        while (unit < end) {
            const int units = units_of<F>(p, n);
            if (unit >= seg_at + units) {  // the segment is done (or the sequence is empty)
                seg_at += units;
                if (units == 0 || ++seg == p.seg_per_seq) {
                    seg = 0;
                    n = tokens_of(p, ++b, false);
                }
                continue;
            }
            const int pages_at = seg_at + edge_units<F>(p), stop = min(seg_at + units, end);
            p0 = max(unit - pages_at, 0);
            take = stop - pages_at - p0;
            unit = stop;
            if (take > 0) return true;
        }
        return false;
    }
};

// The kv head of a segment, without the division in the ordinary case.
__device__ __forceinline__ int kv_head(const DecodeParams &p, int seg) {
    return p.slices == 1 ? seg : seg / p.slices;
}

// What the edge warp tells the computing warps about a chunk.
struct ChunkInfo {
    int b, seg, p0, take, n, seg_at, last;
};

template <class F, int NT>
struct Joined {  // one column of a chunk, this lane's dims
    static constexpr int kPer = F::kDim / 32;
    float m, l, o[kPer];
};

// Joins the warps' states for column c of a chunk.
template <class F, int NT>
__device__ __forceinline__ void join_states(const float2 (*ml_of)[Cfg<F, NT>::kCols],
                                            const float *states, int c, int lane,
                                            Joined<F, NT> &j) {
    using C = Cfg<F, NT>;
    constexpr int kWarps = C::kWarps;
    float2 ml[kWarps];
    j.m = -INFINITY, j.l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        ml[w] = ml_of[w][c];
        j.m = fmaxf(j.m, ml[w].x);
    }
#pragma unroll
    for (int i = 0; i < j.kPer; ++i) j.o[i] = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (ml[w].x == -INFINITY) continue;  // saw nothing of this column
        const float r = ex2(ml[w].x - j.m);
        j.l = fmaf(ml[w].y, r, j.l);
        const float *src = states + (w * C::kCols + c) * C::kRow + lane * j.kPer;
#pragma unroll
        for (int i = 0; i < j.kPer; ++i) j.o[i] = fmaf(src[i], r, j.o[i]);
    }
}

// This lane's dims of an output row, o * r.
template <int kPer>
__device__ __forceinline__ void store_row(bf16 *dst, const float (&o)[kPer], float r) {
    uint32_t v[kPer / 2];
#pragma unroll
    for (int i = 0; i < kPer / 2; ++i) v[i] = pack_bf16(o[2 * i] * r, o[2 * i + 1] * r);
    if ((reinterpret_cast<uintptr_t>(dst) & (2 * kPer - 1)) == 0) {
        if constexpr (kPer == 4)
            *reinterpret_cast<uint2 *>(dst) = make_uint2(v[0], v[1]);
        else
            *reinterpret_cast<uint32_t *>(dst) = v[0];
    } else {
        uint16_t *e = reinterpret_cast<uint16_t *>(dst);
#pragma unroll
        for (int i = 0; i < kPer; ++i) e[i] = (uint16_t)(v[i / 2] >> (i % 2 * 16));
    }
}

// The output row of column c of a chunk from its joined state.
template <class F, int NT>
__device__ __forceinline__ void write_row(const DecodeParams &p, const ChunkInfo &ch, int c,
                                          int lane, const Joined<F, NT> &j) {
    constexpr int HD = F::kDim, kPer = HD / 32;
    const int kvh = kv_head(p, ch.seg), col = (ch.seg - kvh * p.slices) * Cfg<F, NT>::kCols + c;
    if (col >= p.cols) return;
    const int qi = col / p.group, h = col - qi * p.group;
    // A row without tokens gets zeros; one whose scores are all -inf has l = 0 too, and
    // its 0 / 0 stays NaN. (Asking for the length alone costs the products 1.5 %: ptxas
    // spills other registers then.)
    const float r = j.l == 0.f && ch.n <= p.tokens - 1 - qi ? 0.f : p.v_scale / j.l;
    bf16 *dst = p.out + ((int64_t)ch.b * p.tokens + qi) * p.out_stride +
                (int64_t)(kvh * p.group + h) * HD + lane * kPer;
    store_row(dst, j.o, r);
}

// A chunk that is a part of its segment leaves a piece per column, at the place
// of its segment and CTA.
template <class F, int NT>
__device__ __forceinline__ void store_piece(const DecodeParams &p, int64_t place, int c, int lane,
                                            const Joined<F, NT> &j) {
    constexpr int HD = F::kDim, kCols = Cfg<F, NT>::kCols, kPer = HD / 32;
    float *po = p.ws_o + (place * kCols + c) * HD + lane * kPer;
    if constexpr (kPer == 4)
        *reinterpret_cast<float4 *>(po) = make_float4(j.o[0], j.o[1], j.o[2], j.o[3]);
    else
        *reinterpret_cast<float2 *>(po) = make_float2(j.o[0], j.o[1]);
    if (lane == 0) p.ws_ml[place * kCols + c] = make_float2(j.m, j.l);
}

// Joins the warps' states for an edge warp's columns of a chunk and stores rows or pieces. A
// lane works out one column's maximum, sum, the warps' factors and the place of its row, for
// all columns at once; then they are joined one by one, the lanes over the dims. (By
// join_states and write_row, column after column, it took 2 to 4 us, which short chunks
// waited for: 256 sequences of 100 .. 300 tokens, 28/4 heads of 128, 8-bit pages, 24.4 us
// like this, 27.9 us.)
template <class F, int NT>
__device__ __forceinline__ void join_columns(const DecodeParams &p, const ChunkInfo &ch, bool whole,
                                             int64_t place, int edge, int lane,
                                             const float2 (*ml_of)[Cfg<F, NT>::kCols],
                                             const float *states) {
    using C = Cfg<F, NT>;
    constexpr int HD = F::kDim, kPer = HD / 32, kWarps = C::kWarps, kEdges = C::kEdges;
    const int own = edge + kEdges * (lane & 7);  // this lane's column
    float2 ml[kWarps];
    float m = -INFINITY, l = 0.f, r[kWarps], scale = 0.f;
    uint32_t seen = 0;
    int64_t row = -1;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        ml[w] = ml_of[w][own];
        m = fmaxf(m, ml[w].x);
    }
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        const bool some = ml[w].x != -INFINITY;  // not: saw nothing of this column
        r[w] = some ? ex2(ml[w].x - m) : 0.f;
        if (some) l = fmaf(ml[w].y, r[w], l);
        seen |= (uint32_t)some << w;
    }
    if (whole) {  // as in write_row
        const int kvh = kv_head(p, ch.seg), col = (ch.seg - kvh * p.slices) * C::kCols + own;
        if (col < p.cols) {
            const int qi = col / p.group, h = col - qi * p.group;
            scale = l == 0.f && ch.n <= p.tokens - 1 - qi ? 0.f : p.v_scale / l;
            row = ((int64_t)ch.b * p.tokens + qi) * p.out_stride + (int64_t)(kvh * p.group + h) * HD;
        }
    }
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
        const int c = edge + kEdges * i;
        const uint32_t see = __shfl_sync(0xffffffffu, seen, i);
        // all reads first
        float x[kWarps][kPer];
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float *src = states + (w * C::kCols + c) * C::kRow + lane * kPer;
            if constexpr (kPer == 4) {
                const float4 v = *reinterpret_cast<const float4 *>(src);
                x[w][0] = v.x, x[w][1] = v.y, x[w][2] = v.z, x[w][3] = v.w;
            } else {
                const float2 v = *reinterpret_cast<const float2 *>(src);
                x[w][0] = v.x, x[w][1] = v.y;
            }
        }
        Joined<F, NT> j;
#pragma unroll
        for (int d = 0; d < kPer; ++d) j.o[d] = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float rw = __shfl_sync(0xffffffffu, r[w], i);
            const bool some = see >> w & 1;
#pragma unroll
            for (int d = 0; d < kPer; ++d) j.o[d] = some ? fmaf(x[w][d], rw, j.o[d]) : j.o[d];
        }
        if (whole) {
            const int64_t at = __shfl_sync(0xffffffffu, row, i);
            const float by = __shfl_sync(0xffffffffu, scale, i);
            if (at >= 0) store_row(p.out + at + lane * kPer, j.o, by);
        } else {
            j.m = __shfl_sync(0xffffffffu, m, i);
            j.l = __shfl_sync(0xffffffffu, l, i);
            store_piece<F, NT>(p, place, c, lane, j);
        }
    }
}

// Pieces are joined by the warp that leaves the last one: up to kTreePieces at once,
// more in groups of kTreeGroup, whose results take the place of their first piece and
// are joined by the group that ends last, so that one CTA does not read them all.
// Groups and orders are those of the stream. (One sequence of 32768 tokens, 28/4 heads
// of 128, 64 pieces per column: 14.3 us, 16.8 us joined by one; 12345 tokens, 49: 11.3,
// 13.6.)
constexpr int kTreePieces = 32, kTreeGroup = 8;

// Counts piece `mine` (or, `top`, a joined group) of column c of the segment whose first
// piece is CTA c0's; true for the last one of its group or segment. One lane, after the
// warp's stores and a __syncwarp.
//
// A counter's place is that of a CTA, not of a segment, so that the counters take the same
// room in a call of any shape and no call's pieces lie on another's counters. One place
// per CTA is enough: a CTA holds at most one piece that begins a segment (its last chunk)
// and one that does not (its first chunk), and so the first piece of at most one group
// that begins a segment and of one that does not.
template <int kCols>
__device__ __forceinline__ bool last_piece(const DecodeParams &p, int c0, int pieces, int mine,
                                           int c, bool top) {
    int *cnt = p.ws_cnt + c0 * kCols + c;
    int count = pieces;
    if (pieces > kTreePieces) {
        const int first = mine / kTreeGroup * kTreeGroup;
        count = top ? (pieces + kTreeGroup - 1) / kTreeGroup : min(kTreeGroup, pieces - first);
        if (!top) cnt = p.ws_group + ((first ? 0 : (int)gridDim.x) + c0 + first) * kCols + c;
    }
    if (atom_add_acq_rel_gpu(cnt, 1) != count - 1) return false;
    *cnt = 0;  // ready for the next call
    return true;
}

// 16 bytes from L2, after the waits before it.
__device__ __forceinline__ uint4 load_l2(const void *src) {
    uint4 v;
    asm volatile("ld.global.cg.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(src)
                 : "memory");
    return v;
}

__device__ __forceinline__ void cp_async16(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src)
                 : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() {
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// Joins `pieces` pieces of column c, at `place` and `stride` apart, in order. Up to
// eight come in one round of reads to registers, more through `buf`, 8 KB of this
// warp's own, 16 (32 at hd 64) at a time.
template <class F, int NT>
__device__ __forceinline__ void join_pieces(const DecodeParams &p, int64_t place, int pieces,
                                            int stride, int c, int lane, float *buf,
                                            Joined<F, NT> &j) {
    constexpr int HD = F::kDim, kCols = Cfg<F, NT>::kCols, kPer = HD / 32;
    const float2 *bml = p.ws_ml + place * kCols + c;
    const float *bo = p.ws_o + (place * kCols + c) * HD;
    const int apart = stride * kCols;
    j.m = -INFINITY, j.l = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) j.o[i] = 0.f;
    constexpr int kFew = 8;
    if (pieces <= kFew) {
        float2 ml[kFew];
        float x[kFew][kPer];
#pragma unroll
        for (int i = 0; i < kFew; ++i) {
            ml[i] = make_float2(-INFINITY, 0.f);
            if (i >= pieces) continue;
            const float *src = bo + (int64_t)i * apart * HD + lane * kPer;
            ml[i] = __ldcg(&bml[i * apart]);
            if constexpr (kPer == 4) {
                const float4 v = __ldcg(reinterpret_cast<const float4 *>(src));
                x[i][0] = v.x, x[i][1] = v.y, x[i][2] = v.z, x[i][3] = v.w;
            } else {
                const float2 v = __ldcg(reinterpret_cast<const float2 *>(src));
                x[i][0] = v.x, x[i][1] = v.y;
            }
        }
#pragma unroll
        for (int i = 0; i < kFew; ++i) j.m = fmaxf(j.m, ml[i].x);
#pragma unroll
        for (int i = 0; i < kFew; ++i) {
            if (ml[i].x == -INFINITY) continue;
            const float r = ex2(ml[i].x - j.m);
            j.l = fmaf(ml[i].y, r, j.l);
#pragma unroll
            for (int d = 0; d < kPer; ++d) j.o[d] = fmaf(x[i][d], r, j.o[d]);
        }
        return;
    }
    constexpr int kRows = 2048 / HD, kLanes = HD / 4;  // pieces at a time, lanes per piece
    auto read = [&](int k0) {
#pragma unroll
        for (int i = 0; i < kRows; i += 32 / kLanes) {
            const int row = i + lane / kLanes, at = lane % kLanes * 4;
            if (k0 + row < pieces)
                cp_async16(buf + row * HD + at, bo + (int64_t)(k0 + row) * apart * HD + at);
        }
    };
    read(0);
    float2 ml = make_float2(-INFINITY, 0.f);  // of piece lane, then lane + 32, ..
    if (lane < pieces) ml = __ldcg(&bml[lane * apart]);
    j.m = ml.x;
    for (int k = lane + 32; k < pieces; k += 32) j.m = fmaxf(j.m, __ldcg(&bml[k * apart].x));
#pragma unroll
    for (int d = 16; d; d >>= 1) j.m = fmaxf(j.m, __shfl_xor_sync(0xffffffffu, j.m, d));
    for (int k0 = 0; k0 < pieces; k0 += kRows) {
        if (k0 > 0 && k0 % 32 == 0) {
            ml = make_float2(-INFINITY, 0.f);
            if (k0 + lane < pieces) ml = __ldcg(&bml[(k0 + lane) * apart]);
        }
        const float r = ml.x == -INFINITY ? 0.f : ex2(ml.x - j.m);
        const uint32_t seen = __ballot_sync(0xffffffffu, ml.x != -INFINITY);
        cp_async_wait_all();
        __syncwarp();
        const int rows = min(kRows, pieces - k0);
#pragma unroll 4
        for (int i = 0; i < rows; ++i) {
            const int from = (k0 + i) % 32;
            const float ri = __shfl_sync(0xffffffffu, r, from);
            const float li = __shfl_sync(0xffffffffu, ml.y, from);
            if (!(seen >> from & 1)) continue;
            j.l = fmaf(li, ri, j.l);
            const float *x = buf + i * HD + lane * kPer;
#pragma unroll
            for (int d = 0; d < kPer; ++d) j.o[d] = fmaf(x[d], ri, j.o[d]);
        }
        __syncwarp();
        if (k0 + kRows < pieces) read(k0 + kRows);
    }
}

// After the last piece of this warp's column (or of its group): true when j holds all of it.
template <class F, int NT>
__device__ __forceinline__ bool finish_column(const DecodeParams &p, int64_t seg, int c0,
                                              int pieces, int mine, int c, int lane, float *buf,
                                              Joined<F, NT> &j) {
    if (pieces <= kTreePieces) {
        join_pieces<F, NT>(p, seg + c0, pieces, 1, c, lane, buf, j);
        return true;
    }
    const int first = mine / kTreeGroup * kTreeGroup;
    join_pieces<F, NT>(p, seg + c0 + first, min(kTreeGroup, pieces - first), 1, c, lane, buf, j);
    store_piece<F, NT>(p, seg + c0 + first, c, lane, j);
    __syncwarp();
    const int last = lane == 0 && last_piece<Cfg<F, NT>::kCols>(p, c0, pieces, mine, c, true);
    if (!__shfl_sync(0xffffffffu, last, 0)) return false;
    __syncwarp();  // lane 0's count saw the groups; now the other lanes' reads do
    join_pieces<F, NT>(p, seg + c0, (pieces + kTreeGroup - 1) / kTreeGroup, kTreeGroup, c, lane, buf,
                        j);
    return true;
}

// The pieces of a chunk's segment: the CTA of the first one, and how many.
template <class F>
__device__ __forceinline__ int pieces_of(const DecodeParams &p, const Cut &cut,
                                         const ChunkInfo &ch, int &c0) {
    const int first = ch.seg_at + edge_units<F>(p);
    c0 = cut.owner(first);
    return cut.owner(first + pages_of(ch.n) - 1) - c0 + 1;
}

template <class F, int NT>
__global__ void __launch_bounds__(Cfg<F, NT>::kThreads, Cfg<F, NT>::kCtasPerSm)
    decode_stream_kernel(const DecodeParams p) {
    using C = Cfg<F, NT>;
    constexpr int HD = F::kDim, kGroup = C::kGroup;
    constexpr int kCols = C::kCols, kWarps = C::kWarps;
    constexpr int kLoadWarp = C::kLoadWarp, kEdgeWarp = C::kEdgeWarp, kEdges = C::kEdges;
    constexpr int kSteps = HD / 16;   // k-steps of S, m-tiles of O
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t full[kWarps][C::kStages], empty[kWarps][C::kStages];
    __shared__ __align__(8) uint64_t q_full[2], states_full, states_empty, edge_done;
    __shared__ ChunkInfo s_chunk[2];
    // Columns of the CTA's first chunk whose last piece it was, to be joined at the end.
    __shared__ ChunkInfo s_left;
    __shared__ uint32_t s_left_cols;
    __shared__ float s_f[2][kCols];
    __shared__ float2 s_ml[kWarps][kCols];
    __shared__ int s_abort;
    __shared__ Cut s_cut;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int cta = blockIdx.x;
    float *states = reinterpret_cast<float *>(smem + C::kRing);  // [kWarps][kCols][kRow]
    uint8_t *q_ops = smem + C::kRing + C::kStates;               // [2][NT][kSteps][32 lanes] 8 bytes
    if (p.pdl_mode > 0) {
        griddep_launch_dependents();
        if (p.pdl_mode == 1) griddep_wait();
    }
    // The side warps need the lengths first: their reads go out before the barriers are set up.
    int mine = 0;  // units of this lane's sequences
    const int per = (p.batch + 31) / 32;
    const int q0 = min(p.batch, lane * per), q1 = min(p.batch, q0 + per);
    if (warp >= kWarps)
        for (int b = q0; b < q1; ++b)
            mine += units_of<F>(p, tokens_of(p, b, cta == 0 && warp == kEdgeWarp));
    if (warp < kWarps && lane < C::kStages) {
        mbar_init(&full[warp][lane], kGroup);
        mbar_init(&empty[warp][lane], 1);
    }
    if (tid == 0) {
        mbar_init(&q_full[0], C::kEdges);
        mbar_init(&q_full[1], C::kEdges);
        mbar_init(&states_full, kWarps);
        mbar_init(&states_empty, C::kEdges);
        mbar_init(&edge_done, C::kEdges);
        s_abort = 0;
        s_left_cols = 0;
    }
    fence_barrier_init();
    __syncthreads();

    // ---- the side warps: the stream's length, this CTA's range of it and the
    // sequence that it starts in
    if (warp >= kWarps) {
        if constexpr (C::kRegs != 0)
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kSideRegs));
        int first = 0, end = 0, b0 = 0, before = 0;
        const int pages = __shfl_sync(0xffffffffu, mine, 0);
        mine *= p.seg_per_seq;
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += u;
        }
        const int total = __shfl_sync(0xffffffffu, upto, 31);
        const Cut cut{total, ctas_of<F>(p, total, pages)};
        if (cta < cut.ctas) {
            first = cut.start(cta);
            end = cut.start(cta + 1);
        }
        if (first < end) {
            const int at = __ffs(__ballot_sync(0xffffffffu, upto > first)) - 1;
            before = __shfl_sync(0xffffffffu, upto - mine, at);
            for (b0 = at * per;; ++b0) {
                const int k = units_of<F>(p, tokens_of(p, b0, false)) * p.seg_per_seq;
                if (first < before + k) break;
                before += k;
            }
        }
        if (p.pdl_mode == 2) griddep_wait();

        if (warp == kLoadWarp) {
            // ---- loads: lane 2 w + k brings page k of each of warp w's groups, which are
            // group w, w + kWarps, ... of every chunk
            if (first >= end) return;
            const int w = lane / kGroup, k = lane % kGroup;
            const int64_t page_stride = F::offset(1, 0, 0, p.num_layers, p.num_kv_heads);
            const uint32_t dst0 = smem_u32(smem) + w * C::kStages * C::kStage + k * C::kPage;
            Walk<F> lw;
            lw.start(p, first, b0, before);
            bool more = lane < kGroup * kWarps && lw.next(p, end);
            int base = w * kGroup;  // first page of the next group, within its chunk
            int phys = -1;          // this lane's table entry in it, -1: no page
            const uint8_t *head = nullptr;
            auto advance = [&]() {
                while (more && base >= lw.take) {
                    more = lw.next(p, end);
                    base = w * kGroup;
                }
                phys = -1;
                if (more && base + k < lw.take) {
                    phys = __ldg(p.tables + (int64_t)lw.b * p.table_stride + lw.p0 + base + k);
                    if (phys < 0) phys = INT_MAX;  // a bad entry, reported when it is loaded
                }
                head = p.kv_pool + F::offset(0, p.layer, kv_head(p, lw.seg), p.num_layers,
                                             p.num_kv_heads);
            };
            advance();
            int stage = 0, issued = 0;
            uint32_t phase = 1;  // the first round finds every stage free
            uint64_t since = 0;
            for (uint32_t it = 0; __any_sync(0xffffffffu, more); ++it) {
                const bool ready = more && test_wait(&empty[w][stage], phase);
                if (ready) {
                    uint64_t *bar = &full[w][stage];
                    const uint32_t dst = dst0 + stage * C::kStage;
                    if ((uint32_t)phys < p.num_blocks) {
                        mbar_arrive_expect_tx(bar, C::kPage);
                        bulk_load(dst, head + phys * page_stride, C::kPage, bar);
                    } else {
                        if (phys != -1) {  // a table entry outside the pool reads as zeros
                            set_status(p.status, LC_DEV_BAD_BLOCK);
                            for (int i = 0; i < C::kPage / 16; ++i)
                                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst + 16 * i),
                                             "r"(0) : "memory");
                            // before the copies that fill the stage later
                            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        }
                        mbar_arrive(bar);
                    }
                    ++issued;
                    if (++stage == C::kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                    base += kGroup * kWarps;
                    advance();
                }
                if (__any_sync(0xffffffffu, ready)) {
                    since = 0;
                    continue;
                }
                // nothing to do: wait a little, for 2 s at most
                __nanosleep(40);
                if ((it & 63) == 0) {
                    const uint64_t now = global_timer_ns();
                    if (since == 0) since = now;
                    if (now - since > kWaitLimitNs) {
                        s_abort = 1;
                        set_status(p.status, LC_DEV_TIMEOUT);
                    }
                    if (*(volatile int *)&s_abort) break;
                }
            }
            // After a timeout the computing warps may leave stages unread: no copy may land
            // in a CTA that is gone.
            __syncwarp();
            if (*(volatile int *)&s_abort && lane < kGroup * kWarps)
                for (int i = max(0, issued - C::kStages); i < issued; ++i)
                    mbar_wait_drain(&full[w][i % C::kStages], i / C::kStages & 1);
            return;
        }

        // ---- the edge warps
        const int edge = kEdges == 1 ? 0 : warp - kEdgeWarp;
        // rows of sequences without tokens are zeros
        for (int b = cta + edge * gridDim.x; b < p.batch; b += kEdges * gridDim.x) {
            if (tokens_of(p, b, false) > 0) continue;
            const int width = p.num_q_heads * HD;
            for (int i = lane; i < p.tokens * width; i += 32)
                p.out[((int64_t)b * p.tokens + i / width) * p.out_stride + i % width] =
                    __float2bfloat16(0.f);
        }
        if (edge == 0 && lane == 0) s_cut = cut;  // seen with the first chunk's barrier
        Walk<F> cw;
        bool more = first < end;
        if (more) {
            cw.start(p, first, b0, before);
            more = cw.next(p, end);
        }
        if (!more) {
            if (lane == 0) {
                if (edge == 0) s_chunk[0].take = 0;
                mbar_arrive(&q_full[0]);
            }
            return;
        }
        // q: column c of the slice is query token c / group, head c % group. Lane (g, t)
        // holds a quarter of column g's dims, as the products need them. A chunk's rows
        // are read while the chunk before it is prepared and the one before that joined.
        // From L2 and not through the read-only path (__ldg): a launch that starts early is
        // there while the append still writes these rows, and griddep_wait orders ordinary
        // reads alone; L1 may hold neighbours of q from before that, where q lies over qkv.
        uint4 raw[HD / 32];
        auto read_q = [&]() {
            const int kvh = kv_head(p, cw.seg);
            const int col = (cw.seg - kvh * p.slices) * kCols + edge * 8 + g;
            const int i = col / p.group, h = col - i * p.group;
            const bf16 *src = p.q + ((int64_t)cw.b * p.tokens + i) * p.q_stride +
                              (int64_t)(kvh * p.group + h) * HD + F::q_dim(t, 0);
#pragma unroll
            for (int k = 0; k < HD / 32; ++k)
                raw[k] = col < p.cols ? load_l2(src + (F::q_dim(0, k) - F::q_dim(0, 0)))
                                      : make_uint4(0, 0, 0, 0);
        };
        read_q();
        ChunkInfo prev{};
        for (uint32_t chunk = 0; more; ++chunk) {
            // Buffer chunk & 1 is free: chunk - 2 was joined here in the turn before.
            const int buf = chunk & 1;
            ChunkInfo ch{cw.b, cw.seg, cw.p0, cw.take, cw.n, cw.seg_at, 0};
            more = cw.next(p, end);
            ch.last = !more;
            const uint32_t *r = reinterpret_cast<const uint32_t *>(raw);
            uint32_t top = 0;  // largest magnitude, as bf16 bits
#pragma unroll
            for (int k = 0; k < HD / 8; ++k)
                top = max(top, max(r[k] & 0x7fffu, (r[k] >> 16) & 0x7fffu));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^-e and 2^e, kept within the normal numbers
            const int e = max((int)(top >> 7) - 127 - kQTop, -126);
            // A NaN scale goes into q, so that the masked scores, which it must not reach, stay
            // -inf; for their sake the factor is never zero either.
            const float down = p.scale_log2 == p.scale_log2 ? __int_as_float((127 - e) << 23) : NAN;
            if (t == 0)
                s_f[buf][edge * 8 + g] =
                    fmaxf(p.scale_log2 * __int_as_float((127 + e) << 23), FLT_MIN);
            uint2 *dst = reinterpret_cast<uint2 *>(q_ops + buf * C::kQ) + edge * kSteps * 32 + lane;
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) {
                uint32_t v[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t x = r[2 * k + i];
                    const __half2 y = __floats2half2_rn(__uint_as_float(x << 16) * down,
                                                        __uint_as_float(x & 0xffff0000u) * down);
                    v[i] = *reinterpret_cast<const uint32_t *>(&y) ^ p.q_sign;
                }
                dst[k * 32] = make_uint2(v[0], v[1]);
            }
            if (edge == 0 && lane == 0) s_chunk[buf] = ch;
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[buf]);
            if (more) read_q();

            if (chunk > 0) {
                if (!mbar_wait_bounded(&states_full, (chunk - 1) & 1, &s_abort, p.status)) return;
                const bool whole = prev.take == pages_of(prev.n);
                const int64_t seg = (int64_t)prev.b * p.seg_per_seq + prev.seg;
                if constexpr (C::kRegs == 0) {
                    join_columns<F, NT>(p, prev, whole, seg + cta, edge, lane, s_ml, states);
                } else {  // three edge warps of 72 registers: spills would cost more (3 %)
                    for (int c = edge; c < kCols; c += kEdges) {
                        Joined<F, NT> j;
                        join_states<F, NT>(s_ml, states, c, lane, j);
                        if (whole)
                            write_row<F, NT>(p, prev, c, lane, j);
                        else
                            store_piece<F, NT>(p, seg + cta, c, lane, j);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&states_empty);
                if (!whole) {  // the CTA's first chunk, the end of a segment
                    int c0;
                    const int pieces = pieces_of<F>(p, cut, prev, c0);
                    const bool mine = lane < kCols && lane % kEdges == edge &&
                                      last_piece<kCols>(p, c0, pieces, cta - c0, lane, false);
                    const uint32_t cols = __ballot_sync(0xffffffffu, mine);
                    if (lane == 0) {
                        if (edge == 0) s_left = prev;
                        if (cols) atomicOr(&s_left_cols, cols);
                    }
                }
            }
            prev = ch;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&edge_done);
        return;
    }

    // ---- computing warps
    if constexpr (C::kRegs != 0)
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kRegs ? C::kRegs : 24));
    if (p.pdl_mode == 2) griddep_wait();
    const int pi0 = g & 1 ? 7 - (g >> 1) : g >> 1;  // token of tile row g
    const uint8_t *ring = smem + warp * C::kStages * C::kStage;
    int stage = 0;
    uint32_t phase = 0;
    for (uint32_t chunk = 0;; ++chunk) {
        const int buf = chunk & 1;
        if (!mbar_wait_bounded(&q_full[buf], chunk >> 1 & 1, &s_abort, p.status)) return;
        const ChunkInfo &info = s_chunk[buf];
        const int take = info.take, p0 = info.p0, n = info.n;
        if (take == 0) return;
        const uint2 *qs = reinterpret_cast<const uint2 *>(q_ops + buf * C::kQ) + lane;
        float f[NT][2];
        int lim[NT][2];  // tokens that a column sees
        // Tokens that every column sees, and those of the chunk's pages.
        const int col0 = info.seg % p.slices * kCols;
        const int all = n - (p.tokens - 1 - col0 / p.group);
        const int held = min(n, (p0 + take) * kBlockSize);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int c = nt * 8 + 2 * t + k;
                f[nt][k] = s_f[buf][c];
                lim[nt][k] = min(held, n - (p.tokens - 1 - min(col0 + c, p.cols - 1) / p.group));
            }

        float o[kSteps][NT][4];
        float m[NT][2], l[NT][2];
        float off[NT][2];  // m, or 0 while it is -inf
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = off[nt][0] = off[nt][1] = 0.f;
#pragma unroll
            for (int j = 0; j < kSteps; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[j][nt][k] = 0.f;
        }

        // One group. kTail: it reaches past the tokens that every column sees, or past
        // the chunk (a page that was not loaded is masked; its stage holds anything).
        auto group = [&](auto tail_c, int base) {
            constexpr bool kTail = decltype(tail_c)::value;
            const int tok0 = (p0 + base) * kBlockSize;
            // after a timeout the stage holds anything; the status word says so
            mbar_wait_bounded(&full[warp][stage], phase, &s_abort, p.status);
            const uint8_t *st = ring + stage * C::kStage;

            // S^T = K . Q^T
            float s[kGroup][NT][4];
            F::template scores<NT>(st, qs, pi0, t, s);
            if constexpr (kTail) {
#pragma unroll
                for (int pg = 0; pg < kGroup; ++pg)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (tok0 + pg * kBlockSize + pi0 + (k >> 1) * 8 >=
                                lim[nt][k & 1])
                                s[pg][nt][k] = -INFINITY;
            }

            // A page's scales: K's goes into the factor of its scores, V's into the exponent of
            // its probabilities, so that m is the largest of s + log2(V's scale) and O needs
            // no other; l takes V's out again.
            float fk[kGroup][NT][2], lv[kGroup], out_v[kGroup];
            if constexpr (F::kPageScales) {
#pragma unroll
                for (int pg = 0; pg < kGroup; ++pg) {
                    float ks;
                    F::page_scales(st + pg * C::kPage, ks, lv[pg], out_v[pg]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int k = 0; k < 2; ++k)  // not zero, for the masked scores' sake
                            fk[pg][nt][k] = fmaxf(f[nt][k] * ks, FLT_MIN);
                }
            }
            // running maximum less kLift: raised only where some p would pass 2^15
            bool raise = false;
            float top[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if constexpr (F::kPageScales) {
                        top[nt][k] = fmaf(fmaxf(s[0][nt][k], s[0][nt][k + 2]), fk[0][nt][k], lv[0]);
#pragma unroll
                        for (int pg = 1; pg < kGroup; ++pg)
                            top[nt][k] = fmaxf(top[nt][k], fmaf(fmaxf(s[pg][nt][k], s[pg][nt][k + 2]),
                                                                fk[pg][nt][k], lv[pg]));
                    } else {
                        float x = fmaxf(s[0][nt][k], s[0][nt][k + 2]);
#pragma unroll
                        for (int pg = 1; pg < kGroup; ++pg)
                            x = fmaxf(x, fmaxf(s[pg][nt][k], s[pg][nt][k + 2]));
                        top[nt][k] = x * f[nt][k];
                    }
                    raise |= top[nt][k] > m[nt][k] + (kLift + kLazy);
                }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float x = top[nt][k];
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1)
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                        x = fmaxf(x - kLift, m[nt][k]);
                        const float r = m[nt][k] == -INFINITY ? 0.f : ex2(m[nt][k] - x);
                        m[nt][k] = x;
                        off[nt][k] = x == -INFINITY ? 0.f : x;
                        l[nt][k] *= r;
#pragma unroll
                        for (int j = 0; j < kSteps; ++j) {
                            o[j][nt][k] *= r;
                            o[j][nt][k + 2] *= r;
                        }
                    }
            }
            uint32_t pf[kGroup][NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int pg = 0; pg < kGroup; ++pg) {
                    if constexpr (F::kPageScales) {
                        float sum[2] = {0.f, 0.f};
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const float p0 =
                                ex2(fmaf(s[pg][nt][2 * k], fk[pg][nt][0], lv[pg] - off[nt][0]));
                            const float p1 =
                                ex2(fmaf(s[pg][nt][2 * k + 1], fk[pg][nt][1], lv[pg] - off[nt][1]));
                            sum[0] = k == 0 ? p0 : sum[0] + p0;
                            sum[1] = k == 0 ? p1 : sum[1] + p1;
                            const __half2 v = __floats2half2_rn(p0, p1);
                            pf[pg][nt][k] = movmatrix_trans(*reinterpret_cast<const uint32_t *>(&v));
                        }
                        l[nt][0] = fmaf(sum[0], out_v[pg], l[nt][0]);
                        l[nt][1] = fmaf(sum[1], out_v[pg], l[nt][1]);
                    } else {
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const float p0 = ex2(fmaf(s[pg][nt][2 * k], f[nt][0], -off[nt][0]));
                            const float p1 = ex2(fmaf(s[pg][nt][2 * k + 1], f[nt][1], -off[nt][1]));
                            l[nt][0] += p0;
                            l[nt][1] += p1;
                            const __half2 v = __floats2half2_rn(p0, p1);
                            pf[pg][nt][k] = movmatrix_trans(*reinterpret_cast<const uint32_t *>(&v));
                        }
                    }
                }
            }

            // O^T += V^T . P^T
#pragma unroll
            for (int pg = 0; pg < kGroup; ++pg) {
                F::template values<NT, kTail>(st, pg, g, t, pf[pg], o, tok0, held, all, p.tokens, lim);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[warp][stage]);
            if (++stage == C::kStages) {
                stage = 0;
                phase ^= 1;
            }
        };
        int base = warp * kGroup;
        const int plain = (min(all, held) / kBlockSize - p0) - kGroup;  // last base without a tail
        for (; base <= plain; base += kGroup * kWarps) group(std::false_type(), base);
        for (; base < take; base += kGroup * kWarps) group(std::true_type(), base);

        // ---- the chunk's end: leave this warp's state for the join
        if (chunk > 0) mbar_wait_bounded(&states_empty, (chunk - 1) & 1, &s_abort, p.status);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[nt][k] += __shfl_xor_sync(0xffffffffu, l[nt][k], d);
                const int c = nt * 8 + 2 * t + k;
                // Scores that are all NaN leave m at -inf, which says that the warp saw
                // nothing of the column; any other m lets their NaN sums through.
                const float seen = m[nt][k] == -INFINITY && l[nt][k] != 0.f ? 0.f : m[nt][k];
                if (g == 0) s_ml[warp][c] = make_float2(seen, l[nt][k]);
                float *dst = states + (warp * kCols + c) * C::kRow + g * (HD / 8);
#pragma unroll
                for (int j = 0; j < kSteps; j += 2)
                    *reinterpret_cast<float4 *>(dst + 2 * j) = make_float4(
                        o[j][nt][k], o[j][nt][k + 2], o[j + 1][nt][k], o[j + 1][nt][k + 2]);
            }
        const bool last = info.last;
        __syncwarp();
        if (lane == 0) mbar_arrive(&states_full);
        if (!last) continue;
        // Every page of this warp has been read: its ring takes the pieces.
        float *join_buf = reinterpret_cast<float *>(smem + warp * C::kStages * C::kStage);
        static_assert(C::kStages * C::kStage >= 8192 && C::kStages * C::kStage % 16 == 0);
        if (!mbar_wait_bounded(&states_full, chunk & 1, &s_abort, p.status)) return;
        const ChunkInfo ch = s_chunk[buf];
        const Cut cut = s_cut;
        const bool whole = ch.take == pages_of(ch.n);
        const int64_t seg = (int64_t)ch.b * p.seg_per_seq + ch.seg;
        int c0 = 0, pieces = 0;
        if (!whole) pieces = pieces_of<F>(p, cut, ch, c0);
#pragma unroll 1
        for (int c = warp; c < kCols; c += kWarps) {
            Joined<F, NT> j;
            join_states<F, NT>(s_ml, states, c, lane, j);
            if (!whole) {
                store_piece<F, NT>(p, seg + cta, c, lane, j);
                __syncwarp();
                const int mine = lane == 0 && last_piece<kCols>(p, c0, pieces, cta - c0, c, false);
                if (!__shfl_sync(0xffffffffu, mine, 0)) continue;
                __syncwarp();  // lane 0's count saw the pieces; now the other lanes' reads do
                if (!finish_column<F, NT>(p, seg, c0, pieces, cta - c0, c, lane, join_buf, j))
                    continue;
            }
            write_row<F, NT>(p, ch, c, lane, j);
        }
        if (chunk == 0 || !mbar_wait_bounded(&edge_done, 0, &s_abort, p.status)) return;
        const uint32_t left = s_left_cols;
        if (!left) return;
        const ChunkInfo lc = s_left;
        pieces = pieces_of<F>(p, cut, lc, c0);
        __syncwarp();
        __threadfence();  // the edge warp's count saw the pieces; now this warp's reads do
#pragma unroll 1
        for (int c = warp; c < kCols; c += kWarps) {
            if (!(left >> c & 1)) continue;
            Joined<F, NT> j;
            if (finish_column<F, NT>(p, (int64_t)lc.b * p.seg_per_seq + lc.seg, c0, pieces, cta - c0,
                                      c, lane, join_buf, j))
                write_row<F, NT>(p, lc, c, lane, j);
        }
        return;
    }
}

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// Counters of segments, of groups, int32 | m, l [pieces][cols] | o [pieces][cols][hd], with
// pieces = segments + CTAs (a piece's place is its segment + its CTA). The counters, which
// a call leaves zero, take the same room whatever the call's shape, that of the most
// columns; what lies behind them is written before it is read.
struct WsLayout {
    size_t seg, cnt, ml, o;  // cnt: of both, seg: of the segments alone
    size_t total() const { return cnt + ml + o; }
};

// Tiles of 8 columns that a segment takes at once: K and V unpack once for all of
// them, so as few slices as three tiles allow, and then no more tiles than needed.
// (24 columns, 8 sequences of 1024 .. 32768 tokens of 64/8 heads of 128: 66 us with
// three tiles, 100 us as two slices of two.)
int tiles(int64_t cols) {
    if (cols <= 8) return 1;
    return (cols + 23) / 24 < (cols + 15) / 16 ? 3 : 2;
}

WsLayout ws_layout(int64_t batch, int hq, int hkv, int hd, int tokens) {
    const int64_t cols = (int64_t)(hq / hkv) * tokens;
    const int nc = 8 * tiles(cols);
    const int64_t segs = batch * hkv * ((cols + nc - 1) / nc);
    const int64_t pieces = segs + (int64_t)sm_count() * (nc == 8 ? 2 : 1);
    constexpr size_t kCounters = std::max({2 * 8, 16, 24});  // per SM: CTAs * columns
    const size_t seg = align256(sm_count() * kCounters * 4);
    return {seg, 3 * seg, align256(pieces * nc * 8), (size_t)pieces * nc * hd * 4};
}

size_t decode_workspace(int batch, int num_q_heads, int num_kv_heads, int head_dim,
                        int tokens_per_seq) {
    if (batch <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads ||
        tokens_per_seq <= 0 || (head_dim != 64 && head_dim != 128))
        return 0;
    return ws_layout(batch, num_q_heads, num_kv_heads, head_dim, tokens_per_seq).total();
}

template <class F, int NT>
int launch(DecodeParams p, int max_context_len, cudaStream_t stream) {
    using C = Cfg<F, NT>;
    auto kern = decode_stream_kernel<F, NT>;
    const int rc = ensure_smem_attr((const void *)kern, C::kSmem);
    if (rc) return rc;
    if constexpr (C::kRegs != 0) {  // the registers handed over are those of the launch, no more
        static const bool fits = [&] {
            cudaFuncAttributes a = {};
            return cudaFuncGetAttributes(&a, kern) == cudaSuccess &&
                   C::kWarps * C::kRegs + (1 + C::kEdges) * C::kSideRegs <=
                       C::kThreads / 32 * a.numRegs;
        }();
        if (!fits) return LC_ERR_NOT_SUPPORTED;
    }
    p.slices = (p.cols + C::kCols - 1) / C::kCols;
    p.seg_per_seq = p.num_kv_heads * p.slices;
    // the stream's indexes are int32
    if ((int64_t)p.batch * (p.table_stride + F::kEdgeUnits) > INT_MAX / p.seg_per_seq)
        return LC_ERR_UNSUPPORTED_SHAPE;
    int64_t grid = (int64_t)sm_count() * C::kCtasPerSm;
    if (max_context_len > 0) {  // less work than F::kMinPages pages per CTA
        const int64_t pages = ((int64_t)max_context_len + kBlockSize - 1) / kBlockSize;
        grid = std::min<int64_t>(grid, (pages + F::kMinPages - 1) / F::kMinPages *
                                           ((int64_t)p.batch * p.seg_per_seq));
    }
    grid = std::max<int64_t>(grid, 1);
    p.seg_ctas = (int)(grid / p.seg_per_seq);
    p.seg_alone = C::kCtasPerSm > 1 ? std::min(p.seg_ctas, sm_count() / p.seg_per_seq) : 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    p.pdl_mode = dependent_launch_mode();
    cfg.numAttrs = p.pdl_mode > 0 ? 1 : 0;
    if (cudaLaunchKernelEx(&cfg, kern, p) != cudaSuccess) {
        cudaGetLastError();
        return LC_ERR_CUDA;
    }
    return LC_OK;
}

// The checks the entries share; fills all but the pool's factors.
template <template <int> class Format>
int decode_stream(DecodeParams p, void *out, int64_t out_stride, const void *q, int64_t q_stride,
                  const void *kv_pool, int64_t num_blocks, int num_layers, int layer, int num_q_heads,
                  int num_kv_heads, int head_dim, const int *block_tables, int table_stride,
                  const int *context_lens, int len_offset, int batch, int tokens_per_seq,
                  int max_context_len, void *workspace, size_t workspace_bytes, int *dev_status,
                  lc_stream_t stream) {
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
    const WsLayout wl = ws_layout(batch, num_q_heads, num_kv_heads, head_dim, tokens_per_seq);
    if (!workspace || workspace_bytes < wl.total()) return LC_ERR_WORKSPACE_TOO_SMALL;
    if (!aligned16(workspace)) return LC_ERR_MISALIGNED;
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
    p.group = num_q_heads / num_kv_heads;
    p.cols = p.group * tokens_per_seq;
    uint8_t *ws = (uint8_t *)workspace;
    p.ws_cnt = (int *)ws;
    p.ws_group = (int *)(ws + wl.seg);
    p.ws_ml = (float2 *)(ws + wl.cnt);
    p.ws_o = (float *)(ws + wl.cnt + wl.ml);
    p.status = dev_status;
    cudaStream_t s = as_stream(stream);
    switch (tiles(p.cols) * 1000 + head_dim) {
        case 1064: return launch<Format<64>, 1>(p, max_context_len, s);
        case 1128: return launch<Format<128>, 1>(p, max_context_len, s);
        case 2064: return launch<Format<64>, 2>(p, max_context_len, s);
        case 2128: return launch<Format<128>, 2>(p, max_context_len, s);
        case 3064: return launch<Format<64>, 3>(p, max_context_len, s);
        default: return launch<Format<128>, 3>(p, max_context_len, s);
    }
}

}  // namespace
}  // namespace lc
