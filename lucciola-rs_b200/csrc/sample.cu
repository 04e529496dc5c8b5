// sample.cu - the next token of each row from its logits, with temperature, top-k, top-p
// and min-p of its own and a uniform number that the caller draws (lc_sample).
//
// Order the tokens by (larger logit, then lower index) and let, for the logits x above -1e30,
//     w = exp((x - max) / temperature).
// Kept are the first top_k tokens; of these the shortest prefix whose weight reaches top_p of
// theirs; of these the ones with w >= min_p (the largest weight is 1). The choice is the first
// token at which the running weight of the kept ones exceeds rand times their weight.
//
// Weights and sums are in 64 bits. A sum in 32 bits would move every border between two
// tokens by 1e-7 of the whole and more, and with a few thousand tokens in play the draws
// near one would differ from run to run of another split; here they differ by 1e-14.
//
// bf16 logits take 65536 values, and tokens of one value have one weight. So a row is a
// histogram over the values: everything above is a question to the running count and the
// running weight along it, and only the last step, the r-th token of one value, looks at
// tokens again.
//
// The histogram has a bin for each value of a magnitude in [2^-22, 2^10), one for zero and
// one for each of the four ranges beside them, 8197 in all: 33 KB of shared memory, where all
// 65536 would fill more than an SM has. In such a range a row may have one token (a tiny logit
// turns up in one of 100 rows of 151936 normal ones); a row with more in one takes the slow
// way, window by window of the values, in one CTA. So does a row whose mask is finite and above
// -1e30: with a sixteenth of 151936 tokens at -1e4, -65504 or -1e9 one row takes 213 us, 64
// rows 315 to 319 and 256 rows 398, against 14.0, 23.4 and 48.4 us with -inf in their place
// (the type's lowest value is as quick); with two tiny logits in every row 209, 304 to 309, 359.
//
// Bounds. 256 rows of 151936 logits (78 MB, 12 us at a device copy's rate): 47.5 us. Counting
// takes 12 instructions for 32 tokens, and 3.75 cycles of shared memory, since 32 addresses out
// of 8192 fall on 3.5 of a bank: about 5 tokens per cycle and SM, 16 us a row, and 256 rows are
// two rows on most SMs. Then the questions, 5 to 8 us. One row is latency: 13.4 us, of them 2.3
// the launch, 2.6 the reads and counts of its eight CTAs, 2.2 their addition, 1.9 the weights,
// 0.7 each question, 1.5 the choice's way to the others and their look for the token. Rejected:
// 17 bins of two binades per thread walked one by one (14.6 us), one warp that asks for all
// (16.5), clusters of 2 or 4 CTAs (18.5, 15.3; with eight 14.2 then).
//
// One cluster of CTAs per row (one CTA where there are rows enough): each counts a slice,
// the others add their bins to the first one's, that one answers the questions, and all look
// for the token. Of each chunk of a slice the largest logit is kept, so that this last look
// reads the few chunks that can hold it.
#include <climits>
#include <cmath>

#include "lc_common.cuh"
#include "lc_host.h"

namespace lc {
namespace {

constexpr int kSampleThreads = 512, kSampleWarps = kSampleThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kMaxChunks = 1024;  // of a slice
constexpr int kAhead = 4;         // words of 16 bytes that a lane loads at a time
constexpr int kHotLow = 0x3480, kHotHigh = 0x4480, kHot = kHotHigh - kHotLow;  // magnitudes, as bits
static_assert(kHot == 4096);  // see count_token
constexpr int kRanges = 4;  // beyond kHotHigh, below kHotLow, and the same of the negative ones
constexpr int kBins = 2 * kHot + 1 + kRanges;
constexpr int kOwn = 16;  // bins of a thread, in a binade
static_assert(2 * kHot == kOwn * kSampleThreads);
constexpr int kCounters = (kBins + 32 + 3) / 4 * 4;
// Of the slow way: windows of the values, which are numbered by their rank.
constexpr int kWindowBins = 4096, kWindows = 65536 / kWindowBins;
constexpr int kWindowOwn = kWindowBins / kSampleThreads;

struct SampleParams {
    const uint16_t *logits;
    int64_t stride;
    int vocab;
    const float *temperature;
    const int *top_k;
    const float *top_p, *min_p, *rand_vals;
    unsigned *out;
};

// Rank of a value, the largest first: +inf 0x7f .. the smallest above -1e30 0xf149; NaN and
// what is never chosen lie outside. +0 and -0 are one value.
constexpr int kFirstRank = 0x7f, kLastRank = 0xf149, kZeroRank = 0x7fff;
__device__ __forceinline__ int rank_of(uint32_t bits) {
    const int r = (int)(bits & 0x8000u ? bits : bits ^ 0x7fffu);
    return r == 0x8000 ? kZeroRank : r;
}
__device__ __forceinline__ bool eligible(int rank) {
    return rank >= kFirstRank && rank <= kLastRank;
}
__device__ __forceinline__ double value_of(int rank) {
    const uint32_t bits = rank & 0x8000 ? (uint32_t)rank : (uint32_t)rank ^ 0x7fffu;
    return (double)__uint_as_float(bits << 16);
}
// Ranks of the first bins of either sign.
constexpr int kRankPos = 0x8000 - kHotHigh, kRankNeg = 0x8000 + kHotLow;
// After the words of the values come those of the first range, the second, zero, the others.
constexpr int kWordZero = 2 * kHot + 2;
__device__ __forceinline__ int word_of_range(int range) { return 2 * kHot + range + (range >= 2); }

// What a thread has of the histogram: from the largest values on 16 bins each, and before or
// after them, as items 0 and 17 or 18, the bins beside the values of a sign.
constexpr int kItems = kOwn + 3, kHalfThreads = kSampleThreads / 2;
struct Item {
    int word, rank;  // word -1: none
};
__device__ __forceinline__ Item item_of(int t, int i, const int *in_range) {
    if (i >= 1 && i <= kOwn)
        return t < kHalfThreads
                   ? Item{kHot - t * kOwn - i, kRankPos + t * kOwn + i - 1}
                   : Item{kHot + (t - kHalfThreads) * kOwn + i - 1, kRankNeg + (t - kHalfThreads) * kOwn + i - 1};
    if (t == kHalfThreads - 1 && i == kOwn + 2) return Item{kWordZero, kZeroRank};
    const int range = t == 0 && i == 0                         ? 0
                      : t == kHalfThreads - 1 && i == kOwn + 1 ? 1
                      : t == kHalfThreads && i == 0            ? 2
                      : t == kSampleThreads - 1 && i == kOwn + 1 ? 3 : -1;
    return range < 0 ? Item{-1, 0} : Item{word_of_range(range), in_range[range]};
}
// The thread that has the item of a rank.
__device__ __forceinline__ int thread_of(int rank) {
    if (rank <= kZeroRank) return min(max(rank - kRankPos, 0) / kOwn, kHalfThreads - 1);
    return kHalfThreads + min(max(rank - kRankNeg, 0) / kOwn, kHalfThreads - 1);
}
__device__ __forceinline__ int range_of(uint32_t bits) {
    const bool tiny = (bits & 0x7fffu) < (uint32_t)kHotLow;
    return bits & 0x8000u ? (tiny ? 2 : 3) : (tiny ? 1 : 0);
}

// Weights of the values of a row.
struct Weights {
    int best;         // rank of the largest
    double top, inv;  // its logit, 1 / temperature
    __device__ __forceinline__ double exponent(double x) const {
        const double d = x - top;  // -inf below an infinite logit
        return d == -INFINITY ? d : d * inv;
    }
    __device__ __forceinline__ double operator()(int rank) const {
        return rank == best ? 1.0 : exp(exponent(value_of(rank)));
    }
};

// What a row is sampled with. Read before the logits, so that the reads' latency is theirs.
struct RowParams {
    float temperature, top_p, min_p;
    int top_k;
    double rand;
    __device__ __forceinline__ RowParams(const SampleParams &p, int b)
        : temperature(p.temperature ? __ldg(p.temperature + b) : 1.f),
          top_p(p.top_p ? __ldg(p.top_p + b) : 1.f), min_p(p.min_p ? __ldg(p.min_p + b) : 0.f),
          top_k(p.top_k ? __ldg(p.top_k + b) : 0), rand(__ldg(p.rand_vals + b)) {}
};

struct Mass {
    int count;
    double weight;
};

struct Shared {
    union {
        alignas(16) unsigned hist[kCounters];  // the bins, then a word per lane for what has none
        int in_chunk[kMaxChunks];  // tokens of the value sought, once the histogram is done with
    };
    double upto_weight[kSampleThreads];  // inclusive, of the bins of threads 0 .. t
    int upto_count[kSampleThreads];
    uint16_t best_of[kMaxChunks];  // smallest rank of a chunk
    double warp_weight[kSampleWarps];
    int warp_count[kSampleWarps];
    Mass before[kWindows + 1];  // slow way: of all windows before
    int in_window[kWindows], built, number;
    int in_range[kRanges];  // rank of the token in each range
    int best;
    // the value sought, which of its tokens, whether it has several; rank -1: no token
    int rank, at, several;
    double weight;  // up to that token
    int below, at_least;  // first rank below min_p, tokens before it
    double inv;           // 1 / temperature
    struct Answer {
        double weight;  // up to and with the token
        int rank, at, several, number;
    } answers[2];  // in turns
    int found[kMaxCluster];  // tokens of that value in each slice
};

// The larger of two pairs of logits; a NaN is smaller than all others.
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// All ones in the halves of two pairs of logits that are equal (as +0 and -0 are).
__device__ __forceinline__ uint32_t equal_bf16x2(uint32_t a, uint32_t b) {
    return __heq2_mask(*reinterpret_cast<const __nv_bfloat162 *>(&a),
                       *reinterpret_cast<const __nv_bfloat162 *>(&b));
}

// Counts a token; true for one without a bin, but not for logits of -1e30 and below. z: four
// times its bits; `trash`: this lane's word for what has no bin, as bytes; hist: where the
// histogram lies. With y = z - 4 kHotLow a magnitude has a bin if 4 * 4096 and the next two
// bits of y are zero, and its word is that of the magnitude's low 12 bits, of the second half
// where the sign, three bits on, is set. No branch; an atom whose result nobody reads takes
// two instructions less than a red (38.9 million tokens: 23.1 us, 26.0; with a branch 27.2).
__device__ __forceinline__ bool count_token(uint32_t z, uint32_t trash, uint32_t hist) {
    const uint32_t y = z - 4 * kHotLow;
    const bool hot = (y & 0x1c000u) == 0;
    const uint32_t at = hot ? (y & 0x3fffu) | (y >> 3 & ~0x3fffu) : trash;
    asm volatile("{\n\t.reg .b32 old;\n\tatom.shared.add.u32 old, [%0], 1;\n\t}" ::"r"(at + hist)
                 : "memory");
    return !hot && z <= 4 * kLastRank;
}

// A row as 16-byte words from an aligned address on; tokens before and after it are -inf.
struct Row {
    const uint16_t *p;
    int skip, vocab;  // tokens of the first word that are not the row's
    __device__ __forceinline__ Row(const uint16_t *row, int n)
        : p(row - ((uintptr_t)row & 15) / 2), skip((int)((uintptr_t)row & 15) / 2), vocab(n) {}
    __device__ __forceinline__ int words() const { return (int)(((int64_t)skip + vocab + 7) / 8); }
    __device__ __forceinline__ uint4 word(int w) const {
        const int64_t at = (int64_t)w * 8 - skip;  // index of its first token
        if (at >= 0 && at + 8 <= vocab) return __ldg(reinterpret_cast<const uint4 *>(p) + w);
        uint32_t x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t i = at + 2 * e;
            const uint32_t lo = i >= 0 && i < vocab ? __ldg(p + skip + i) : 0xff80u;
            const uint32_t hi = i + 1 >= 0 && i + 1 < vocab ? __ldg(p + skip + i + 1) : 0xff80u;
            x[e] = lo | hi << 16;
        }
        return make_uint4(x[0], x[1], x[2], x[3]);
    }
    __device__ __forceinline__ bool inside(int w0, int w1) const {  // words without such tokens
        return (w0 > 0 || skip == 0) && (int64_t)w1 * 8 - skip <= vocab;
    }
    __device__ __forceinline__ uint4 inner(int w) const {
        return __ldg(reinterpret_cast<const uint4 *>(p) + w);
    }
    // f(bits) for all tokens, by one CTA
    template <class F>
    __device__ __forceinline__ void all(F f) const {
        for (int w = threadIdx.x; w < words(); w += kSampleThreads) {
            const uint4 u = word(w);
            const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) f(x[e / 2] >> e % 2 * 16 & 0xffffu);
        }
    }
};

__device__ __forceinline__ void cluster_arrive() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Address of `p`, of this CTA's shared memory, in that of CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t in_cta(const void *p, int rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ void remote_add(uint32_t at, uint64_t v) {
    asm volatile("red.relaxed.cluster.shared::cluster.add.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory");
}
__device__ __forceinline__ void remote_store(uint32_t at, int v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}

// Running counts and weights of the threads' bins: (c, w) of thread t's, into upto_*. The
// warps' sums are added in their order, so that the weight does not fall from one warp's end
// to the next one's; within a warp it may, by a rounding.
__device__ __forceinline__ void running(int c, double w, Shared &s) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int uc = __shfl_up_sync(0xffffffffu, c, d);
        const double uw = __shfl_up_sync(0xffffffffu, w, d);
        if (lane >= d) c += uc, w += uw;
    }
    if (lane == 31) s.warp_count[warp] = c, s.warp_weight[warp] = w;
    __syncthreads();
    int cs = 0;
    double ws = 0.0;
#pragma unroll
    for (int i = 0; i < kSampleWarps - 1; ++i)
        if (i < warp) cs += s.warp_count[i], ws += s.warp_weight[i];
    s.upto_count[tid] = cs + c;
    s.upto_weight[tid] = ws + w;
    __syncthreads();
}

// ------------------------------------------------------------ the slow way --
// The window's histogram and its running counts and weights.
__device__ __noinline__ void build(const Row &row, int window, const Weights &weight, Shared &s) {
    const int tid = threadIdx.x;
    __syncthreads();
    for (int i = tid; i < kWindowBins; i += kSampleThreads) s.hist[i] = 0;
    __syncthreads();
    row.all([&](uint32_t bits) {
        const int r = rank_of(bits);
        if (eligible(r) && r / kWindowBins == window) atomicAdd(&s.hist[r % kWindowBins], 1u);
    });
    __syncthreads();
    int c = 0;
    double w = 0.0;
    for (int i = 0; i < kWindowOwn; ++i) {
        const int b = tid * kWindowOwn + i, n = (int)s.hist[b];
        if (n == 0) continue;
        c += n;
        w += n * weight(window * kWindowBins + b);
    }
    if (tid == 0) s.built = window;
    running(c, w, s);
}

// The value chosen and which of its tokens into s.rank and s.at, by the whole CTA.
__device__ __noinline__ void choose_slowly(const RowParams &r, const Row &row, Shared &s) {
    const int tid = threadIdx.x;
    __syncthreads();
    if (tid == 0) s.best = INT_MAX, s.built = -1;
    if (tid < kWindows) s.in_window[tid] = 0;
    __syncthreads();
    int best = INT_MAX;
    row.all([&](uint32_t bits) {
        const int r = rank_of(bits);
        if (!eligible(r)) return;
        best = min(best, r);
        atomicAdd(&s.in_window[r / kWindowBins], 1);
    });
    best = __reduce_min_sync(0xffffffffu, best);
    if ((tid & 31) == 0) atomicMin(&s.best, best);
    __syncthreads();
    best = s.best;
    const float t = r.temperature;
    if (best == INT_MAX || !(t > 0.f)) {
        __syncthreads();
        if (tid == 0) s.rank = best == INT_MAX ? -1 : best, s.at = 0, s.several = 1;
        __syncthreads();
        return;
    }
    const Weights weight{best, value_of(best), 1.0 / (double)t};
    for (int w = 0; w < kWindows; ++w) {
        if (s.in_window[w]) build(row, w, weight, s);
        if (tid == 0) {
            if (w == 0) s.before[0] = Mass{0, 0.0};
            s.before[w + 1] = s.before[w];
            if (s.in_window[w]) {
                s.before[w + 1].count += s.upto_count[kSampleThreads - 1];
                s.before[w + 1].weight += s.upto_weight[kSampleThreads - 1];
            }
        }
        __syncthreads();
    }
    // The token number n of the order: its value, which of them, the weight up to it.
    auto by_count = [&](int n) {
        __syncthreads();
        int w = 0;
        while (s.before[w + 1].count <= n) ++w;
        if (s.built != w) build(row, w, weight, s);
        const int from = s.before[w].count;
        const int mine = tid ? s.upto_count[tid - 1] : 0;
        if (n >= from + mine && n < from + s.upto_count[tid]) {
            int c = from + mine;
            double sum = s.before[w].weight + (tid ? s.upto_weight[tid - 1] : 0.0);
            for (int i = 0; i < kWindowOwn; ++i) {
                const int bin = tid * kWindowOwn + i, h = (int)s.hist[bin];
                if (h == 0) continue;
                const double each = weight(w * kWindowBins + bin);
                if (n < c + h) {
                    s.rank = w * kWindowBins + bin;
                    s.at = n - c;
                    s.several = h > 1;
                    s.weight = sum + (n - c + 1) * each;
                    break;
                }
                c += h;
                sum += h * each;
            }
        }
        __syncthreads();
    };
    // The number of the first token at which the running weight reaches (or, strict, exceeds)
    // x > 0 (or, strict, x >= 0); INT_MAX where none does.
    auto by_weight = [&](double x, bool strict) {
        auto reached = [&](double y) { return strict ? y > x : y >= x; };
        int w = 0;
        while (w < kWindows - 1 && !reached(s.before[w + 1].weight)) ++w;
        while (w > 0 && s.before[w + 1].count == s.before[w].count) --w;  // none reaches it
        if (s.built != w) build(row, w, weight, s);
        const double from = s.before[w].weight;
        const double mine = from + (tid ? s.upto_weight[tid - 1] : 0.0);
        if (tid == 0) s.number = INT_MAX;
        __syncthreads();
        // the first of the threads that reach it: the running weight may fall by a rounding
        const int count = s.upto_count[tid] - (tid ? s.upto_count[tid - 1] : 0);
        if (count && reached(from + s.upto_weight[tid])) {
            int c = s.before[w].count + (tid ? s.upto_count[tid - 1] : 0), last = c;
            double sum = mine;
            for (int i = 0; i < kWindowOwn; ++i) {
                const int bin = tid * kWindowOwn + i, h = (int)s.hist[bin];
                if (h == 0) continue;
                const double each = weight(w * kWindowBins + bin);
                last = c + h - 1;
                if (reached(sum + h * each)) {
                    const double k = strict ? floor((x - sum) / each) : ceil((x - sum) / each) - 1;
                    last = c + (int)fmin(fmax(k, 0.0), h - 1.0);
                    break;
                }
                c += h;
                sum += h * each;
            }
            atomicMin(&s.number, last);
        }
        __syncthreads();
        const int n = s.number;
        __syncthreads();
        return n == INT_MAX && reached(s.before[w + 1].weight) ? s.before[w + 1].count - 1 : n;
    };
    const int all = s.before[kWindows].count;
    int keep = all;
    if (r.top_k > 0) keep = min(keep, r.top_k);
    const float tp = r.top_p;
    if (tp <= 0.f) {
        keep = 1;
    } else if (tp < 1.f) {
        double kept = s.before[kWindows].weight;
        if (keep < all) {
            by_count(keep - 1);
            kept = s.weight;
        }
        keep = min(keep, min(by_weight((double)tp * kept, false), INT_MAX - 1) + 1);
    }
    const float mp = r.min_p;
    if (mp > 0.f) {
        // the weights fall along the order: the first value whose weight is below min_p
        int lo = best, hi = kLastRank + 1;
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (weight(mid) >= (double)mp) lo = mid + 1;
            else hi = mid;
        }
        if (tid == 0) s.number = 0;
        __syncthreads();
        int n = 0;
        row.all([&](uint32_t bits) {
            const int r = rank_of(bits);
            n += eligible(r) && r < lo;
        });
        n = __reduce_add_sync(0xffffffffu, n);
        if ((tid & 31) == 0) atomicAdd(&s.number, n);
        __syncthreads();
        keep = min(keep, max(1, s.number));
        __syncthreads();
    }
    by_count(keep - 1);
    const double goal = r.rand * s.weight;
    __syncthreads();
    const int n = by_weight(goal > 0.0 ? goal : 0.0, true);
    by_count(min(n, keep - 1));
}

// ------------------------------------------------------------ the fast way --
// The first rank whose weight is below mp > 0, by one warp: the weights fall along the ranks,
// and it lies where the logarithm says, or beside it.
__device__ __forceinline__ int first_below(const Weights &weight, double mp) {
    const int lane = threadIdx.x & 31;
    if (weight.inv == 0.0) return mp <= 1.0 ? kLastRank + 1 : kFirstRank;
    const float x = (float)fmin(fmax(weight.top + log(mp) / weight.inv, -3e38), 3e38);
    int at = rank_of(__float_as_uint(x) >> 16) - 16;
    for (;;) {
        const int r = at + lane;
        const bool below = r > kLastRank || (r >= kFirstRank && !(weight(r) >= mp));
        const uint32_t m = __ballot_sync(0xffffffffu, below);
        if ((m & 1) && at <= kFirstRank) return kFirstRank;
        if (m & 1) at -= 31;
        else if (m == 0) at += 31;
        else return at + __ffs(m) - 1;
    }
}

// The value chosen and which of its tokens into s.rank, s.at and s.several, from the
// histogram, by the whole CTA. A thread's 16 bins lie in one binade: their values are evenly
// spaced, their weights a geometric sequence, and their sum is a polynomial in its ratio (two
// exponentials, not 16). A question (a number of tokens, or a weight) goes to all threads, and
// the warp of the one in whose bins the answer lies looks at them one by lane. Most rows fill
// a fifth of the bins; warps without tokens skip the sums.
__device__ __forceinline__ void choose(const RowParams &r, Shared &s) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int best = s.best;
    if (best > kLastRank) {
        if (tid == 0) s.rank = -1;
        return;
    }
    const Weights weight{best, value_of(best), s.inv};
    const float tp = r.top_p, mp = r.min_p;
    // One thread's items, one per lane: tokens, weight of each.
    struct Seen {
        int h, rank;
        double each;
    };
    auto look = [&](int t) {
        const Item item = lane < kItems ? item_of(t, lane, s.in_range) : Item{-1, 0};
        Seen x;
        x.rank = item.rank;
        x.h = item.word >= 0 ? (int)s.hist[item.word] : 0;
        x.each = x.h ? weight(item.rank) : 0.0;
        return x;
    };
    int c = 0;
    double w = 0.0;
    const bool pos = tid < kHalfThreads;
    const int word0 = pos ? kHot - (tid + 1) * kOwn : kHot + (tid - kHalfThreads) * kOwn;  // lowest one
    const uint4 *quads = reinterpret_cast<const uint4 *>(s.hist);
    uint32_t any = 0;  // of the warp's 512 bins, read side by side
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint4 q = quads[(word0 - (pos ? 31 - lane : lane) * kOwn) / 4 + i * 32 + lane];
        any |= q.x | q.y | q.z | q.w;
    }
    int extra = 0;  // tokens beside the bins
    if (tid == 0) extra = (int)s.hist[word_of_range(0)];
    if (tid == kHalfThreads - 1) extra = (int)(s.hist[word_of_range(1)] + s.hist[kWordZero]);
    if (tid == kHalfThreads) extra = (int)s.hist[word_of_range(2)];
    if (tid == kSampleThreads - 1) extra = (int)s.hist[word_of_range(3)];
    if (__any_sync(0xffffffffu, any != 0 || extra != 0)) {
        const int mag = kHotLow + (pos ? word0 + kOwn - 1 : word0 - kHot);  // of the largest value
        const double step = __longlong_as_double((int64_t)((mag >> 7) - 134 + 1023) << 52);
        const double by = exp(-step * weight.inv);
        const double first = exp(weight.exponent(value_of(pos ? mag ^ 0x7fff : mag | 0x8000)));
        const double by2 = by * by, by4 = by2 * by2, by8 = by4 * by4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int q = (i + lane / 2) & 3;  // in turns: side by side they hit the same banks
            const uint4 h = quads[word0 / 4 + q];
            // from the largest value on
            const uint32_t a0 = pos ? h.w : h.x, a1 = pos ? h.z : h.y, a2 = pos ? h.y : h.z,
                           a3 = pos ? h.x : h.w;
            c += (int)(a0 + a1 + a2 + a3);
            const double sum = fma(fma(fma((double)a3, by, (double)a2), by, (double)a1), by, (double)a0);
            const int turn = pos ? 3 - q : q;
            w = fma(sum, (turn & 1 ? by4 : 1.0) * (turn & 2 ? by8 : 1.0), w);
        }
        w = c ? w * first : 0.0;
        // A thread with the best value (above it the sequence may overflow) or with tokens beside
        // its bins is looked at.
        const int rank0 = pos ? kRankPos + tid * kOwn : kRankNeg + (tid - kHalfThreads) * kOwn;
        uint32_t odd = __ballot_sync(0xffffffffu, extra || (best >= rank0 && best < rank0 + kOwn));
        while (odd) {
            const int from = __ffs(odd) - 1;
            odd &= odd - 1;
            const Seen x = look(tid - lane + from);
            double sum = x.h * x.each;
#pragma unroll
            for (int k = 16; k; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
            const int count = __reduce_add_sync(0xffffffffu, x.h);
            if (lane == from) c = count, w = sum;
        }
    }
    if (mp > 0.f && warp == kSampleWarps - 1) {  // the smallest logits' warp, which has time
        const int below = first_below(weight, mp);
        if (lane == 0) s.below = below;
    }
    running(c, w, s);
    const int upto_c = s.upto_count[tid], from_c = upto_c - c;
    const double upto_w = s.upto_weight[tid], from_w = tid ? s.upto_weight[tid - 1] : 0.0;
    const int all = s.upto_count[kSampleThreads - 1];
    if (mp > 0.f) {
        const int t = thread_of(s.below);
        if (t / 32 == warp) {
            const Seen x = look(t);
            const int n = __reduce_add_sync(0xffffffffu, x.rank < s.below ? x.h : 0) +
                          __shfl_sync(0xffffffffu, from_c, t % 32);
            if (lane == 0) s.at_least = n;
        }
        __syncthreads();
    }
    // The token number n of the order (by_count), or the first one at which the running weight
    // reaches (strict: exceeds) x, or the last one.
    int turn = 0;
    auto ask = [&](bool by_count, bool strict, int n, double x) -> const Shared::Answer & {
        auto reached = [&](int count, double y) {
            return by_count ? count > n : strict ? y > x : y >= x;
        };
        // an answer stays while the next one is worked out, so one barrier is enough
        Shared::Answer &answer = s.answers[turn ^= 1];
        // the warp at whose end it is reached and before which it was not: there is one
        const uint32_t by_end =
            __ballot_sync(0xffffffffu, upto_c == all || reached(upto_c, upto_w));
        const uint32_t before = __ballot_sync(
            0xffffffffu, from_c > 0 && (from_c == all || reached(from_c, from_w)));
        if (by_end >> 31 && !(before & 1)) {
            const uint32_t some = __ballot_sync(0xffffffffu, c > 0), first = some & by_end;
            const int from = first ? __ffs(first) - 1 : 31 - __clz(some);
            const Seen seen = look(tid - lane + from);
            const int h = seen.h;
            int count = h;
            double sum = h * seen.each;
#pragma unroll
            for (int k = 1; k < 32; k <<= 1) {
                const int uc = __shfl_up_sync(0xffffffffu, count, k);
                const double uw = __shfl_up_sync(0xffffffffu, sum, k);
                if (lane >= k) count += uc, sum += uw;
            }
            count += __shfl_sync(0xffffffffu, from_c, from) - h;  // before this lane's tokens
            sum += __shfl_sync(0xffffffffu, from_w, from) - h * seen.each;
            const uint32_t full = __ballot_sync(0xffffffffu, h > 0);
            const uint32_t m =
                __ballot_sync(0xffffffffu, h > 0 && reached(count + h, sum + h * seen.each));
            // where none reaches it, the thread's sum was another rounding's: the last token
            if (lane == (m ? __ffs(m) - 1 : 31 - __clz(full))) {
                int at = h - 1;
                if (by_count) {
                    at = n - count;
                } else if (m && h > 1) {  // near it in 32 bits, then exactly
                    at = (int)fminf(__fdividef((float)(x - sum), (float)seen.each), (float)(h - 1));
                    at = max(at, 0);
                    while (at > 0 && reached(0, sum + at * seen.each)) --at;
                    while (at < h - 1 && !reached(0, sum + (at + 1) * seen.each)) ++at;
                }
                answer.at = at;
                answer.number = count + at;
                answer.weight = sum + (at + 1) * seen.each;
                answer.several = h > 1;
                answer.rank = seen.rank;
            }
        }
        __syncthreads();
        return answer;
    };
    // top-k, top-p, min-p, the draw, and the last token kept where the draw lies behind it
    int keep = all;
    double kept = s.upto_weight[kSampleThreads - 1];
    const int n_min = mp > 0.f ? max(1, s.at_least) : all;
    if (r.top_k > 0 && r.top_k < keep) {
        keep = r.top_k;
        kept = ask(true, false, keep - 1, 0.0).weight;
    }
    if (tp <= 0.f) {
        keep = 1, kept = 1.0;
    } else if (tp < 1.f) {
        const Shared::Answer &last = ask(false, false, 0, (double)tp * kept);
        if (last.number + 1 < keep) keep = last.number + 1, kept = last.weight;
    }
    if (n_min < keep) {
        keep = n_min;
        kept = ask(true, false, keep - 1, 0.0).weight;
    }
    const Shared::Answer *got = &ask(false, true, 0, fmax(r.rand * kept, 0.0));
    if (got->number >= keep) got = &ask(true, false, keep - 1, 0.0);
    if (tid == 0) s.rank = got->rank, s.at = got->at, s.several = got->several;
}

__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(SampleParams p, int ctas, int chunk_words) {
    __shared__ Shared s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int b = blockIdx.x / ctas, cta = blockIdx.x % ctas;  // a cluster is a row's CTAs
    const Row row(p.logits + (int64_t)b * p.stride, p.vocab);
    // this CTA's slice, in whole chunks
    const int words = row.words(), chunks_in_all = (words + chunk_words - 1) / chunk_words;
    const int per = (chunks_in_all + ctas - 1) / ctas;
    const int chunk0 = min(chunks_in_all, cta * per), chunks = min(chunks_in_all, chunk0 + per) - chunk0;
    const RowParams with(p, b);
    const bool greedy = !(with.temperature > 0.f);

#pragma unroll 1
    for (int i = tid; i < kCounters / 4; i += kSampleThreads)
        reinterpret_cast<uint4 *>(s.hist)[i] = make_uint4(0, 0, 0, 0);
    if (tid < kRanges) s.in_range[tid] = kLastRank;
    if (tid == 0) s.best = INT_MAX, s.inv = 1.0 / (double)with.temperature;
    __syncthreads();
    if (ctas > 1 && cta != 0) cluster_arrive();
    const uint32_t hist = smem_u32(s.hist), trash = (kBins + lane) * 4;
    // one word of a chunk: its largest logits go into `most`, its tokens into the histogram
    auto take = [&](const uint4 &u, uint32_t &most) {
        const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) most = max_bf16x2(most, x[e]);
        if (greedy) return;
        bool other = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            other |= count_token(x[e] << 2 & 0x3fffcu, trash, hist);
            other |= count_token(x[e] >> 14 & 0x3fffcu, trash, hist);
        }
        if (!other) return;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t bits = x[e / 2] >> e % 2 * 16 & 0xffffu;
            if ((bits & 0x7fffu) - kHotLow < (uint32_t)kHot) continue;
            if ((bits & 0x7fffu) == 0) {
                atomicAdd(&s.hist[kWordZero], 1u);
            } else if (eligible(rank_of(bits))) {
                const int range = range_of(bits);
                atomicAdd(&s.hist[word_of_range(range)], 1u);
                s.in_range[range] = rank_of(bits);  // of one token, where one is there
            }
        }
    };
    for (int c = warp; c < chunks; c += kSampleWarps) {
        uint32_t most = 0xff80ff80u;
        const int w0 = (chunk0 + c) * chunk_words, w1 = min(words, w0 + chunk_words);
        if (row.inside(w0, w0 + chunk_words)) {
            for (int w = w0 + lane; w < w1; w += 32 * kAhead) {
                uint4 u[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) u[i] = row.inner(w + 32 * i);
#pragma unroll
                for (int i = 0; i < kAhead; ++i) take(u[i], most);
            }
        } else {
            for (int w = w0 + lane; w < w1; w += 32) take(row.word(w), most);
        }
        const int least =
            __reduce_min_sync(0xffffffffu, min(rank_of(most & 0xffffu), rank_of(most >> 16)));
        if (lane != 0) continue;
        s.best_of[c] = (uint16_t)least;
        atomicMin(&s.best, least);
    }
    __syncthreads();
    if (ctas > 1) {
        // The first CTA has counted before the others add to its bins two at a time: its own
        // 32-bit atomics and these never meet. (One bin at a time, without this order: 64 rows
        // of 151936 22.8 us, 21.9 like this; one row 13.2, 13.4.)
        if (cta == 0) cluster_arrive();
        cluster_wait();
        if (cta != 0) {
            const uint32_t to = in_cta(s.hist, 0);
            if (!greedy) {
#pragma unroll 4
                for (int i = tid; i < (kBins + 1) / 2; i += kSampleThreads) {  // two bins at a time
                    const uint64_t two = reinterpret_cast<const uint64_t *>(s.hist)[i];
                    if (two) remote_add(to + 8 * i, two);
                }
                if (tid < kRanges && s.hist[word_of_range(tid)])
                    remote_store(in_cta(&s.in_range[tid], 0), s.in_range[tid]);
            }
            if (tid == 0)
                asm volatile("red.relaxed.cluster.shared::cluster.min.s32 [%0], %1;" ::"r"(
                                 in_cta(&s.best, 0)), "r"(s.best) : "memory");
        }
        cluster_arrive();
        cluster_wait();
    }
    if (cta == 0) {
        bool slow = false;
        if (!greedy)
            for (int i = 0; i < kRanges; ++i) slow |= s.hist[word_of_range(i)] > 1;
        if (slow) {
            choose_slowly(with, row, s);
        } else if (greedy) {
            if (tid == 0) s.rank = s.best <= kLastRank ? s.best : -1, s.at = 0, s.several = 1;
        } else {
            choose(with, s);
        }
        __syncthreads();
        if (tid < 3 * (ctas - 1)) {
            const int *from = tid % 3 == 0 ? &s.rank : tid % 3 == 1 ? &s.at : &s.several;
            remote_store(in_cta(from, 1 + tid / 3), *from);
        }
    }
    if (ctas > 1) {
        cluster_arrive();
        cluster_wait();
    }
    // ---- the token
    const int want = s.rank, several = s.several;
    int at = s.at;
    if (want < 0) {
        if (cta == 0 && tid == 0) p.out[b] = 0xffffffffu;
    }
    const uint32_t want2 = (uint32_t)(want & 0x8000 ? want : want ^ 0x7fff) * 0x10001u;
    auto matches = [&](const uint4 &u) {  // bits of the word's tokens that have the value
        const uint32_t x[4] = {equal_bf16x2(u.x, want2), equal_bf16x2(u.y, want2),
                               equal_bf16x2(u.z, want2), equal_bf16x2(u.w, want2)};
        uint32_t m = 0;
        if (x[0] | x[1] | x[2] | x[3]) {
#pragma unroll
            for (int e = 0; e < 4; ++e) m |= (x[e] & 1u) << 2 * e | (x[e] >> 31) << (2 * e + 1);
        }
        return m;
    };
    if (want >= 0) {
        for (int c = warp; c < chunks; c += kSampleWarps) {
            int n = 0;
            if (s.best_of[c] <= want) {
                const int w0 = (chunk0 + c) * chunk_words, w1 = min(words, w0 + chunk_words);
                const bool inside = row.inside(w0, w1);
                bool any = false;
                for (int w = w0 + lane; w < w1; w += 32) {
                    const uint32_t m = matches(inside ? row.inner(w) : row.word(w));
                    if (m == 0) continue;
                    if (!several) p.out[b] = (unsigned)(w * 8 - row.skip + __ffs(m) - 1);
                    n += __popc(m);
                    any = true;
                }
                n = __any_sync(0xffffffffu, any) ? __reduce_add_sync(0xffffffffu, n) : 0;
            }
            if (lane == 0) s.in_chunk[c] = n;
        }
    }
    if (want < 0 || !several) return;  // the same in all CTAs of the cluster
    __syncthreads();
    if (warp == 0) {
        int n = 0;
        for (int c = lane; c < chunks; c += 32) n += s.in_chunk[c];
        n = __reduce_add_sync(0xffffffffu, n);
        if (lane < ctas) remote_store(in_cta(&s.found[cta], lane), n);
    }
    if (ctas > 1) {
        cluster_arrive();
        cluster_wait();
    }
    if (warp != 0) return;
    __syncwarp();
    for (int i = 0; i < cta; ++i) at -= s.found[i];
    if (at < 0 || at >= s.found[cta]) return;
    for (int c0 = 0; c0 < chunks; c0 += 32) {  // the chunk that holds it
        const int n = c0 + lane < chunks ? s.in_chunk[c0 + lane] : 0;
        int upto = n;
#pragma unroll
        for (int k = 1; k < 32; k <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, upto, k);
            if (lane >= k) upto += u;
        }
        const uint32_t m = __ballot_sync(0xffffffffu, upto > at);
        if (m == 0) {
            at -= __shfl_sync(0xffffffffu, upto, 31);
            continue;
        }
        const int j = __ffs(m) - 1;
        at -= __shfl_sync(0xffffffffu, upto - n, j);
        const int w0 = (chunk0 + c0 + j) * chunk_words, w1 = min(words, w0 + chunk_words);
        for (int w = w0; w < w1; w += 32) {
            const uint32_t in = w + lane < w1 ? matches(row.word(w + lane)) : 0u;
            int sum = __popc(in);
#pragma unroll
            for (int k = 1; k < 32; k <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, sum, k);
                if (lane >= k) sum += u;
            }
            const int left = at - (sum - __popc(in));  // which of this lane's
            if (left >= 0 && left < __popc(in)) {
                uint32_t rest = in;
                for (int i = 0; i < left; ++i) rest &= rest - 1;
                p.out[b] = (unsigned)((w + lane) * 8 - row.skip + __ffs(rest) - 1);
            }
            at -= __shfl_sync(0xffffffffu, sum, 31);
            if (at < 0) return;
        }
        return;
    }
}

}  // namespace
}  // namespace lc

using namespace lc;

extern "C" int lc_sample(const void *logits, int64_t row_stride, int vocab, int batch,
                         const float *temperature, const int *top_k, const float *top_p,
                         const float *min_p, const float *rand_vals, unsigned *out_idx,
                         lc_stream_t stream) {
    if (!logits || !rand_vals || !out_idx || vocab <= 0 || batch < 0 || row_stride < vocab)
        return LC_ERR_INVALID_ARGUMENT;
    if ((uintptr_t)logits & 1) return LC_ERR_MISALIGNED;
    if (vocab > INT_MAX - 16 || batch > INT_MAX / kMaxCluster) return LC_ERR_INVALID_ARGUMENT;
    if (batch == 0) return LC_OK;
    SampleParams p{(const uint16_t *)logits, row_stride, vocab, temperature, top_k, top_p, min_p,
                   rand_vals, out_idx};
    // CTAs per row: as many as run at once (two to an SM), of 4096 tokens at least
    int ctas = 1;
    while (ctas < kMaxCluster && (int64_t)batch * ctas * 2 <= (int64_t)sm_count() * 2 &&
           vocab >= 4096 * ctas * 2)
        ctas *= 2;
    int64_t chunk_words = 32 * kAhead;  // what a warp loads at a time
    const int64_t words = ((int64_t)vocab + 7 + 7) / 8;
    while ((words + chunk_words - 1) / chunk_words > (int64_t)kMaxChunks * ctas) chunk_words *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(batch * ctas));
    cfg.blockDim = dim3(kSampleThreads);
    cfg.stream = as_stream(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, sample_kernel, p, ctas, (int)chunk_words) != cudaSuccess) {
        cudaGetLastError();
        return LC_ERR_CUDA;
    }
    return LC_OK;
}
