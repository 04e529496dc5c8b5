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
// The histogram has a bin for each value of a magnitude in [2^-23, 2^10) and one for zero,
// 8449 in all: 34 KB of shared memory, where all 65536 would fill more than an SM has. A row
// with a logit elsewhere (not counting those that are never chosen) takes the slow way,
// window by window of the values.
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
constexpr int kHotLow = 0x3400, kHotHigh = 0x4480, kHot = kHotHigh - kHotLow;  // magnitudes, as bits
constexpr int kBins = 2 * kHot + 1;
constexpr int kOwn = 17;  // bins of a thread
static_assert(kOwn * kSampleThreads >= kBins && kOwn <= 32);
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
// Rank of the histogram's d-th value, the largest first, and the word that counts it.
__device__ __forceinline__ int rank_of_bin(int d) {
    return d < kHot ? d + 0x8000 - kHotHigh : d == kHot ? kZeroRank : d - kHot - 1 + 0x8000 + kHotLow;
}
__device__ __forceinline__ int word_of_bin(int d) {
    return d < kHot ? kHot - 1 - d : d == kHot ? 2 * kHot : d - 1;
}

// Weights of the values of a row.
struct Weights {
    int best;         // rank of the largest
    double top, inv;  // its logit, 1 / temperature
    __device__ __forceinline__ double operator()(int rank) const {
        if (rank == best) return 1.0;
        const double d = value_of(rank) - top;  // -inf below an infinite logit
        return d == -INFINITY ? 0.0 : exp(d * inv);
    }
};

struct Mass {
    int count;
    double weight;
};

struct Shared {
    union {
        unsigned hist[kBins];
        int in_chunk[kMaxChunks];  // tokens of the value sought, once the histogram is done with
    };
    double upto_weight[kSampleThreads];  // inclusive, of the bins of threads 0 .. t
    int upto_count[kSampleThreads];
    uint16_t best_of[kMaxChunks];  // smallest rank of a chunk
    double warp_weight[kSampleWarps];
    int warp_count[kSampleWarps];
    Mass before[kWindows + 1];  // slow way: of all windows before
    int in_window[kWindows], built, number;
    unsigned cold;  // a logit outside the histogram
    int best;
    // the value sought, which of its tokens, whether it has several; rank -1: no token
    int rank, at, several;
    double weight;
    int found[kMaxCluster];  // tokens of that value in each slice
};

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
__device__ __forceinline__ void remote_add(uint32_t at, unsigned v) {
    asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
__device__ __forceinline__ void remote_store(uint32_t at, int v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}

// Running counts and weights of the threads' bins: (c, w) of thread t's, into upto_*.
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
    double before = 0.0;
    for (int i = 0; i < warp; ++i) c += s.warp_count[i], before += s.warp_weight[i];
    s.upto_count[tid] = c;
    s.upto_weight[tid] = before + w;
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
__device__ __noinline__ void choose_slowly(const SampleParams &p, int b, const Row &row, Shared &s) {
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
    const float t = p.temperature ? p.temperature[b] : 1.f;
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
        if (!reached(mine) && reached(from + s.upto_weight[tid])) {
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
            s.number = last;
        }
        __syncthreads();
        const int n = s.number;
        __syncthreads();
        return n;
    };
    const int all = s.before[kWindows].count;
    int keep = all;
    const int k = p.top_k ? p.top_k[b] : 0;
    if (k > 0) keep = min(keep, k);
    const float tp = p.top_p ? p.top_p[b] : 1.f;
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
    const float mp = p.min_p ? p.min_p[b] : 0.f;
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
    const double goal = (double)p.rand_vals[b] * s.weight;
    __syncthreads();
    const int n = by_weight(goal > 0.0 ? goal : 0.0, true);
    by_count(min(n, keep - 1));
}

// ------------------------------------------------------------ the fast way --
// One warp's questions to the histogram.
struct Asker {
    const Shared &s;
    const Weights &weight;
    int lane;

    struct Bins {  // of thread t, bin j in lane j
        int h, c;  // tokens, and those up to it with the threads before
        double each, w;
    };
    __device__ __forceinline__ Bins bins(int t) const {
        Bins x;
        const int d = t * kOwn + lane;
        x.h = lane < kOwn && d < kBins ? (int)s.hist[word_of_bin(d)] : 0;
        x.each = x.h ? weight(rank_of_bin(d)) : 0.0;
        x.c = x.h;
        x.w = x.h * x.each;
#pragma unroll
        for (int k = 1; k < 32; k <<= 1) {
            const int uc = __shfl_up_sync(0xffffffffu, x.c, k);
            const double uw = __shfl_up_sync(0xffffffffu, x.w, k);
            if (lane >= k) x.c += uc, x.w += uw;
        }
        if (t) x.c += s.upto_count[t - 1], x.w += s.upto_weight[t - 1];
        return x;
    }
    // First thread whose running value passes `test`; the last one where none does.
    template <class T>
    __device__ __forceinline__ int first_thread(T test) const {
        constexpr int kEach = kSampleThreads / 32;
        uint32_t m = __ballot_sync(0xffffffffu, test(lane * kEach + kEach - 1));
        if (m == 0) return kSampleThreads - 1;
        const int at = (__ffs(m) - 1) * kEach;
        m = __ballot_sync(0xffffffffu, lane < kEach && test(at + min(lane, kEach - 1)));
        return at + __ffs(m) - 1;
    }
    struct Token {
        int d, at, h;   // its value's bin, which of its tokens, and how many it has
        int number;     // of the order
        double weight;  // up to it
    };
    // Token number n of the order.
    __device__ __forceinline__ Token by_count(int n) const {
        const int t = first_thread([&](int i) { return s.upto_count[i] > n; });
        const Bins x = bins(t);
        const int j = __ffs(__ballot_sync(0xffffffffu, x.c > n)) - 1;
        Token k;
        k.d = t * kOwn + j;
        k.h = __shfl_sync(0xffffffffu, x.h, j);
        k.at = n - (__shfl_sync(0xffffffffu, x.c, j) - k.h);
        k.number = n;
        k.weight = __shfl_sync(0xffffffffu, x.w - (x.h - 1 - k.at) * x.each, j);
        return k;
    }
    // The first token at which the running weight reaches (or, strict, exceeds) x; the last
    // one of the row where none does.
    __device__ __forceinline__ Token by_weight(double x, bool strict) const {
        auto reached = [&](double y) { return strict ? y > x : y >= x; };
        int t = first_thread([&](int i) { return reached(s.upto_weight[i]); });
        while (t > 0 && s.upto_count[t] == s.upto_count[t - 1]) --t;  // none reaches it
        const Bins b = bins(t);
        const uint32_t full = __ballot_sync(0xffffffffu, b.h > 0);
        uint32_t m = __ballot_sync(0xffffffffu, b.h > 0 && reached(b.w));
        const bool some = m != 0;  // not: the thread's sum was another rounding's
        const int j = some ? __ffs(m) - 1 : 31 - __clz(full);
        Token k;
        k.d = t * kOwn + j;
        k.h = __shfl_sync(0xffffffffu, b.h, j);
        const double each = __shfl_sync(0xffffffffu, b.each, j);
        const double from = __shfl_sync(0xffffffffu, b.w, j) - k.h * each;
        const double y = strict ? floor((x - from) / each) : ceil((x - from) / each) - 1;
        k.at = some ? (int)fmin(fmax(y, 0.0), k.h - 1.0) : k.h - 1;
        k.number = __shfl_sync(0xffffffffu, b.c, j) - k.h + k.at;
        k.weight = from + (k.at + 1) * each;
        return k;
    }
    // Tokens with weight >= mp. The weights fall along the order (and are above 1 before it).
    __device__ __forceinline__ int at_least(double mp) const {
        int lo = 0, hi = kBins;  // the first bin below mp lies in lo .. hi
        while (lo < hi) {
            const int each = (hi - lo + 31) / 32, d = lo + lane * each;
            const uint32_t below = __ballot_sync(0xffffffffu, d < hi && !(weight(rank_of_bin(d)) >= mp));
            const int probes = (hi - lo + each - 1) / each;
            const int not_below = below ? __ffs(below) - 1 : probes;
            if (below) hi = lo + not_below * each;
            if (not_below) lo += (not_below - 1) * each + 1;
        }
        return count_before(lo);
    }
    __device__ __forceinline__ int count_before(int d) const {
        const int t = min(d / kOwn, kSampleThreads - 1);
        const int k = t * kOwn + lane;
        const int h = k < d && k < kBins ? (int)s.hist[word_of_bin(k)] : 0;
        return __reduce_add_sync(0xffffffffu, h) + (t ? s.upto_count[t - 1] : 0);
    }
};

// The value chosen and which of its tokens into s.rank, s.at and s.several, from the
// histogram, by the whole CTA.
__device__ __forceinline__ void choose(const SampleParams &p, int b, float t, Shared &s) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int c = 0, first = INT_MAX;
    for (int j = kOwn - 1; j >= 0; --j) {
        const int d = tid * kOwn + j, n = d < kBins ? (int)s.hist[word_of_bin(d)] : 0;
        c += n;
        if (n) first = d;
    }
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) atomicMin(&s.best, first);
    __syncthreads();
    const int best = s.best;
    if (best == INT_MAX) {
        if (tid == 0) s.rank = -1;
        return;
    }
    const Weights weight{rank_of_bin(best), value_of(rank_of_bin(best)), 1.0 / (double)t};
    double w = 0.0;
#pragma unroll 1
    for (int j = 0; j < kOwn; ++j) {
        const int d = tid * kOwn + j;
        const unsigned n = d < kBins ? s.hist[word_of_bin(d)] : 0u;
        if (n) w += n * weight(rank_of_bin(d));
    }
    running(c, w, s);
    if (warp != 0) return;
    const Asker ask{s, weight, lane};
    const int all = s.upto_count[kSampleThreads - 1];
    int keep = all;
    double kept = s.upto_weight[kSampleThreads - 1];
    const int k = p.top_k ? p.top_k[b] : 0;
    const float tp = p.top_p ? p.top_p[b] : 1.f, mp = p.min_p ? p.min_p[b] : 0.f;
    const double u = p.rand_vals[b];
    if (k > 0 && k < keep) {
        keep = k;
        kept = ask.by_count(keep - 1).weight;
    }
    if (tp < 1.f) {
        const int n = tp > 0.f ? ask.by_weight((double)tp * kept, false).number + 1 : 1;
        if (n < keep) {
            keep = n;
            kept = ask.by_count(keep - 1).weight;
        }
    }
    if (mp > 0.f) {
        const int n = max(1, ask.at_least((double)mp));
        if (n < keep) {
            keep = n;
            kept = ask.by_count(keep - 1).weight;
        }
    }
    const double goal = u * kept;
    Asker::Token got = ask.by_weight(goal > 0.0 ? goal : 0.0, true);
    if (got.number >= keep) got = ask.by_count(keep - 1);
    if (lane == 0) {
        s.rank = rank_of_bin(got.d);
        s.at = got.at;
        s.several = got.h > 1;
    }
}

__global__ void __launch_bounds__(kSampleThreads) sample_kernel(SampleParams p, int ctas, int chunk_words) {
    __shared__ Shared s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int b = blockIdx.x / ctas, cta = blockIdx.x % ctas;  // a cluster is a row's CTAs
    const Row row(p.logits + (int64_t)b * p.stride, p.vocab);
    // this CTA's slice, in whole chunks
    const int words = row.words(), chunks_in_all = (words + chunk_words - 1) / chunk_words;
    const int per = (chunks_in_all + ctas - 1) / ctas;
    const int chunk0 = min(chunks_in_all, cta * per), chunks = min(chunks_in_all, chunk0 + per) - chunk0;
    const float t = p.temperature ? __ldg(p.temperature + b) : 1.f;
    const bool greedy = !(t > 0.f);

    for (int i = tid; i < kBins; i += kSampleThreads) s.hist[i] = 0;
    if (tid == 0) s.cold = 0, s.best = INT_MAX;
    __syncthreads();
    if (ctas > 1) cluster_arrive();
    bool cold = false;
    for (int c = warp; c < chunks; c += kSampleWarps) {
        const int w0 = (chunk0 + c) * chunk_words, w1 = min(words, w0 + chunk_words);
        uint32_t least = 0xffffffffu;  // ranks, two at a time
        for (int w = w0 + lane; w < w1; w += 32) {
            const uint4 u = row.word(w);
            const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t neg = (x[e] >> 15 & 0x00010001u) * 0x7fffu;
                least = __vminu2(least, x[e] ^ 0x7fff7fffu ^ neg);
            }
            if (greedy) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t bits = e & 1 ? x[e / 2] >> 16 : x[e / 2] & 0xffffu;
                const uint32_t m = bits & 0x7fffu, i = m - kHotLow;
                if (i < (uint32_t)kHot) {
                    atomicAdd(&s.hist[i + (bits >> 15) * kHot], 1u);
                } else if (m == 0) {
                    atomicAdd(&s.hist[2 * kHot], 1u);
                } else {
                    cold |= eligible(rank_of(bits));
                }
            }
        }
        least = __reduce_min_sync(0xffffffffu, min(least & 0xffffu, least >> 16));
        if (least == 0x8000u) least = kZeroRank;
        if (lane == 0) {
            s.best_of[c] = (uint16_t)least;
            if (greedy) atomicMin(&s.best, (int)least);
        }
    }
    if (__any_sync(0xffffffffu, cold) && lane == 0) s.cold = 1;
    __syncthreads();
    if (ctas > 1) {
        cluster_wait();  // the first CTA's histogram was zero before this
        if (cta != 0) {
            const uint32_t to = in_cta(s.hist, 0);
            if (!greedy)
                for (int i = tid; i < kBins; i += kSampleThreads)
                    if (s.hist[i]) remote_add(to + 4 * i, s.hist[i]);
            if (tid == 0) {
                if (s.cold) remote_add(in_cta(&s.cold, 0), 1);
                if (greedy)
                    asm volatile("red.relaxed.cluster.shared::cluster.min.s32 [%0], %1;" ::"r"(
                                     in_cta(&s.best, 0)), "r"(s.best) : "memory");
            }
        }
        cluster_arrive();
        cluster_wait();
    }
    if (cta == 0) {
        if (s.cold || (greedy && s.best < kFirstRank)) {  // NaN counts as a value that is looked for
            choose_slowly(p, b, row, s);
        } else if (greedy) {
            if (tid == 0) s.rank = s.best <= kLastRank ? s.best : -1, s.at = 0, s.several = 1;
        } else {
            choose(p, b, t, s);
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
    auto matches = [&](int w) {  // bits of the word's tokens that have the value
        const uint4 u = row.word(w);
        const uint32_t x[4] = {u.x, u.y, u.z, u.w};
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) m |= (uint32_t)(rank_of(x[e / 2] >> e % 2 * 16 & 0xffffu) == want) << e;
        return m;
    };
    if (want >= 0) {
        for (int c = warp; c < chunks; c += kSampleWarps) {
            int n = 0;
            if (s.best_of[c] <= want) {
                const int w0 = (chunk0 + c) * chunk_words, w1 = min(words, w0 + chunk_words);
                for (int w = w0 + lane; w < w1; w += 32) {
                    const uint32_t m = matches(w);
                    if (m && !several) p.out[b] = (unsigned)(w * 8 - row.skip + __ffs(m) - 1);
                    n += __popc(m);
                }
                n = __reduce_add_sync(0xffffffffu, n);
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
            const uint32_t in = w + lane < w1 ? matches(w + lane) : 0u;
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
    // CTAs per row: as many as run at once (four to an SM), of 4096 tokens at least
    int ctas = 1;
    while (ctas < kMaxCluster && (int64_t)batch * ctas * 2 <= (int64_t)sm_count() * 4 &&
           vocab >= 4096 * ctas * 2)
        ctas *= 2;
    int64_t chunk_words = 32;  // a warp's load
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
