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
// near one would differ from run to run of another split; here they differ by 1e-16.
//
// bf16 logits take 65536 values, and tokens of one value have one weight. So a row is a
// histogram over the values: everything above is a question to the running count and the
// running weight along it, and only the last step, the r-th token of one value, looks at
// tokens again.
#include <climits>
#include <cmath>

#include "lc_common.cuh"
#include "lc_host.h"

namespace lc {
namespace {

constexpr int kSampleThreads = 1024;
constexpr int kWindowBins = 4096, kWindows = 65536 / kWindowBins;
constexpr int kOwn = kWindowBins / kSampleThreads;  // bins of one thread
constexpr float kLeast = -1e30f;                    // a logit must exceed it to be chosen

struct SampleParams {
    const uint16_t *logits;
    int64_t stride;
    int vocab;
    const float *temperature;
    const int *top_k;
    const float *top_p, *min_p, *rand_vals;
    unsigned *out;
};

// Rank of a logit among the values, the largest first; -1: never chosen (NaN, not above
// -1e30). +0 and -0 are one value.
__device__ __forceinline__ int rank_of(uint32_t bits) {
    const float x = __uint_as_float(bits << 16);
    if (!(x > kLeast)) return -1;
    if (bits == 0x8000u) bits = 0;
    return bits & 0x8000u ? (int)bits : 0x7fff - (int)bits;
}
__device__ __forceinline__ double value_of(int rank) {
    const uint32_t bits = rank & 0x8000 ? (uint32_t)rank : 0x7fffu - (uint32_t)rank;
    return (double)__uint_as_float(bits << 16);
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

// f(index, bits) for the tokens [lo, hi) of a row, by the threads tid of n.
template <class F>
__device__ __forceinline__ void for_tokens(const uint16_t *row, int lo, int hi, int tid, int n, F f) {
    const int head = min(hi, lo + (int)((16 - ((uintptr_t)(row + lo) & 15)) % 16 / 2));
    const int words = (hi - head) / 8;
    for (int i = lo + tid; i < head; i += n) f(i, (uint32_t)__ldg(row + i));
    for (int w = tid; w < words; w += n) {
        const uint4 u = __ldg(reinterpret_cast<const uint4 *>(row + head) + w);
        const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) f(head + 8 * w + e, x[e / 2] >> e % 2 * 16 & 0xffffu);
    }
    for (int i = head + 8 * words + tid; i < hi; i += n) f(i, (uint32_t)__ldg(row + i));
}

struct Mass {
    int count;
    double weight;
};

struct Shared {
    int hist[kWindowBins];
    int in_window[kWindows];
    Mass before[kWindows + 1];       // of all windows before
    int warp_count[32];
    double warp_weight[32];
    int upto_count[kSampleThreads];  // inclusive, of the window's bins of threads 0 .. t
    double upto_weight[kSampleThreads];
    int built;                       // window in hist
    int best;
    int kept_least;
    // answers
    int rank, at;  // value and which of its tokens
    double weight;
};

// The window's histogram and its running counts and weights.
__device__ void build(const uint16_t *row, int vocab, int window, const Weights &weight, Shared &s) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    __syncthreads();
    for (int i = tid; i < kWindowBins; i += kSampleThreads) s.hist[i] = 0;
    __syncthreads();
    for_tokens(row, 0, vocab, tid, kSampleThreads, [&](int, uint32_t bits) {
        const int r = rank_of(bits);
        if (r >= 0 && r / kWindowBins == window) atomicAdd(&s.hist[r % kWindowBins], 1);
    });
    __syncthreads();
    int c = 0;
    double w = 0.0;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
        const int b = tid * kOwn + i, n = s.hist[b];
        if (n == 0) continue;
        c += n;
        w += n * weight(window * kWindowBins + b);
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int uc = __shfl_up_sync(0xffffffffu, c, d);
        const double uw = __shfl_up_sync(0xffffffffu, w, d);
        if (lane >= d) c += uc, w += uw;
    }
    if (lane == 31) s.warp_count[warp] = c, s.warp_weight[warp] = w;
    __syncthreads();
    for (int i = 0; i < warp; ++i) c += s.warp_count[i];
    double before = 0.0;
    for (int i = 0; i < warp; ++i) before += s.warp_weight[i];
    s.upto_count[tid] = c;
    s.upto_weight[tid] = before + w;
    if (tid == 0) s.built = window;
    __syncthreads();
}

__global__ void __launch_bounds__(kSampleThreads) sample_kernel(SampleParams p) {
    __shared__ Shared s;
    const int tid = threadIdx.x;
    const uint16_t *row = p.logits + (int64_t)blockIdx.x * p.stride;
    const float t = p.temperature ? p.temperature[blockIdx.x] : 1.f;
    if (tid == 0) s.best = INT_MAX, s.kept_least = 0, s.built = -1;
    if (tid < kWindows) s.in_window[tid] = 0;
    __syncthreads();
    int best = INT_MAX;
    for_tokens(row, 0, p.vocab, tid, kSampleThreads, [&](int, uint32_t bits) {
        const int r = rank_of(bits);
        if (r < 0) return;
        best = min(best, r);
        atomicAdd(&s.in_window[r / kWindowBins], 1);
    });
    best = __reduce_min_sync(0xffffffffu, best);
    if ((tid & 31) == 0) atomicMin(&s.best, best);
    __syncthreads();
    best = s.best;
    if (best == INT_MAX) {
        if (tid == 0) p.out[blockIdx.x] = 0xffffffffu;
        return;
    }
    int want_rank = best, want_at = 0;
    if (t > 0.f) {
        const Weights weight{best, value_of(best), 1.0 / (double)t};
        for (int w = 0; w < kWindows; ++w) {
            if (s.in_window[w]) build(row, p.vocab, w, weight, s);
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
            if (s.built != w) build(row, p.vocab, w, weight, s);
            const int from = s.before[w].count;
            const int mine = tid ? s.upto_count[tid - 1] : 0;
            if (n >= from + mine && n < from + s.upto_count[tid]) {
                int c = from + mine;
                double sum = s.before[w].weight + (tid ? s.upto_weight[tid - 1] : 0.0);
                for (int i = 0; i < kOwn; ++i) {
                    const int b = tid * kOwn + i, h = s.hist[b];
                    if (h == 0) continue;
                    const double each = weight(w * kWindowBins + b);
                    if (n < c + h) {
                        s.rank = w * kWindowBins + b;
                        s.at = n - c;
                        s.weight = sum + (n - c + 1) * each;
                        break;
                    }
                    c += h;
                    sum += h * each;
                }
            }
            __syncthreads();
        };
        // The first token at which the running weight reaches (or, strict, exceeds) x: its
        // number, with s.rank and s.at.
        auto by_weight = [&](double x, bool strict) {
            auto reached = [&](double y) { return strict ? y > x : y >= x; };
            int w = 0;
            while (w < kWindows - 1 && !reached(s.before[w + 1].weight)) ++w;
            while (w > 0 && s.before[w + 1].count == s.before[w].count) --w;  // none reaches it
            if (s.built != w) build(row, p.vocab, w, weight, s);
            const double from = s.before[w].weight;
            const double mine = from + (tid ? s.upto_weight[tid - 1] : 0.0);
            if (tid == 0) s.kept_least = INT_MAX;
            __syncthreads();
            if (!reached(mine) && reached(from + s.upto_weight[tid])) {
                int c = s.before[w].count + (tid ? s.upto_count[tid - 1] : 0);
                double sum = mine;
                for (int i = 0; i < kOwn; ++i) {
                    const int b = tid * kOwn + i, h = s.hist[b];
                    if (h == 0) continue;
                    const double each = weight(w * kWindowBins + b);
                    const double need = (x - sum) / each;
                    if (need < h) {
                        int k = (int)need;  // tokens before
                        if (!strict && (double)k == need && k > 0) --k;
                        atomicMin(&s.kept_least, c + min(max(k, 0), h - 1));
                        break;
                    }
                    c += h;
                    sum += h * each;
                    if (!strict && need == h) {
                        atomicMin(&s.kept_least, c - 1);
                        break;
                    }
                }
            }
            __syncthreads();
            const int n = s.kept_least;
            __syncthreads();
            return n;
        };
        const int eligible = s.before[kWindows].count;
        int keep = eligible;
        const int k = p.top_k ? p.top_k[blockIdx.x] : 0;
        if (k > 0) keep = min(keep, k);
        const float tp = p.top_p ? p.top_p[blockIdx.x] : 1.f;
        double kept = s.before[kWindows].weight;
        if (keep < eligible) {
            by_count(keep - 1);
            kept = s.weight;
        }
        if (tp <= 0.f)
            keep = 1;
        else if (tp < 1.f)
            keep = min(keep, min(by_weight((double)tp * kept, false), INT_MAX - 1) + 1);
        const float mp = p.min_p ? p.min_p[blockIdx.x] : 0.f;
        if (mp > 0.f) {
            // the weights fall along the order: the number of tokens at or above min_p
            int lo = best, hi = 0x10000;  // the first value whose weight is below it
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (weight(mid) >= (double)mp) lo = mid + 1;
                else hi = mid;
            }
            if (tid == 0) s.kept_least = 0;
            __syncthreads();
            int n = 0;
            for_tokens(row, 0, p.vocab, tid, kSampleThreads, [&](int, uint32_t bits) {
                const int r = rank_of(bits);
                n += r >= 0 && r < lo;
            });
            n = __reduce_add_sync(0xffffffffu, n);
            if ((tid & 31) == 0) atomicAdd(&s.kept_least, n);
            __syncthreads();
            keep = min(keep, max(1, s.kept_least));
            __syncthreads();
        }
        by_count(keep - 1);
        const double goal = (double)p.rand_vals[blockIdx.x] * s.weight;
        __syncthreads();
        const int n = min(by_weight(goal > 0.0 ? goal : 0.0, true), keep - 1);
        by_count(n);
        want_rank = s.rank;
        want_at = s.at;
    }
    // token number want_at of the value, by index: counted by 32 pieces of the row, then found
    const int lane = tid & 31, warp = tid >> 5;
    const int per = (p.vocab + 31) / 32;
    const int lo = min(p.vocab, warp * per), hi = min(p.vocab, lo + per);
    int n = 0;
    for (int i = lo + lane; i < hi; i += 32) n += rank_of(__ldg(row + i)) == want_rank;
    n = __reduce_add_sync(0xffffffffu, n);
    __syncthreads();
    if (lane == 0) s.warp_count[warp] = n;
    __syncthreads();
    int before = 0;
    for (int i = 0; i < warp; ++i) before += s.warp_count[i];
    if (want_at < before || want_at >= before + n) return;
    for (int i = lo; i < hi; i += 32) {
        const bool is = i + lane < hi && rank_of(__ldg(row + i + lane)) == want_rank;
        const uint32_t which = __ballot_sync(0xffffffffu, is);
        const int left = want_at - before;
        if (left < __popc(which)) {
            if (is && __popc(which & ((1u << lane) - 1)) == left) p.out[blockIdx.x] = (unsigned)(i + lane);
            return;
        }
        before += __popc(which);
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
    if (batch == 0) return LC_OK;
    SampleParams p{(const uint16_t *)logits, row_stride, vocab, temperature, top_k, top_p, min_p,
                   rand_vals, out_idx};
    sample_kernel<<<batch, kSampleThreads, 0, as_stream(stream)>>>(p);
    return launch_status();
}
