// step_tables.cu - the page bookkeeping of a serving step on the GPU: pages from
// a device free list, block-table rows, positions and the slot map, all from the
// requests' lengths (lc_step_tables), and the way back (lc_step_release).
//
// For request b with c cached and m new tokens, have = ceil(c / 16), want =
// ceil((c + m) / 16), need = want - have. With S(b) the sum of the needs of the
// requests up to and including b, b is served if need = 0 or S(b) <= free_count;
// its page j >= have is then free_pages[free_count - 1 - (S(b) - want + j)].
// This is the order in which lc_block_alloc_reserve, called for b = 0, 1, ...,
// pops its LIFO list.
//
// Every CTA scans the lengths itself (a few KB from L2) instead of waiting for
// another one, so the call is one launch without a device-wide barrier. The
// outputs that a caller may let alias inputs (free_count, the context lengths)
// are written by whichever CTA is last to have read them: each takes a ticket
// after its scan and looks at it at its end, when the answer has long come. Small
// steps are launch latency and three dependent reads (64 requests: 5.1 us); a wide
// step is bound by the rounds of warp tasks that follow the scan, which move table
// rows, positions and slots 16 bytes a lane (1024 requests, rows of 2048 entries,
// 14.5 MB: 14.2 us; 14.7 with one 16-byte read per lane in flight, 16.0 with four; one
// CTA per SM 14.8, three 14.5).
#include <algorithm>

#include "lc_common.cuh"
#include "lc_host.h"

namespace lc {
namespace {

constexpr int kStepThreads = 512;
constexpr int kStepWarps = kStepThreads / 32;
constexpr int kStepMaxBatch = 8192;  // four ints of shared memory per request
// Dynamic shared memory that a launch gets without asking: 48 KB less room for the
// kernels' static arrays (under 200 bytes), which count against the same limit.
constexpr int kSmemUnasked = 47 * 1024;
constexpr int kTokenSegment = 128;   // token rows of a warp's task
constexpr int kRowTurns = 2;         // 16-byte reads per lane in flight
constexpr int kRowSegment = 128 * kRowTurns;  // table entries of a warp's task

struct StepParams {
    int *tables;
    int table_stride, num_slots;
    const int *slots;
    const int *ctx, *add;
    int batch;
    const int *free_pages, *free_count;
    int num_blocks;
    int *step_tables;
    int step_stride;
    int table_vec, step_vec;  // rows start 16-byte aligned
    int *positions, *slot_map;
    int max_tokens, tokens_vec;
    int *row_starts, *ctx_out, *count_out;
    int *ticket, *status;
};

struct ReleaseParams {
    int *free_pages;
    const int *free_count;
    int num_blocks;
    const int *tables;
    int table_stride, num_slots;
    const int *slots, *ctx;
    int count;
    int *count_out, *ticket, *status;
};

__device__ __forceinline__ int pages_of(int tokens) {
    return tokens / kBlockSize + (tokens % kBlockSize != 0);
}

// Exclusive sums over the block of (x, y), one pair per thread; totals in *tx, *ty.
__device__ __forceinline__ void block_scan2(int &x, int &y, int *tx, int *ty) {
    __shared__ int wx[kStepWarps], wy[kStepWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int ix = x, iy = y;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int ux = __shfl_up_sync(0xffffffffu, ix, d), uy = __shfl_up_sync(0xffffffffu, iy, d);
        if (lane >= d) ix += ux, iy += uy;
    }
    if (lane == 31) wx[warp] = ix, wy[warp] = iy;
    __syncthreads();
    int bx = 0, by = 0, sx = 0, sy = 0;
#pragma unroll
    for (int w = 0; w < kStepWarps; ++w) {
        if (w == warp) bx = sx, by = sy;
        sx += wx[w], sy += wy[w];
    }
    x = bx + ix - x;
    y = by + iy - y;
    *tx = sx;
    *ty = sy;
}

// One thread, after the CTA's reads of what the last CTA will overwrite (and a
// barrier): true in the CTA that comes last. It leaves the ticket at zero.
__device__ __forceinline__ bool take_ticket(int *ticket) {
    if (gridDim.x == 1) return true;
    const bool last = atom_add_acq_rel_gpu(ticket, 1) == (int)gridDim.x - 1;
    if (last) *ticket = 0;
    return last;
}

__device__ __forceinline__ int slot_of(const int *slots, int i) {
    return slots ? __ldg(slots + i) : i;
}

// Positions and slots of the four token rows from r0 on.
__device__ __forceinline__ void token_rows(const StepParams &p, const int *start, const int *before,
                                           const int *cached, const int *slots, int count, int tokens,
                                           int r0) {
    if (r0 >= p.max_tokens) return;
    int b = 0;
    if (r0 < tokens) {  // the request of row r0: start[b] <= r0 < start[b + 1]
        int hi = p.batch;
        while (hi - b > 1) {
            const int mid = (b + hi) >> 1;
            if (start[mid] <= r0) b = mid; else hi = mid;
        }
    }
    int pos[4], page[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = r0 + i;
        pos[i] = page[i] = -1;
        if (r >= tokens) continue;
        while (start[b + 1] <= r) ++b;
        const int c = cached[b];
        pos[i] = (c < 0 ? -1 - c : c) + r - start[b];
        if (c < 0) continue;
        const int j = pos[i] / kBlockSize, have = pages_of(c);
        const int *at = j < have ? p.tables + (int64_t)slots[b] * p.table_stride + j
                                 : p.free_pages + (count - 1 - before[b] + have - j);
        page[i] = *at;
        if (page[i] < 0 || page[i] >= p.num_blocks) page[i] = -2;  // not a page
    }
    int slot[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (page[i] == -2) set_status(p.status, LC_DEV_BAD_BLOCK);
        slot[i] = page[i] < 0 ? -1 : page[i] * kBlockSize + pos[i] % kBlockSize;
    }
    if (p.tokens_vec && r0 + 4 <= p.max_tokens) {
        *reinterpret_cast<int4 *>(p.positions + r0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
        *reinterpret_cast<int4 *>(p.slot_map + r0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (r0 + i < p.max_tokens) {
                p.positions[r0 + i] = pos[i];
                p.slot_map[r0 + i] = slot[i];
            }
    }
}

__global__ void __launch_bounds__(kStepThreads) step_tables_kernel(StepParams p) {
    extern __shared__ int sm[];
    int *start = sm;                  // [batch + 1] first token row of a request
    int *before = start + p.batch + 1;  // [batch] pages that earlier requests need
    int *cached = before + p.batch;   // [batch] cached tokens, -1 - them if refused
    int *slots = cached + p.batch;    // [batch] slot, -1 if invalid
    const int tid = threadIdx.x, lane = tid & 31;
    const bool first_cta = blockIdx.x == 0;

    int count = *p.free_count;
    if (count < 0 || count > p.num_blocks) {
        if (first_cta && tid == 0) set_status(p.status, LC_DEV_BAD_BLOCK);
        count = max(0, min(count, p.num_blocks));
    }
    const int per = (p.batch + kStepThreads - 1) / kStepThreads;
    const int b0 = tid * per, b1 = min(p.batch, b0 + per);
    const int cap = p.table_stride * kBlockSize;
    int tok = 0, need = 0;
    for (int b = b0; b < b1; ++b) {
        int c = p.ctx[b], m = p.add[b];
        const int slot = slot_of(p.slots, b);
        if (c < 0 || m < 0 || c > cap || m > cap - c || slot < 0 || slot >= p.num_slots) {
            if (first_cta) set_status(p.status, LC_DEV_BAD_POS);
            if (c < 0 || c > cap || slot < 0 || slot >= p.num_slots) c = 0;
            m = 0;  // an invalid request has no rows
        }
        cached[b] = c;
        slots[b] = slot >= 0 && slot < p.num_slots ? slot : -1;
        start[b] = m;  // its length, until the scan is known
        tok += m;
        need += pages_of(c + m) - pages_of(c);
    }
    __shared__ int most;  // pages taken: the sum up to the last served request that needs one
    if (tid == 0) most = 0;
    int tokens, needed;
    block_scan2(tok, need, &tokens, &needed);
    int taken = 0;
    for (int b = b0; b < b1; ++b) {
        const int c = cached[b], m = start[b], k = pages_of(c + m) - pages_of(c);
        start[b] = tok;
        before[b] = need;
        tok += m;
        need += k;
        if (k > 0) {
            if (need > count) cached[b] = -1 - c;
            else taken = need;
        }
    }
    if (tid == 0) start[p.batch] = tokens;
    if (taken) atomicMax(&most, taken);
    if (first_cta && tid == 0) {
        if (needed > count) set_status(p.status, LC_DEV_OUT_OF_BLOCKS);
        if (tokens > p.max_tokens) set_status(p.status, LC_DEV_BAD_POS);
    }
    __syncthreads();
    bool last = false;
    if (tid == 0) last = take_ticket(p.ticket);

    // Tasks of one warp: kRowSegment entries of a table row, then kTokenSegment token
    // rows, so that in a small step the two kinds run side by side.
    const int warps = gridDim.x * kStepWarps, warp = blockIdx.x * kStepWarps + (tid >> 5);
    const int width = p.step_tables ? max(p.step_stride, p.table_stride) : p.table_stride;
    const int segs = (width + kRowSegment - 1) / kRowSegment, row_tasks = p.batch * segs;
    const int tasks = row_tasks + (p.max_tokens + kTokenSegment - 1) / kTokenSegment;
    for (int t = warp; t < tasks; t += warps) {
        if (t >= row_tasks) {
            token_rows(p, start, before, cached, slots, count, tokens,
                       (t - row_tasks) * kTokenSegment + 4 * lane);
            continue;
        }
        const int b = t / segs, j0 = (t - b * segs) * kRowSegment;
        const int j1 = min(width, j0 + kRowSegment), s1 = min(p.step_stride, j1);
        const int c = cached[b];
        const int n = c < 0 ? -1 - c : c, m = start[b + 1] - start[b];
        const int have = pages_of(n), want = c < 0 ? have : pages_of(n + m);
        const int slot = slots[b];
        if (slot < 0) {
            if (p.step_tables)
                for (int j = j0 + lane; j < s1; j += 32)
                    p.step_tables[(int64_t)b * p.step_stride + j] = -1;
            continue;
        }
        int *row = p.tables + (int64_t)slot * p.table_stride;
        const int *top = p.free_pages + (count - 1 - before[b] + have);  // page j: top[-j]
        for (int j = max(have, j0) + lane; j < min(want, j1); j += 32) {
            const int page = __ldg(top - j);
            if (page < 0 || page >= p.num_blocks) set_status(p.status, LC_DEV_BAD_BLOCK);
            row[j] = page;
        }
        if (!p.step_tables) continue;
        if (want > p.step_stride && j0 == 0 && lane == 0) set_status(p.status, LC_DEV_BAD_POS);
        int *out = p.step_tables + (int64_t)b * p.step_stride;
        auto entry = [&](int j) {
            return j < min(have, p.table_stride) ? row[j] : j < want ? __ldg(top - j) : -1;
        };
        int4 v[kRowTurns];
#pragma unroll
        for (int i = 0; i < kRowTurns; ++i) {
            const int j = j0 + 128 * i + 4 * lane;
            if (p.table_vec && j + 4 <= have)
                v[i] = *reinterpret_cast<const int4 *>(row + j);
            else if (j < want)
                v[i] = make_int4(entry(j), entry(j + 1), entry(j + 2), entry(j + 3));
            else
                v[i] = make_int4(-1, -1, -1, -1);
        }
#pragma unroll
        for (int i = 0; i < kRowTurns; ++i) {
            const int j = j0 + 128 * i + 4 * lane;
            if (j >= s1) break;
            if (p.step_vec && j + 4 <= s1) {
                *reinterpret_cast<int4 *>(out + j) = v[i];
            } else {
                out[j] = v[i].x;
                if (j + 1 < s1) out[j + 1] = v[i].y;
                if (j + 2 < s1) out[j + 2] = v[i].z;
                if (j + 3 < s1) out[j + 3] = v[i].w;
            }
        }
    }

    if (__syncthreads_or(last)) {
        for (int b = tid; b < p.batch; b += kStepThreads) {
            const int c = cached[b], m = start[b + 1] - start[b];
            p.ctx_out[b] = c < 0 ? -1 - c : c + m;
            p.row_starts[b] = start[b];
        }
        if (tid == 0) {
            p.row_starts[p.batch] = tokens;
            *p.count_out = count - most;
        }
    }
}

__global__ void __launch_bounds__(kStepThreads) step_release_kernel(ReleaseParams p) {
    extern __shared__ int sm[];
    int *before = sm;             // [count] pages that earlier requests give back
    int *pages = before + p.count;  // [count]
    const int tid = threadIdx.x, lane = tid & 31;
    const bool first_cta = blockIdx.x == 0;
    int count = *p.free_count;
    if (count < 0 || count > p.num_blocks) {
        if (first_cta && tid == 0) set_status(p.status, LC_DEV_BAD_BLOCK);
        count = max(0, min(count, p.num_blocks));
    }
    const int per = (p.count + kStepThreads - 1) / kStepThreads;
    const int b0 = tid * per, b1 = min(p.count, b0 + per);
    const int cap = p.table_stride * kBlockSize;
    int sum = 0, unused = 0;
    for (int b = b0; b < b1; ++b) {
        int c = p.ctx[b];
        const int slot = slot_of(p.slots, b);
        if (c < 0 || c > cap || slot < 0 || slot >= p.num_slots) {
            if (first_cta) set_status(p.status, LC_DEV_BAD_POS);
            c = 0;
        }
        pages[b] = pages_of(c);
        sum += pages[b];
    }
    int total, none;
    block_scan2(sum, unused, &total, &none);
    for (int b = b0; b < b1; ++b) {
        before[b] = sum;
        sum += pages[b];
    }
    const int room = p.num_blocks - count;
    if (first_cta && tid == 0 && total > room) set_status(p.status, LC_DEV_BAD_BLOCK);
    __syncthreads();
    bool last = false;
    if (tid == 0) last = take_ticket(p.ticket);

    // Tasks of kRowSegment pages, one warp each; a request's last page first, so that
    // the stack hands them out again in order.
    const int warps = gridDim.x * kStepWarps, warp = blockIdx.x * kStepWarps + (tid >> 5);
    const int segs = (p.table_stride + kRowSegment - 1) / kRowSegment;
    for (int t = warp; t < p.count * segs; t += warps) {
        const int b = t / segs, j0 = (t - b * segs) * kRowSegment;
        const int n = pages[b];
        if (j0 >= n) continue;
        const int *row = p.tables + (int64_t)slot_of(p.slots, b) * p.table_stride;
        int page[kRowSegment / 32];
#pragma unroll
        for (int i = 0; i < kRowSegment / 32; ++i) {
            const int j = j0 + lane + 32 * i;
            page[i] = j < n ? row[j] : 0;
        }
#pragma unroll
        for (int i = 0; i < kRowSegment / 32; ++i) {
            const int j = j0 + lane + 32 * i, at = before[b] + n - 1 - j;
            if (j >= n) continue;
            if (page[i] < 0 || page[i] >= p.num_blocks) set_status(p.status, LC_DEV_BAD_BLOCK);
            if (at < room) p.free_pages[count + at] = page[i];
        }
    }
    if (last) *p.count_out = count + min(total, room);
}

bool aligned4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

}  // namespace
}  // namespace lc

using namespace lc;

extern "C" size_t lc_step_workspace_size(void) { return 256; }

extern "C" int lc_step_tables(int *block_tables, int table_stride, int num_slots,
                              const int *slots, const int *context_lens, const int *new_lens,
                              int batch, const int *free_pages, const int *free_count,
                              int64_t num_blocks, int *step_tables, int step_stride,
                              int *positions, int *slot_map, int max_tokens, int *row_starts,
                              int *context_out, int *free_count_out, void *workspace,
                              size_t workspace_bytes, int *dev_status, lc_stream_t stream) {
    if (!block_tables || !context_lens || !new_lens || !free_pages || !free_count || !positions ||
        !slot_map || !row_starts || !context_out || !free_count_out)
        return LC_ERR_INVALID_ARGUMENT;
    if (batch < 0 || table_stride <= 0 || num_slots <= 0 || num_blocks <= 0 || max_tokens < 0 ||
        (step_tables && step_stride <= 0) || (!slots && batch > num_slots))
        return LC_ERR_INVALID_ARGUMENT;
    if (num_blocks > INT32_MAX / kBlockSize) return LC_ERR_INVALID_ARGUMENT;  // slots are int32
    if (batch > kStepMaxBatch) return LC_ERR_UNSUPPORTED_SHAPE;
    // sums of tokens and of pages stay int32
    if ((int64_t)std::max(batch, 1) * table_stride > INT32_MAX / kBlockSize ||
        (step_tables && (int64_t)std::max(batch, 1) * step_stride > INT32_MAX))
        return LC_ERR_UNSUPPORTED_SHAPE;
    if (!workspace || workspace_bytes < lc_step_workspace_size()) return LC_ERR_WORKSPACE_TOO_SMALL;
    if (!aligned4(workspace)) return LC_ERR_MISALIGNED;
    if (batch == 0 && max_tokens == 0 && free_count == free_count_out) return LC_OK;
    StepParams p{};
    p.tables = block_tables;
    p.table_stride = table_stride;
    p.num_slots = num_slots;
    p.slots = slots;
    p.ctx = context_lens;
    p.add = new_lens;
    p.batch = batch;
    p.free_pages = free_pages;
    p.free_count = free_count;
    p.num_blocks = (int)num_blocks;
    p.step_tables = step_tables;
    p.step_stride = step_stride;
    p.table_vec = aligned16(block_tables) && (table_stride & 3) == 0;
    p.step_vec = step_tables && aligned16(step_tables) && (step_stride & 3) == 0;
    p.positions = positions;
    p.slot_map = slot_map;
    p.max_tokens = max_tokens;
    p.tokens_vec = aligned16(positions) && aligned16(slot_map);
    p.row_starts = row_starts;
    p.ctx_out = context_out;
    p.count_out = free_count_out;
    p.ticket = (int *)workspace;
    p.status = dev_status;
    const int smem = (4 * batch + 1) * (int)sizeof(int);
    if (smem > kSmemUnasked) {
        const int rc = ensure_smem_attr((const void *)step_tables_kernel, smem);
        if (rc) return rc;
    }
    // A warp per task, two CTAs per SM at most.
    const int64_t width = step_tables ? std::max(step_stride, table_stride) : table_stride;
    const int64_t tasks = (int64_t)batch * ((width + kRowSegment - 1) / kRowSegment) +
                          ((int64_t)max_tokens + kTokenSegment - 1) / kTokenSegment;
    if (tasks > INT32_MAX / 2) return LC_ERR_UNSUPPORTED_SHAPE;
    const int grid = (int)std::min<int64_t>(std::max<int64_t>((tasks + kStepWarps - 1) / kStepWarps, 1),
                                            2 * sm_count());
    step_tables_kernel<<<grid, kStepThreads, smem, as_stream(stream)>>>(p);
    return launch_status();
}

extern "C" int lc_step_release(int *free_pages, const int *free_count, int64_t num_blocks,
                               const int *block_tables, int table_stride, int num_slots,
                               const int *slots, const int *context_lens, int count,
                               int *free_count_out, void *workspace, size_t workspace_bytes,
                               int *dev_status, lc_stream_t stream) {
    if (!free_pages || !free_count || !block_tables || !context_lens || !free_count_out)
        return LC_ERR_INVALID_ARGUMENT;
    if (count < 0 || table_stride <= 0 || num_slots <= 0 || num_blocks <= 0 ||
        (!slots && count > num_slots))
        return LC_ERR_INVALID_ARGUMENT;
    if (num_blocks > INT32_MAX / kBlockSize) return LC_ERR_INVALID_ARGUMENT;
    if (count > kStepMaxBatch ||
        (int64_t)std::max(count, 1) * table_stride > INT32_MAX / kBlockSize)
        return LC_ERR_UNSUPPORTED_SHAPE;
    if (!workspace || workspace_bytes < lc_step_workspace_size()) return LC_ERR_WORKSPACE_TOO_SMALL;
    if (!aligned4(workspace)) return LC_ERR_MISALIGNED;
    if (count == 0 && free_count == free_count_out) return LC_OK;
    ReleaseParams p{free_pages, free_count, (int)num_blocks, block_tables, table_stride, num_slots,
                    slots, context_lens, count, free_count_out, (int *)workspace, dev_status};
    const int smem = std::max(2 * count * (int)sizeof(int), 4);
    if (smem > kSmemUnasked) {
        const int rc = ensure_smem_attr((const void *)step_release_kernel, smem);
        if (rc) return rc;
    }
    const int64_t tasks = (int64_t)count * ((table_stride + kRowSegment - 1) / kRowSegment);
    const int grid = (int)std::min<int64_t>((tasks + kStepWarps - 1) / kStepWarps, 2 * sm_count());
    step_release_kernel<<<std::max(grid, 1), kStepThreads, smem, as_stream(stream)>>>(p);
    return launch_status();
}
