// The index arrays of a step from its requests' lengths: sums of what is in front of every request, then for every row its request, token and
// slot, and for every new page its entry of the block table.
//
// One CTA goes through the requests 1024 at a time (a sum over the warp, one over the warps, a carry), then over rows and pages, which find
// their request by bisection of the sums.
#include "kernels.hpp"
#include "launch_utils.cuh"

#include "llaisys/paged_kv.h"

#include <climits>

namespace llaisys::kernels {

namespace {

constexpr int kThreads = 1024;

struct Request {
    int row, held, fresh; // table row (-1: not in the table), tokens held and brought
};

__device__ __forceinline__ Request load_request(const PlanArgs &p, int i, int &flags) {
    Request q;
    q.row = p.seq_ids ? p.seq_ids[i] : i;
    q.held = p.held[i];
    q.fresh = p.fresh[i];
    if (q.held < 0 || q.fresh < 0 || q.fresh > INT_MAX - max(q.held, 0)) {
        flags |= LLAISYS_PLAN_BAD_COUNT;
        q.held = max(q.held, 0);
        q.fresh = 0;
    }
    if (p.table != nullptr && (q.row < 0 || q.row >= p.table_rows)) {
        flags |= LLAISYS_PLAN_BAD_ROW;
        q.row = -1;
    }
    return q;
}
__device__ __forceinline__ int pages_of(int tokens, int page_size) { return int((int64_t(tokens) + page_size - 1) / page_size); }
// pages a request takes off the free list
__device__ __forceinline__ int growth(const PlanArgs &p, const Request &q, int &flags) {
    if (p.free_pages == nullptr || q.row < 0 || q.fresh == 0) {
        return 0;
    }
    const int after = pages_of(q.held + q.fresh, p.page_size);
    if (after > p.table_stride) {
        flags |= LLAISYS_PLAN_BAD_ROW;
        return 0;
    }
    return after - pages_of(q.held, p.page_size);
}

// Exclusive sum over the CTA of three numbers; `carry` comes in as the sum of what is in front and leaves with this lot's added.
__device__ __forceinline__ void scan3(int64_t (&v)[3], int64_t (&carry)[3], int64_t (*sums)[3]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t own[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        own[k] = v[k];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t up = __shfl_up_sync(0xffffffffu, v[k], o);
            v[k] += lane >= o ? up : 0;
        }
        if (lane == 31) {
            sums[warp][k] = v[k];
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        int64_t before = 0, all = 0;
        for (int w = 0; w < kThreads / 32; ++w) {
            before += w < warp ? sums[w][k] : 0;
            all += sums[w][k];
        }
        v[k] = carry[k] + before + v[k] - own[k];
        carry[k] += all;
    }
    __syncthreads();
}

__global__ void __launch_bounds__(kThreads) paged_plan_kernel(PlanArgs p) {
    __shared__ int64_t s_sums[kThreads / 32][3];
    __shared__ int s_flags;
    if (threadIdx.x == 0) {
        s_flags = 0;
    }
    __syncthreads();
    int flags = 0;
    // totals first: pages are taken all or not at all
    int64_t total[3] = {0, 0, 0};
    for (int base = 0; base < p.n_seqs; base += kThreads) {
        const int i = base + int(threadIdx.x);
        int64_t v[3] = {0, 0, 0};
        if (i < p.n_seqs) {
            const Request q = load_request(p, i, flags);
            v[2] = growth(p, q, flags);
        }
        scan3(v, total, s_sums);
    }
    const bool enough = total[2] <= p.n_free;
    int64_t carry[3] = {0, 0, 0};
    for (int base = 0; base < p.n_seqs; base += kThreads) {
        const int i = base + int(threadIdx.x);
        int64_t v[3] = {0, 0, 0};
        Request q{-1, 0, 0};
        int grown = 0;
        if (i < p.n_seqs) {
            q = load_request(p, i, flags);
            grown = growth(p, q, flags);
            v[0] = q.fresh;
            v[1] = pages_of(q.held + q.fresh, p.page_size);
            v[2] = grown;
        }
        scan3(v, carry, s_sums);
        if (i < p.n_seqs) {
            const int first = int(min(v[0], int64_t(p.n_rows)));
            if (p.q_starts) {
                p.q_starts[i] = first;
            }
            if (p.kv_lens) {
                p.kv_lens[i] = q.held + q.fresh;
            }
            if (p.page_starts) {
                p.page_starts[i] = int(min(v[1], int64_t(INT_MAX)));
            }
            const int held_pages = pages_of(q.held, p.page_size);
            if (enough) {
                for (int k = 0; k < grown; ++k) {
                    p.table[int64_t(q.row) * p.table_stride + held_pages + k] = p.free_pages[v[2] + k];
                }
            }
            const int rows = int(min(v[0] + q.fresh, int64_t(p.n_rows))) - first;
            for (int r = 0; r < rows; ++r) {
                const int pos = q.held + r, entry = pos / p.page_size;
                if (p.row_seqs) {
                    p.row_seqs[first + r] = p.seq_ids ? p.seq_ids[i] : i;
                }
                if (p.row_positions) {
                    p.row_positions[first + r] = pos;
                }
                if (p.row_slots) {
                    int page = -1;
                    if (q.row >= 0 && entry < p.table_stride && (entry < held_pages || p.free_pages == nullptr || (enough && grown > 0))) {
                        page = p.table[int64_t(q.row) * p.table_stride + entry];
                    }
                    p.row_slots[first + r] = page < 0 ? -1 : int64_t(page) * p.page_size + (pos - entry * p.page_size);
                }
            }
        }
    }
    for (int r = int(min(carry[0], int64_t(p.n_rows))) + int(threadIdx.x); r < p.n_rows; r += kThreads) {
        if (p.row_seqs) {
            p.row_seqs[r] = -1;
        }
        if (p.row_positions) {
            p.row_positions[r] = -1;
        }
        if (p.row_slots) {
            p.row_slots[r] = -1;
        }
    }
    atomicOr(&s_flags, flags);
    __syncthreads();
    if (threadIdx.x == 0) {
        if (p.q_starts) {
            p.q_starts[p.n_seqs] = int(min(carry[0], int64_t(p.n_rows)));
        }
        if (p.page_starts) {
            p.page_starts[p.n_seqs] = int(min(carry[1], int64_t(INT_MAX)));
        }
        if (p.status) {
            p.status[0] = enough ? int(total[2]) : 0;
            p.status[1] = s_flags | (enough ? 0 : LLAISYS_PLAN_NO_PAGES) | (carry[0] > p.n_rows ? LLAISYS_PLAN_ROWS_DROPPED : 0);
        }
    }
}

} // namespace

void paged_plan(stream_t stream, const PlanArgs &args) {
    paged_plan_kernel<<<1, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(args);
    check_launch("paged_plan");
}

} // namespace llaisys::kernels
