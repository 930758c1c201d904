// The index arrays of a step from its requests' lengths: sums of what is in front of every request, then for every row its request, token and
// slot, and for every new page its entry of the block table.
//
// Bound: a launch for batches that decode, bytes (16 a row, 8 a page) for prompts. One launch, and no CTA waits for another: every CTA sums all
// requests by itself -- a CHUNK of neighbours per thread, a sum over warps and CTA -- and then writes its share of the rows, four at a time
// per thread, and of the requests. A row finds its chunk by bisection of the chunks' sums in shared memory and its request by walking the
// chunk. (Handing the sums from CTA to CTA would read the lengths once instead of once per CTA; they are 8 bytes a request out of L2.)
// 64 requests of one token: 6.2 us on the device; 4000 prompts of 1 to 512 tokens (a million rows, 16 MB): 17.2 us, a third of it the sums that every
// CTA makes. (One CTA that went through the requests one by one: 30.8 and 2530 us. Plans that looked for neither rows to drop nor rows without a page
// took 5.8 and 15.7.)
#include "kernels.hpp"
#include "launch_utils.cuh"

#include "llaisys/paged_kv.h"

#include <algorithm>
#include <climits>

namespace llaisys::kernels {

namespace {

constexpr int kRowsAtOnce = 4;

struct Request {
    int row, held, fresh; // table row (-1: not in the table), tokens held and brought
    int held_pages, pages, grown;
};

__device__ __forceinline__ int pages_of(int tokens, const PlanArgs &p) {
    return p.page_shift >= 0 ? int((uint32_t(tokens) + uint32_t(p.page_size) - 1u) >> p.page_shift)
                             : int((uint32_t(tokens) + uint32_t(p.page_size) - 1u) / uint32_t(p.page_size));
}
// room: rows there are for it and whoever comes behind it
__device__ __forceinline__ Request load_request(const PlanArgs &p, int i, int room, int &flags) {
    Request q;
    q.row = p.seq_ids ? p.seq_ids[i] : i;
    q.held = p.held[i];
    q.fresh = p.fresh[i];
    if (q.held < 0 || q.fresh < 0 || q.fresh > INT_MAX - max(q.held, 0)) {
        flags |= LLAISYS_PLAN_BAD_COUNT;
        q.held = max(q.held, 0);
        q.fresh = 0;
    }
    q.fresh = min(q.fresh, room);
    if (p.table != nullptr && (q.row < 0 || q.row >= p.table_rows)) {
        flags |= LLAISYS_PLAN_BAD_ROW;
        q.row = -1;
    }
    q.held_pages = pages_of(q.held, p);
    q.pages = pages_of(q.held + q.fresh, p);
    q.grown = 0;
    if (p.table != nullptr && q.row >= 0 && q.fresh > 0) {
        if (q.pages > p.table_stride) {
            flags |= LLAISYS_PLAN_BAD_ROW;
        } else if (p.free_pages != nullptr) {
            q.grown = q.pages - q.held_pages;
        }
    }
    return q;
}

// The last chunk whose sum in front is not over x (chunks that add nothing in front of it are passed over).
template <int kChunks>
__device__ __forceinline__ int chunk_of(const int *sums, int x) {
    int lo = 0, hi = kChunks - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (sums[mid] <= x) {
            lo = mid;
        } else {
            hi = mid - 1;
        }
    }
    return lo;
}

template <int kThreads>
__global__ void __launch_bounds__(kThreads) paged_plan_kernel(PlanArgs p) {
    constexpr int kWarps = kThreads / 32;
    __shared__ int64_t s_warp[kWarps][3];
    __shared__ int s_rows[kThreads];     // rows in front of a chunk
    __shared__ int s_grown[kThreads];    // pages taken in front of it
    __shared__ int s_flags;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        s_flags = 0;
    }
    const int per = int((int64_t(p.n_seqs) + kThreads - 1) / kThreads), i0 = int(min(int64_t(tid) * per, int64_t(p.n_seqs)));
    const int i1 = i0 + min(per, p.n_seqs - i0);
    int flags;
    int64_t mine[3], before[3], total[3]; // rows, pages, pages taken: of this thread's chunk, in front of it, of all
    bool dropped = false;
    for (;;) {
        int64_t front = dropped ? min(before[0], int64_t(p.n_rows)) : 0;
        flags = 0;
        mine[0] = mine[1] = mine[2] = 0;
        for (int i = i0; i < i1; ++i) {
            const Request q = load_request(p, i, dropped ? int(p.n_rows - front) : INT_MAX, flags);
            front += q.fresh;
            mine[0] += q.fresh;
            mine[1] += q.pages;
            mine[2] += q.grown;
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            before[k] = mine[k];
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                const int64_t up = __shfl_up_sync(0xffffffffu, before[k], o);
                before[k] += lane >= o ? up : 0;
            }
        }
        if (lane == 31) {
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                s_warp[warp][k] = before[k];
            }
        }
        __syncthreads();
        if (flags != 0) {
            atomicOr(&s_flags, flags);
        }
        if (warp == 0) {
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                int64_t v = lane < kWarps ? s_warp[lane][k] : 0;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int64_t up = __shfl_up_sync(0xffffffffu, v, o);
                    v += lane >= o ? up : 0;
                }
                if (lane < kWarps) {
                    s_warp[lane][k] = v;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            before[k] += (warp > 0 ? s_warp[warp - 1][k] : 0) - mine[k];
            total[k] = s_warp[kWarps - 1][k];
        }
        if (dropped || total[0] <= p.n_rows) {
            break;
        }
        // More rows than there is room for: once more, without what is dropped, which then counts as not brought in lengths and pages too.
        dropped = true;
        __syncthreads();
        if (tid == 0) {
            s_flags = 0;
        }
    }
    const bool enough = total[2] <= p.n_free;
    s_rows[tid] = int(before[0]); // (n_rows at most by now)
    s_grown[tid] = int(min(before[2], int64_t(INT_MAX)));
    __syncthreads();

    // ---- this CTA's share of the requests, by warps: what is said about each
    if (warp * int(gridDim.x) / kWarps == int(blockIdx.x)) {
        int rows = int(before[0]);
        int64_t pages = before[1];
        for (int i = i0; i < i1; ++i) {
            const Request q = load_request(p, i, p.n_rows - rows, flags);
            if (p.q_starts) {
                p.q_starts[i] = rows;
            }
            if (p.kv_lens) {
                p.kv_lens[i] = q.held + q.fresh;
            }
            if (p.page_starts) {
                p.page_starts[i] = int(min(pages, int64_t(INT_MAX)));
            }
            rows += q.fresh;
            pages += q.pages;
        }
    }
    // ---- its share of the new entries of the table
    if (enough) {
        for (int64_t e = int64_t(blockIdx.x) * kThreads + tid; e < total[2]; e += int64_t(gridDim.x) * kThreads) {
            const int chunk = chunk_of<kThreads>(s_grown, int(e));
            int i = chunk * per, first = s_grown[chunk];
            int rows = s_rows[chunk];
            Request q = load_request(p, i, p.n_rows - rows, flags);
            while (e >= first + q.grown) {
                first += q.grown;
                rows += q.fresh;
                q = load_request(p, ++i, p.n_rows - rows, flags);
            }
            p.table[int64_t(q.row) * p.table_stride + q.held_pages + (e - first)] = p.free_pages[e];
        }
    }
    if (blockIdx.x == 0 && tid == 0) {
        if (p.q_starts) {
            p.q_starts[p.n_seqs] = int(total[0]);
        }
        if (p.page_starts) {
            p.page_starts[p.n_seqs] = int(min(total[1], int64_t(INT_MAX)));
        }
        if (p.status) {
            p.status[0] = enough ? int(total[2]) : 0;
            p.status[1] = s_flags | (enough ? 0 : LLAISYS_PLAN_NO_PAGES) | (dropped ? LLAISYS_PLAN_ROWS_DROPPED : 0);
        }
    }

    // ---- its share of the rows
    if (p.row_seqs == nullptr && p.row_positions == nullptr && p.row_slots == nullptr) {
        return;
    }
    const int live = int(total[0]);
    for (int64_t r0 = (int64_t(blockIdx.x) * kThreads + tid) * kRowsAtOnce; r0 < p.n_rows; r0 += int64_t(gridDim.x) * kThreads * kRowsAtOnce) {
        int seqs[kRowsAtOnce], positions[kRowsAtOnce];
        int64_t slots[kRowsAtOnce];
        const int lo = r0 < live ? chunk_of<kThreads>(s_rows, int(r0)) : 0;
        int i = lo * per;
        int start = s_rows[lo];
        int grown = s_grown[lo];
        Request q{};
        int entry = -1, page = -1; // the entry of the table that `page` is from
        bool loaded = false;
#pragma unroll
        for (int k = 0; k < kRowsAtOnce; ++k) {
            const int64_t r = r0 + k;
            seqs[k] = positions[k] = -1;
            slots[k] = -1;
            if (r >= live) {
                continue;
            }
            while (!loaded || r >= start + q.fresh) {
                if (loaded) {
                    start += q.fresh;
                    grown += q.grown;
                    ++i;
                }
                q = load_request(p, i, p.n_rows - start, flags);
                loaded = true;
                entry = -1;
            }
            const int pos = q.held + int(r - start);
            const int e = p.table == nullptr ? 0 : p.page_shift >= 0 ? pos >> p.page_shift : pos / p.page_size;
            const bool in_table = q.row >= 0 && e < p.table_stride, read = e < q.held_pages || p.free_pages == nullptr;
            if (p.table != nullptr && !(in_table && (read || (enough && q.grown > 0)))) {
                continue; // no page: what the table holds there is not this request's, so nothing is to be appended through it
            }
            seqs[k] = p.seq_ids ? p.seq_ids[i] : i;
            positions[k] = pos;
            if (p.row_slots != nullptr) {
                if (e != entry) {
                    entry = e;
                    // (a new page's entry may be another CTA's to write)
                    page = read ? p.table[int64_t(q.row) * p.table_stride + e] : p.free_pages[grown + e - q.held_pages];
                }
                slots[k] = page < 0 ? -1 : int64_t(page) * p.page_size + (pos - e * p.page_size);
            }
        }
        if (p.rows_wide && r0 + kRowsAtOnce <= p.n_rows) {
            if (p.row_seqs) {
                *reinterpret_cast<int4 *>(p.row_seqs + r0) = make_int4(seqs[0], seqs[1], seqs[2], seqs[3]);
            }
            if (p.row_positions) {
                *reinterpret_cast<int4 *>(p.row_positions + r0) = make_int4(positions[0], positions[1], positions[2], positions[3]);
            }
            if (p.row_slots) {
                *reinterpret_cast<longlong2 *>(p.row_slots + r0) = make_longlong2(slots[0], slots[1]);
                *reinterpret_cast<longlong2 *>(p.row_slots + r0 + 2) = make_longlong2(slots[2], slots[3]);
            }
            continue;
        }
#pragma unroll
        for (int k = 0; k < kRowsAtOnce; ++k) {
            if (r0 + k < p.n_rows) {
                if (p.row_seqs) {
                    p.row_seqs[r0 + k] = seqs[k];
                }
                if (p.row_positions) {
                    p.row_positions[r0 + k] = positions[k];
                }
                if (p.row_slots) {
                    p.row_slots[r0 + k] = slots[k];
                }
            }
        }
    }
}

} // namespace

void paged_plan(stream_t stream, const PlanArgs &args) {
    PlanArgs p = args;
    p.page_shift = -1;
    for (int s = 0; s < 31; ++s) {
        p.page_shift = p.page_size == 1 << s ? s : p.page_shift;
    }
    p.rows_wide = aligned16(p.row_seqs) && aligned16(p.row_positions) && aligned16(p.row_slots);
    const bool rows_wanted = p.row_seqs != nullptr || p.row_positions != nullptr || p.row_slots != nullptr;
    // Up to 512 requests, four a thread, small CTAs: their sums take two barriers of four warps instead of 32. A turn of a CTA is four rows a thread.
    auto start = [&](auto kernel, int threads) {
        const int64_t turns = (std::max<int64_t>(rows_wanted ? p.n_rows : 0, p.n_seqs) + threads * kRowsAtOnce - 1) / (threads * kRowsAtOnce);
        const int64_t most = int64_t(device_sms()) * (threads == 1024 ? 2 : 4);
        kernel<<<unsigned(std::max<int64_t>(1, std::min(turns, most))), threads, 0, static_cast<cudaStream_t>(stream)>>>(p);
    };
    if (p.n_seqs <= 512) {
        start(paged_plan_kernel<128>, 128);
    } else {
        start(paged_plan_kernel<1024>, 1024);
    }
    check_launch("paged_plan");
}

} // namespace llaisys::kernels
