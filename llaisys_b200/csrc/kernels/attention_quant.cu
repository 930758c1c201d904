// Attention over a page pool held in 8 bits on the tensor cores of a warp (mma.sync m16n8k16): decode, and chunks of any length.
//
// Mathematics. Codes are integers or e4m3 numbers and so are exact in f16: scores are q k8^T times the block's K scale, the product of weights
// and V codes is taken in f16 too, and every sum is f32. Blocks differ in their V scale s_v = 2^e f (1 <= f < 2); with x the score in log2 units,
//     w = 2^(x + e - M + 14),   M = the running maximum of x + e,   out = sum (w f) v8 / sum w 2^-e
// so that the f16 weights w f lie below 2^15 however far the scales are apart, and the smallest normal one is 2^-28 of the largest. Queries are
// scaled by a power of two to below 2^15, row by row. For 32-bit activations q and the weights are taken as two f16 numbers each (22 bits).
//
// Bound: the pool's bytes. 16 tokens of a kv head are a tile of 32 d + 16 bytes that lies in one piece, so one bulk copy fetches it.
//
// Work. A row is (query, head of the group); 16 packed rows of a sequence and kv head are a TILE of rows, which visits its visible blocks of 16
// tokens, one UNIT each, and one more unit for what a tile costs besides. All units, in the order (sequence, row tile, kv head, block), form a line
// that is cut into equal pieces, one per CTA. A piece covers the end of one row tile, whole ones and the beginning of another; each such
// FRAGMENT is worked on by all eight warps, every one with every eighth block, and merged in shared memory. A fragment that is its whole
// row tile stores its rows; otherwise it leaves sums and maxima in a slot of the workspace, and the one that arrives last merges them, in the
// order of the CTAs. Nobody waits for another CTA.
// A warp feeds itself: it has a ring of slots of its own, asks for a block as soon as it has read the one that lay in the slot, and looks one
// fragment ahead, so that nothing but the merge makes warps meet; codes come out of a slot by 16-byte loads in the order the products want
// them (quant_tile.cuh). (A ninth warp for the copies would leave 168 registers a thread instead of 255, and the accumulators spill.)
// Waits for copies are bounded; one that runs out sets bit 8 of the error word, and the warp asks for nothing more.
#include "kernels.hpp"
#include "launch_utils.cuh"
#include "mma_utils.cuh"
#include "quant_tile.cuh"

#include <algorithm>
#include <type_traits>

namespace llaisys::kernels {

namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32, kRows = 16;
constexpr int kRingBytes = 132 * 1024, kMaxSlotsPerWarp = 8;
constexpr int kMinPiece = 8; // units of the shortest piece: a block for every warp
constexpr uint32_t kWaitLimit = 1u << 20;
constexpr int kErrTimeout = 8;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kShift = 14.f; // weights are 2^14 times what they stand for

template <int D>
struct Shape {
    static constexpr int kTile = 2 * kQuantTokens * D + 16;
    static constexpr int kSlots = kRingBytes / kWarps / kTile < kMaxSlotsPerWarp ? kRingBytes / kWarps / kTile : kMaxSlotsPerWarp; // of a warp
    static constexpr int kMergeDims = D < 128 ? D : 128; // dims merged at a time
    static constexpr int kMergeStride = kMergeDims + 8;  // floats between rows in the merge buffer: lanes 4 g + t store at banks 8 g + 2 t
    static constexpr size_t kMerge = size_t(kWarps) * kSlots * kTile, kStats = kMerge + size_t(kWarps) * kRows * kMergeStride * 4;
    static constexpr size_t kBars = kStats + 3 * kWarps * kRows * 4, kWords = kBars + kWarps * kSlots * 8, kQuery = kWords + 32;
    static constexpr size_t kBytes = kQuery + (D > 128 ? 2 * (D / 16) * 512 : 0); // (16 query rows of 256 dims stay in shared memory: 8 or 16 KiB)
};

struct QuantParams {
    QuantView kv;
    const int32_t *seq_ids, *kv_lens, *q_starts;
    int32_t n_seqs, total_q, nh, group;
    const void *q;
    void *out;
    float *part;
    float scale_log2;
    int32_t window, keep_first;
    const float *row_scale;
    int64_t out_stride;
    int32_t bf16; // of 16-bit activations: bfloat16
    float *partials;
    int32_t *counters;
    int32_t *error_flag;
};

// floats of one fragment's sums: accumulators [16][d], maxima, sums and score maxima
__host__ __device__ constexpr int partial_floats(int d) { return kRows * d + 3 * kRows; }

// sum of floor(i / m) over i < n
__device__ __forceinline__ int64_t floor_sum(int64_t n, int m) {
    const int64_t q = n / m, r = n - q * m;
    return m * (q * (q - 1) / 2) + q * r;
}
// sum of max(0, floor((i + c) / m)) over i < n
__device__ __forceinline__ int64_t floor_sum_from(int64_t n, int64_t c, int m) {
    if (n == 1) {
        return c > 0 ? int(c) / m : 0;
    }
    return n + c > 0 ? floor_sum(n + c, m) - floor_sum(max(c, int64_t(0)), m) : 0;
}

// What a sequence brings to the line.
struct SeqGeom {
    int q_start, q_len, off, tokens; // the query at t sees keys j <= t + off; tokens held
    int tiles;                       // row tiles per kv head
    int c_hi, c_gap;                 // blocks of row tile i: max(0, (i + c_hi) / group) less its gap max(0, (i + c_gap) / group)
    bool gaps;
};
__device__ __forceinline__ SeqGeom seq_geom(const QuantParams &p, int a) {
    SeqGeom g;
    if (p.q_starts != nullptr) {
        g.q_start = max(p.q_starts[a], 0);
        g.q_len = max(min(p.q_starts[a + 1], p.total_q) - g.q_start, 0);
    } else {
        g.q_start = a;
        g.q_len = 1;
    }
    const int64_t room = int64_t(p.kv.table_stride) * p.kv.blocks_per_page * kQuantTokens;
    g.tokens = int(min(int64_t(max(p.kv_lens[a], 0)), room));
    g.off = g.tokens - g.q_len;
    g.tiles = int((int64_t(g.q_len) * p.group + kRows - 1) / kRows);
    // keys that the last row of tile i may see end at (16 i + 15) / group + 1 + off: the blocks are that, divided by 16 and rounded up
    g.c_hi = int((kRows - 1 + int64_t(p.group) * (int64_t(g.off) + kQuantTokens)) >> 4);
    const int kept = (p.keep_first + kQuantTokens - 1) / kQuantTokens;
    g.gaps = p.window > 0;
    g.c_gap = int(max(int64_t(p.group) * (int64_t(g.off) + 1 - p.window - int64_t(kQuantTokens) * kept) >> 4, int64_t(-0x40000000))); // (an arithmetic shift: floor)
    return g;
}
__device__ __forceinline__ int64_t units_before(const QuantParams &p, const SeqGeom &g, int64_t tile) { // per kv head
    if (tile == 0) {
        return 0;
    }
    return tile + floor_sum_from(tile, g.c_hi, p.group) - (g.gaps ? floor_sum_from(tile, g.c_gap, p.group) : 0);
}

struct Fragment {
    int a, tile, kvh;
    int b0, b1;           // blocks of the row tile, counted without its gap; b0 = b1: none
    int gap, kept;        // blocks left out behind the first `kept`
    int rows;             // live rows
    bool begins, ends;    // whether the row tile's first and last units are in it
    int64_t first, last;  // the row tile on the line: its first unit, and the one behind its last
    SeqGeom g;
};

// Place on the line; every warp walks the same fragments.
struct Walker {
    int a;
    int64_t seq_begin, pos, end;
    SeqGeom g;
    int64_t seq_units;
};
__device__ __forceinline__ bool next_fragment(const QuantParams &p, Walker &w, Fragment &f) {
    if (w.pos >= w.end) {
        return false;
    }
    while (w.pos >= w.seq_begin + w.seq_units) {
        w.seq_begin += w.seq_units;
        if (++w.a >= p.n_seqs) {
            return false;
        }
        w.g = seq_geom(p, w.a);
        w.seq_units = units_before(p, w.g, w.g.tiles) * p.kv.nkvh;
    }
    const int64_t x = w.pos - w.seq_begin;
    int lo = 0, hi = w.g.tiles - 1; // last row tile whose first unit is not behind x
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (units_before(p, w.g, mid) * p.kv.nkvh <= x) {
            lo = mid;
        } else {
            hi = mid - 1;
        }
    }
    const int64_t before = units_before(p, w.g, lo) * p.kv.nkvh;
    const int span = int(units_before(p, w.g, int64_t(lo) + 1) - units_before(p, w.g, lo)), blocks = span - 1;
    f.a = w.a;
    f.tile = lo;
    f.kvh = int((x - before) / span);
    const int at = int(x - before - int64_t(f.kvh) * span);
    f.first = w.seq_begin + before + int64_t(f.kvh) * span;
    f.last = f.first + span;
    const int to = int(min(f.last, w.end) - f.first);
    f.begins = at == 0;
    f.ends = to == span;
    f.b0 = min(at, blocks);
    f.b1 = min(to, blocks);
    const int64_t gap = w.g.gaps && lo + w.g.c_gap > 0 ? (lo + w.g.c_gap) / p.group : 0;
    f.gap = int(gap);
    f.kept = gap > 0 ? (p.keep_first + kQuantTokens - 1) / kQuantTokens : 0;
    f.rows = int(min(int64_t(kRows), int64_t(w.g.q_len) * p.group - int64_t(lo) * kRows));
    f.g = w.g;
    w.pos = f.first + to;
    return true;
}

// Four codes (a word) as two pairs of f16.
template <bool kF8>
__device__ __forceinline__ void widen(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if constexpr (kF8) {
        const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xffffu), __NV_E4M3);
        const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3);
        lo = uint32_t(a.x) | (uint32_t(a.y) << 16);
        hi = uint32_t(b.x) | (uint32_t(b.y) << 16);
    } else { // 0x6400 | u is 1024 + u: with u = c + 128, 1152 less is c
        const uint32_t u = w ^ 0x80808080u;
        const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&a), off), y = __hsub2(*reinterpret_cast<const __half2 *>(&b), off);
        lo = *reinterpret_cast<const uint32_t *>(&x);
        hi = *reinterpret_cast<const uint32_t *>(&y);
    }
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 rest_of(uint32_t packed, float a, float b) { // what two f16 numbers leave of a and b
    const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&packed));
    return make_float2(a - h.x, b - h.y);
}
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); } // -126 <= e <= 127
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
// The blocks of a fragment that are a warp's: k-th one is block first + 8 k of the fragment. Lanes hold the tiles' places, 32 blocks at a time and
// the next 32 ahead.
struct Feed {
    const int32_t *table; // null: no such sequence
    int count, first, kept, gap, kvh;
    int now, next;
};
__device__ __forceinline__ int tile_place(const QuantParams &p, const Feed &f, int k) { // -1: no page
    if (k >= f.count) {
        return -1;
    }
    int block = f.first + kWarps * k;
    block = block < f.kept ? block : block + f.gap;
    const int entry = block / p.kv.blocks_per_page;
    if (f.table == nullptr || entry >= p.kv.table_stride) {
        atomicOr(p.error_flag, f.table == nullptr ? kErrBadSeq : kErrBadPosition);
        return -1;
    }
    const int page = f.table[entry];
    if (page < 0 || page >= p.kv.num_pages) {
        atomicOr(p.error_flag, kErrBadPage);
        return -1;
    }
    return (page * p.kv.blocks_per_page + block - entry * p.kv.blocks_per_page) * p.kv.nkvh + f.kvh;
}
__device__ __forceinline__ Feed open_feed(const QuantParams &p, const Fragment &f, int first, int lane) {
    Feed feed;
    const int seq = p.seq_ids[f.a];
    feed.table = seq >= 0 && seq < p.kv.table_rows ? p.kv.block_table + int64_t(seq) * p.kv.table_stride : nullptr;
    feed.first = f.b0 + first;
    feed.count = max(0, (f.b1 - feed.first + kWarps - 1) / kWarps);
    feed.kept = f.kept;
    feed.gap = f.gap;
    feed.kvh = f.kvh;
    feed.now = tile_place(p, feed, lane);
    feed.next = tile_place(p, feed, 32 + lane);
    return feed;
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
// Four neighbouring elements of a query row.
template <bool kWide>
__device__ __forceinline__ float4 load4(const void *q, int64_t at, bool bf16) {
    if constexpr (kWide) {
        return *reinterpret_cast<const float4 *>(static_cast<const float *>(q) + at);
    } else {
        const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const unsigned short *>(q) + at);
        if (bf16) {
            return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                               __uint_as_float(w.y & 0xffff0000u));
        }
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&w.y));
        return make_float4(a.x, a.y, b.x, b.y);
    }
}

// D: head dims, or the next of 64, 128 and 256 above them; kWide: 32-bit activations.
template <int D, bool kF8, bool kWide>
__global__ void __launch_bounds__(kThreads, 1) attention_quant_kernel(QuantParams p) {
    using S = Shape<D>;
    constexpr int kVecs = D / 32, kSteps = D / 16, kParts = kWide ? 2 : 1;
    constexpr bool kQueryShared = D > 128;
    extern __shared__ __align__(128) unsigned char smem[];
    float *s_merge = reinterpret_cast<float *>(smem + S::kMerge), *s_m = reinterpret_cast<float *>(smem + S::kStats);
    float *s_l = s_m + kWarps * kRows, *s_top = s_l + kWarps * kRows;
    int64_t *s_start = reinterpret_cast<int64_t *>(smem + S::kWords); // sequence of the piece's first unit, that sequence's first unit
    int *s_last = reinterpret_cast<int *>(s_start + 2);
    uint32_t *s_query = reinterpret_cast<uint32_t *>(smem + S::kQuery); // [part][step][lane][4]
    const uint32_t query_u32 = smem_u32(s_query);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int d = p.kv.d, vecs = d >> 5, tile_bytes = p.kv.tile_bytes;
    unsigned char *my_ring = smem + size_t(warp) * S::kSlots * S::kTile;
    const uint32_t ring = smem_u32(my_ring), bars = smem_u32(smem + S::kBars) + uint32_t(warp) * S::kSlots * 8;

    // ---- this CTA's piece of the line
    Walker w;
    int64_t piece;
    {
        if (lane == 0) {
            for (int i = 0; i < S::kSlots; ++i) {
                mbar_init(bars + 8 * i, 1);
            }
            mbar_init_fence();
        }
        int64_t *sums = reinterpret_cast<int64_t *>(s_merge);
        const int per = (p.n_seqs + kThreads - 1) / kThreads, a0 = min(tid * per, p.n_seqs), a1 = min(a0 + per, p.n_seqs);
        int64_t mine = 0;
        for (int a = a0; a < a1; ++a) {
            const SeqGeom g = seq_geom(p, a);
            mine += units_before(p, g, g.tiles) * p.kv.nkvh;
        }
        int64_t upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t up = __shfl_up_sync(0xffffffffu, upto, o);
            upto += lane >= o ? up : 0;
        }
        if (lane == 31) {
            sums[warp] = upto;
        }
        __syncthreads();
        int64_t line = 0, before = 0;
#pragma unroll
        for (int i = 0; i < kThreads / 32; ++i) {
            before += i < warp ? sums[i] : 0;
            line += sums[i];
        }
        piece = max((line + gridDim.x - 1) / gridDim.x, int64_t(kMinPiece));
        w.pos = min(piece * blockIdx.x, line);
        w.end = min(w.pos + piece, line);
        if (w.pos >= w.end) {
            return; // (the whole CTA)
        }
        int64_t begin = before + upto - mine;
        if (begin <= w.pos && w.pos < begin + mine) {
            int a = a0;
            for (; a < a1; ++a) {
                const SeqGeom g = seq_geom(p, a);
                const int64_t n = units_before(p, g, g.tiles) * p.kv.nkvh;
                if (w.pos < begin + n) {
                    break;
                }
                begin += n;
            }
            s_start[0] = a;
            s_start[1] = begin;
        }
        __syncthreads();
        w.a = int(s_start[0]);
        w.seq_begin = s_start[1];
        w.g = seq_geom(p, w.a);
        w.seq_units = units_before(p, w.g, w.g.tiles) * p.kv.nkvh;
        __syncthreads(); // the sums' place is the merge buffer's
    }
    Fragment f, ahead;
    uint32_t n = 0;                  // blocks of this CTA's fragments so far: the warps take them in turn
    uint32_t asked = 0, taken = 0;   // blocks of this warp: block c lies in slot c % kSlots
    uint32_t found = 0;              // bit s: the page of the block in slot s exists
    bool dead = false;               // a wait ran out
    const int g = lane >> 2, t = lane & 3;
    // asks for blocks of a feed from the k-th on, as far as there are slots
    auto ask = [&](Feed &feed, int &k) {
        while (k < feed.count && asked - taken < uint32_t(S::kSlots) && !dead) {
            const int place = __shfl_sync(0xffffffffu, feed.now, k & 31);
            const uint32_t slot = asked % S::kSlots;
            found = place >= 0 ? found | (1u << slot) : found & ~(1u << slot);
            if (lane == 0) {
                if (place >= 0) {
                    mbar_arrive_expect_tx(bars + 8 * slot, uint32_t(tile_bytes));
                    bulk_load(ring + slot * S::kTile, p.kv.base + int64_t(place) * tile_bytes, uint32_t(tile_bytes), bars + 8 * slot);
                } else {
                    mbar_arrive(bars + 8 * slot);
                }
            }
            ++asked;
            if ((++k & 31) == 0) {
                feed.now = feed.next;
                feed.next = tile_place(p, feed, k + 32 + lane);
            }
        }
    };
    bool more = next_fragment(p, w, ahead);
    Feed feed, feed_ahead = open_feed(p, ahead, warp, lane);
    int k_feed, k_ahead = 0;
    ask(feed_ahead, k_ahead);
    {
        while (more) {
            f = ahead;
            feed = feed_ahead;
            k_feed = k_ahead;
            const int first = int((uint32_t(warp) - n) & 7u);
            n += uint32_t(f.b1 - f.b0);
            k_ahead = 0;
            more = next_fragment(p, w, ahead);
            if (more) {
                feed_ahead = open_feed(p, ahead, int((uint32_t(warp) - n) & 7u), lane);
            } else {
                feed_ahead.count = 0;
            }
            ask(feed, k_feed);
            if (k_feed == feed.count) {
                ask(feed_ahead, k_ahead);
            }
            const int kvh = f.kvh, row0 = f.tile * kRows;
            // rows g and g + 8 of the tile: position of the query, and its fragments
            int pos[2];
            int64_t o_row[2]; // (query, head) as a row of out
            float factor[2];
            uint32_t qf[kParts][kQueryShared ? 1 : kSteps][4];
            auto query = [&](int part, int step) -> const uint32_t(&)[4] { return qf[part][kQueryShared ? 0 : step]; };
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = min(g + 8 * h, f.rows - 1), packed = row0 + r, query = packed / p.group, head = packed - query * p.group;
                pos[h] = query + f.g.off;
                o_row[h] = int64_t(f.g.q_start + query) * p.nh + kvh * p.group + head;
                float most = 0.f;
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
                    if (s < 2 * vecs) {
                        const float4 x = load4<kWide>(p.q, o_row[h] * d + 16 * s + 4 * t, p.bf16);
                        most = fmaxf(most, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
                    }
                }
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                const int e = max(-100, min(126, (__float_as_int(most) >> 23) - 127));
                const float up = power_of_two(14 - e);
                factor[h] = power_of_two(max(e - 14, -126)) * p.scale_log2;
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (s < 2 * vecs) {
                        x = load4<kWide>(p.q, o_row[h] * d + 16 * s + 4 * t, p.bf16);
                    }
                    x.x *= up, x.y *= up, x.z *= up, x.w *= up;
                    const uint32_t lo = pack_half2(x.x, x.y), hi = pack_half2(x.z, x.w);
                    const float2 a = rest_of(lo, x.x, x.y), b = rest_of(hi, x.z, x.w);
                    const uint32_t parts[2][2] = {{lo, hi}, {pack_half2(a.x, a.y), pack_half2(b.x, b.y)}};
#pragma unroll
                    for (int part = 0; part < kParts; ++part) {
                        if constexpr (!kQueryShared) {
                            qf[part][s][h] = parts[part][0];
                            qf[part][s][2 + h] = parts[part][1];
                        } else if (s % kWarps == warp) { // every warp has read the same rows: each leaves a share of the steps
                            uint32_t *to = s_query + ((part * kSteps + s) * 32 + lane) * 4;
                            to[h] = parts[part][0];
                            to[2 + h] = parts[part][1];
                        }
                    }
                }
            }
            if constexpr (kQueryShared) {
                __syncthreads();
            }
            const int first_pos = row0 / p.group + f.g.off, last_pos = (row0 + f.rows - 1) / p.group + f.g.off; // of the tile's rows

            float acc[4 * kVecs][4]; // [dims 8 i ..][row g: two dims, row g + 8: two dims]
#pragma unroll
            for (int i = 0; i < 4 * kVecs; ++i) {
                acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
            }
            float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, top[2] = {-INFINITY, -INFINITY};
            for (int i = first; i < f.b1 - f.b0 && !dead; i += kWarps) {
                const uint32_t slot = taken % S::kSlots;
                if (!mbar_wait_bounded(bars + 8 * slot, (taken / S::kSlots) & 1, kWaitLimit)) {
                    dead = true;
                }
                dead = __any_sync(0xffffffffu, dead);
                if (dead) {
                    // what else is on its way lands before the CTA ends
                    for (uint32_t c = taken; c != asked; ++c) {
                        mbar_wait_bounded(bars + 8 * (c % S::kSlots), (c / S::kSlots) & 1, 1u << 12);
                    }
                    if (lane == 0) {
                        atomicOr(p.error_flag, kErrTimeout);
                    }
                    break;
                }
                if (found >> slot & 1) {
                    const int k = f.b0 + i, token0 = (k < f.kept ? k : k + f.gap) * kQuantTokens;
                    const uint32_t tile = ring + slot * S::kTile;
                    const float2 scales = *reinterpret_cast<const float2 *>(my_ring + slot * S::kTile + quant_scales_at(d));
                    float s[2][4] = {};
#pragma unroll
                    for (int v = 0; v < kVecs; ++v) {
                        if (v < vecs) {
                            const uint4 words = lds128(tile + 16 * (32 * v + lane));
                            const uint32_t u[4] = {words.x, words.y, words.z, words.w};
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                uint32_t lo, hi;
                                widen<kF8>(u[j], lo, hi);
#pragma unroll
                                for (int part = 0; part < kParts; ++part) {
                                    if constexpr (kQueryShared) {
                                        if ((j & 1) == 0) {
                                            const uint4 x = lds128(query_u32 + 16 * ((part * kSteps + 2 * v + (j >> 1)) * 32 + lane));
                                            qf[part][0][0] = x.x, qf[part][0][1] = x.y, qf[part][0][2] = x.z, qf[part][0][3] = x.w;
                                        }
                                    }
                                    mma_16816<false>(s[j & 1], query(part, 2 * v + (j >> 1)), lo, hi);
                                }
                            }
                        }
                    }
                    // scores in log2 units, and whether all rows see all of the block
                    const bool whole = token0 + kQuantTokens - 1 <= first_pos && token0 + kQuantTokens <= f.g.tokens &&
                                       (p.window == 0 || last_pos - token0 < p.window || token0 + kQuantTokens <= p.keep_first);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float by = factor[h] * scales.x;
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            s[j][2 * h] *= by;
                            s[j][2 * h + 1] *= by;
                        }
                    }
                    if (!whole) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                const int token = token0 + 4 * t + 2 * j + (c & 1), at_pos = pos[c >> 1];
                                const bool seen = token <= at_pos && token < f.g.tokens &&
                                                  (p.window == 0 || at_pos - token < p.window || token < p.keep_first);
                                s[j][c] = seen ? s[j][c] : -INFINITY;
                            }
                        }
                    }
                    const int e = max(-100, min(126, ((__float_as_int(scales.y) >> 23) & 255) - 127));
                    const float fe = float(e), mantissa = scales.y * power_of_two(-e), down = power_of_two(-e);
                    uint32_t pf[kParts][4];
                    float alpha[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float most = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
                        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                        top[h] = fmaxf(top[h], most);
                        const float m_new = fmaxf(m[h], most + fe), base = m_new == -INFINITY ? 0.f : m_new - kShift - fe;
                        alpha[h] = m_new == -INFINITY ? 1.f : fast_exp2(m[h] - m_new);
                        m[h] = m_new;
                        float x[4], sum = 0.f;
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            x[c] = fast_exp2(s[c >> 1][2 * h + (c & 1)] - base);
                            sum += x[c];
                        }
                        l[h] = l[h] * alpha[h] + sum * down;
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            x[c] = !whole && s[c >> 1][2 * h + (c & 1)] == -INFINITY ? 0.f : x[c] * mantissa; // (a lost block's NaN stays where it is seen)
                        }
                        pf[0][h] = pack_half2(x[0], x[1]);
                        pf[0][2 + h] = pack_half2(x[2], x[3]);
                        if constexpr (kWide) {
                            const float2 a = rest_of(pf[0][h], x[0], x[1]), b = rest_of(pf[0][2 + h], x[2], x[3]);
                            pf[1][h] = pack_half2(a.x, a.y);
                            pf[1][2 + h] = pack_half2(b.x, b.y);
                        }
                    }
                    if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
                        for (int c = 0; c < 4 * kVecs; ++c) {
                            acc[c][0] *= alpha[0];
                            acc[c][1] *= alpha[0];
                            acc[c][2] *= alpha[1];
                            acc[c][3] *= alpha[1];
                        }
                    }
#pragma unroll
                    for (int v = 0; v < kVecs; ++v) {
                        if (v < vecs) {
                            const uint4 words = lds128(tile + kQuantTokens * d + 16 * (32 * v + lane));
                            const uint32_t u[4] = {words.x, words.y, words.z, words.w};
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                uint32_t lo, hi;
                                widen<kF8>(u[j], lo, hi);
                                mma_16816<false>(acc[4 * v + j], pf[0], lo, hi);
                                if constexpr (kWide) {
                                    mma_16816<false>(acc[4 * v + j], pf[1], lo, hi);
                                }
                            }
                        }
                    }
                }
                __syncwarp();
                ++taken;
                ask(feed, k_feed);
                if (k_feed == feed.count) {
                    ask(feed_ahead, k_ahead);
                }
            }

            // ---- the eight warps' sums
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
                if (t == 0) {
                    s_m[warp * kRows + g + 8 * h] = m[h];
                    s_l[warp * kRows + g + 8 * h] = l[h];
                    s_top[warp * kRows + g + 8 * h] = top[h];
                }
            }
            __syncthreads();
            float share[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float all = -INFINITY;
#pragma unroll
                for (int i = 0; i < kWarps; ++i) {
                    all = fmaxf(all, s_m[i * kRows + g + 8 * h]);
                }
                share[h] = all == -INFINITY ? 1.f : fast_exp2(m[h] - all);
            }
            const bool whole_tile = f.begins && f.ends;
            float *slot_of_mine = p.partials + (int64_t(blockIdx.x) * 2 + (f.begins ? 1 : 0)) * partial_floats(d);
            // statistics of the tile's rows, by every thread for the row it stores
            const int out_row = tid >> 4, out_lane = tid & 15;
            float m_all = -INFINITY, l_all = 0.f, top_all = -INFINITY;
#pragma unroll
            for (int i = 0; i < kWarps; ++i) {
                m_all = fmaxf(m_all, s_m[i * kRows + out_row]);
                top_all = fmaxf(top_all, s_top[i * kRows + out_row]);
            }
#pragma unroll
            for (int i = 0; i < kWarps; ++i) {
                l_all += s_l[i * kRows + out_row] * (m_all == -INFINITY ? 1.f : fast_exp2(s_m[i * kRows + out_row] - m_all));
            }
#pragma unroll
            for (int c0 = 0; c0 < D; c0 += S::kMergeDims) {
                if (c0 < d) {
#pragma unroll
                    for (int i = 0; i < S::kMergeDims / 8; ++i) {
                        const float *x = acc[c0 / 8 + i];
                        float *at = s_merge + (warp * kRows + g) * S::kMergeStride + 8 * i + 2 * t;
                        *reinterpret_cast<float2 *>(at) = make_float2(x[0] * share[0], x[1] * share[0]);
                        *reinterpret_cast<float2 *>(at + 8 * S::kMergeStride) = make_float2(x[2] * share[1], x[3] * share[1]);
                    }
                    __syncthreads();
                    const float inv = l_all == 0.f ? 0.f : 1.f / l_all;
                    const int packed = row0 + out_row, query = packed / p.group, head = packed - query * p.group;
                    const int64_t row = int64_t(f.g.q_start + query), o = row * p.nh + kvh * p.group + head;
#pragma unroll
                    for (int i = 0; i < S::kMergeDims / 64; ++i) { // four dims at a time
                        const int dim = 64 * i + 4 * out_lane;
                        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                        for (int k = 0; k < kWarps; ++k) {
                            const float4 x = *reinterpret_cast<const float4 *>(s_merge + (k * kRows + out_row) * S::kMergeStride + dim);
                            sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
                        }
                        if (c0 + dim >= d) {
                            continue;
                        }
                        if (!whole_tile) {
                            __stcg(reinterpret_cast<float4 *>(slot_of_mine + out_row * d + c0 + dim), sum);
                        } else if (out_row < f.rows) {
                            sum.x *= inv, sum.y *= inv, sum.z *= inv, sum.w *= inv;
                            if (p.part != nullptr) {
                                float *to = p.part + o * (d + 2) + c0 + dim;
                                to[0] = sum.x, to[1] = sum.y, to[2] = sum.z, to[3] = sum.w;
                            } else {
                                const float by = p.row_scale != nullptr ? p.row_scale[o] : 1.f;
                                const int64_t to = row * p.out_stride + int64_t(kvh * p.group + head) * d + c0 + dim;
                                const float v[4] = {sum.x * by, sum.y * by, sum.z * by, sum.w * by};
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    if constexpr (kWide) {
                                        static_cast<float *>(p.out)[to + k] = v[k];
                                    } else if (p.bf16) {
                                        static_cast<__nv_bfloat16 *>(p.out)[to + k] = __float2bfloat16_rn(v[k]);
                                    } else {
                                        static_cast<__half *>(p.out)[to + k] = __float2half_rn(v[k]);
                                    }
                                }
                            }
                        }
                    }
                    __syncthreads(); // the buffer is free again
                }
            }
            if (whole_tile) {
                if (p.part != nullptr && out_lane == 0 && out_row < f.rows) {
                    const int packed = row0 + out_row, query = packed / p.group, head = packed - query * p.group;
                    float *to = p.part + (int64_t(f.g.q_start + query) * p.nh + kvh * p.group + head) * (d + 2) + d;
                    to[0] = top_all * kLn2;
                    to[1] = top_all == -INFINITY ? l_all : l_all * fast_exp2(m_all - kShift - top_all);
                }
                continue;
            }
            // ---- one of several fragments of its tile
            if (out_lane == 0) {
                float *stats = slot_of_mine + kRows * d;
                __stcg(stats + out_row, m_all);
                __stcg(stats + kRows + out_row, l_all);
                __stcg(stats + 2 * kRows + out_row, top_all);
            }
            const int c_first = int(f.first / piece), c_last = int((f.last - 1) / piece);
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const int seen = atomicAdd(p.counters + c_first, 1);
                *s_last = seen == c_last - c_first;
                if (*s_last) {
                    p.counters[c_first] = 0;
                }
            }
            __syncthreads();
            if (*s_last) {
                __threadfence();
                float m_tile = -INFINITY, l_tile = 0.f, top_tile = -INFINITY;
                for (int c = c_first; c <= c_last; ++c) {
                    const float *stats = p.partials + (int64_t(c) * 2 + (c == c_first ? 1 : 0)) * partial_floats(d) + kRows * d;
                    m_tile = fmaxf(m_tile, __ldcg(stats + out_row));
                    top_tile = fmaxf(top_tile, __ldcg(stats + 2 * kRows + out_row));
                }
                float4 sum[D / 64] = {};
                for (int c = c_first; c <= c_last; ++c) {
                    const float *from = p.partials + (int64_t(c) * 2 + (c == c_first ? 1 : 0)) * partial_floats(d);
                    const float by = m_tile == -INFINITY ? 1.f : fast_exp2(__ldcg(from + kRows * d + out_row) - m_tile);
                    l_tile += __ldcg(from + kRows * d + kRows + out_row) * by;
#pragma unroll
                    for (int i = 0; i < D / 64; ++i) {
                        const int dim = 64 * i + 4 * out_lane;
                        if (dim < d) {
                            const float4 x = __ldcg(reinterpret_cast<const float4 *>(from + out_row * d + dim));
                            sum[i].x += x.x * by, sum[i].y += x.y * by, sum[i].z += x.z * by, sum[i].w += x.w * by;
                        }
                    }
                }
                if (out_row < f.rows) {
                    const float inv = l_tile == 0.f ? 0.f : 1.f / l_tile;
                    const int packed = row0 + out_row, query = packed / p.group, head = packed - query * p.group;
                    const int64_t row = int64_t(f.g.q_start + query), o = row * p.nh + kvh * p.group + head;
                    const float by = inv * (p.row_scale != nullptr && p.part == nullptr ? p.row_scale[o] : 1.f);
#pragma unroll
                    for (int i = 0; i < D / 64; ++i) {
                        const int dim = 64 * i + 4 * out_lane;
                        if (dim < d) {
                            const float v[4] = {sum[i].x * by, sum[i].y * by, sum[i].z * by, sum[i].w * by};
                            const int64_t to = row * p.out_stride + int64_t(kvh * p.group + head) * d + dim;
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                if (p.part != nullptr) {
                                    p.part[o * (d + 2) + dim + k] = v[k];
                                } else if constexpr (kWide) {
                                    static_cast<float *>(p.out)[to + k] = v[k];
                                } else if (p.bf16) {
                                    static_cast<__nv_bfloat16 *>(p.out)[to + k] = __float2bfloat16_rn(v[k]);
                                } else {
                                    static_cast<__half *>(p.out)[to + k] = __float2half_rn(v[k]);
                                }
                            }
                        }
                    }
                    if (p.part != nullptr && out_lane == 0) {
                        float *to = p.part + o * (d + 2) + d;
                        to[0] = top_tile * kLn2;
                        to[1] = top_tile == -INFINITY ? l_tile : l_tile * fast_exp2(m_tile - kShift - top_tile);
                    }
                }
            }
        }
    }
}

} // namespace

void attention_quant_scratch(int32_t d, size_t *floats, size_t *counters) {
    *floats = size_t(device_sms()) * 2 * partial_floats(d);
    *counters = size_t(device_sms());
}

void attention_quant(stream_t stream, llaisysDataType_t dtype, const QuantView &kv, const AttnBatch &batch, const void *q, float scale,
                     const AttnOut &out, const AttnScratch &scratch) {
    QuantParams p{};
    p.kv = kv;
    p.seq_ids = batch.seq_ids;
    p.kv_lens = batch.kv_lens;
    p.q_starts = batch.q_starts;
    p.n_seqs = batch.n_seqs;
    p.total_q = batch.total_q;
    p.nh = batch.nh;
    p.group = batch.nh / kv.nkvh;
    p.q = q;
    p.out = out.out;
    p.part = out.part;
    p.scale_log2 = scale * kLog2e;
    p.window = batch.window;
    p.keep_first = batch.window > 0 ? batch.keep_first : 0;
    p.row_scale = out.row_scale;
    p.out_stride = out.row_stride ? out.row_stride : int64_t(batch.nh) * kv.d;
    p.bf16 = dtype == LLAISYS_DTYPE_BF16;
    p.partials = scratch.partials;
    p.counters = scratch.counters;
    p.error_flag = scratch.error_flag;
    const unsigned sms = unsigned(device_sms());
    CHECK_ARGUMENT(aligned16(q), "attention: queries must be 16-byte aligned");
    CHECK_ARGUMENT(int64_t(batch.total_q) * p.group <= 0x7fffffff - kRows, "attention: too many rows for one launch");
    CHECK_ARGUMENT(scratch.partials_floats >= size_t(sms) * 2 * partial_floats(kv.d) && scratch.counters_len >= sms, "attention: workspace too small");
    auto launch = [&](auto d) {
        constexpr int D = decltype(d)::value;
        auto start = [&](auto kernel) {
            LLAISYS_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(Shape<D>::kBytes)));
            kernel<<<sms, kThreads, Shape<D>::kBytes, static_cast<cudaStream_t>(stream)>>>(p);
        };
        if (dtype == LLAISYS_DTYPE_F32) {
            start(kv.f8 ? attention_quant_kernel<D, true, true> : attention_quant_kernel<D, false, true>);
        } else {
            start(kv.f8 ? attention_quant_kernel<D, true, false> : attention_quant_kernel<D, false, false>);
        }
    };
    if (kv.d <= 64) {
        launch(std::integral_constant<int, 64>{});
    } else if (kv.d <= 128) {
        launch(std::integral_constant<int, 128>{});
    } else {
        launch(std::integral_constant<int, 256>{});
    }
    check_launch("attention_quant");
}

} // namespace llaisys::kernels
