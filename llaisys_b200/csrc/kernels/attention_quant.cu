// Attention over a page pool held in 8 bits on the tensor cores of a warp (mma.sync m16n8k16): decode, and chunks of any length.
//
// Mathematics. Codes are integers or e4m3 numbers and so are exact in f16: scores are q k8^T times the block's K scale, the product of weights
// and V codes is taken in f16 too, and every sum is f32. Blocks differ in their V scale s_v = 2^e f (1 <= f < 2); with x the score in log2 units,
//     w = 2^(x + e - M + 14),   M = the running maximum of x + e,   out = sum (w f) v8 / sum w 2^-e
// so that the f16 weights w f lie below 2^15 however far the scales are apart, and the smallest normal one is 2^-28 of the largest. Queries are
// scaled by a power of two to below 2^15, row by row. For 32-bit activations q and the weights are taken as two f16 numbers each (22 bits), and
// the tensor cores, which cut their sums where additions round, add up only 16 dims or 32 tokens at a time: over 8000 tokens of
// 256 dims the error is 5.7e-7 of the outputs instead of 1.2e-6, for 0.5 us of 29.6 (24 sequences, windows of 2000 tokens). The sum of the weights
// loses tokens whose x + e lies 140 below M: of blocks whose V scales are that many powers of two below the largest, at like scores.
//
// Bound: the pool's bytes. 16 tokens of a kv head are a tile of 32 d + 16 bytes that lies in one piece, so one bulk copy fetches it.
//
// Work. A row is (query, head of the group); 16 packed rows of a sequence and kv head are a TILE of rows, which visits its visible blocks of 16
// tokens, one UNIT each, and kTileUnits more for what a tile costs besides. All units, in the order (sequence, row tile, kv head, block), form a line
// that is cut into equal pieces, one per CTA. A piece covers the end of one row tile, whole ones and the beginning of another; each such
// FRAGMENT is worked on by all warps, which take its blocks in turn (heads of up to 128: two at a time), and merged in shared memory. A fragment that is its whole
// row tile stores its rows; otherwise it leaves sums and maxima in a slot of the workspace, and the one that arrives last merges them, in the
// order of the CTAs. Nobody waits for another CTA.
// A warp feeds itself: it has a ring of slots of its own, asks for a block as soon as it has read the one that lay in the slot, and looks one
// fragment ahead, so that nothing but the merge makes warps meet; codes come out of a slot by 16-byte loads in the order the products want
// them (quant_tile.cuh). (A ninth warp for the copies would leave 168 registers a thread instead of 255, and the accumulators spill.)
// Measured: 64 sequences of 4096 tokens, 12 / 2 heads of 128, integers, 33 us (135 MB: 4.1 TB/s; the loop over blocks runs at about 6, the rest is the
// start, the queries, the merge of the warps and the join of the 2.3 parts that a tile is in); one sequence of 777 tokens 10.3 us.
// Waits for copies are bounded; one that runs out sets bit 8 of the error word, and the warp asks for nothing more.
#include "kernels.hpp"
#include "launch_utils.cuh"
#include "mma_utils.cuh"
#include "quant_tile.cuh"

#include <algorithm>
#include <type_traits>

namespace llaisys::kernels {

namespace {

constexpr int kRows = 16;
constexpr int kMinPiece = 12; // units of the shortest piece
constexpr int kTileUnits = 24; // what a row tile costs besides its blocks, in units of a block's time
constexpr int kSnap = 8;       // a piece's border that comes this near a row tile's first or last block moves there: no fragments of a few blocks
constexpr uint32_t kDrainLimit = 1u << 20;
constexpr int kErrTimeout = 8;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kShift = 14.f; // weights are 2^14 times what they stand for
// Smallest power of two taken out of a V scale. A row's sum has 2^14 2^-e for a token of the largest weight: 2^31 tokens of the smallest scale (values
// all zero, say) stay below 2^128. What is left of scales below 2^-82 is in the weights, of which the f16 numbers then carry fewer bits below the largest.
constexpr int kLeastPower = -82;
constexpr size_t kPlaceBytes = 512;
// Blocks of a warp after which what the outputs of integer codes have too much is taken off them. It is 128 sum w beside sums of a few w, the tensor cores
// cut every addition to 2^-23 of that, always downwards, and so what an output lacks grew with the tokens: at 16384 tokens a sequence, equal weights, 5e-3
// of the output; taken off every 256 tokens of a warp it stays where 256 tokens have it.
constexpr int kFold = 16;

// Heads of up to 128: two CTAs of four warps on an SM, each warp with two blocks at a time and 255 registers. Longer ones: one CTA of eight warps.
// Three CTAs where 168 registers do (tiles of 8 rows, heads of up to 64): 24 sequences, windows of 2000 tokens, 24.7 us instead of 26.4; with heads of
// 128 the shorter rings cost more than the third CTA brings, 64 sequences of 4096 tokens 33.8 us instead of 33.0.
// R: rows that a warp multiplies at a time, 16 or 8 (see the kernel).
template <int D, int R>
struct Shape {
    static constexpr int kCtas = D <= 64 && R == 8 ? 3 : D <= 128 ? 2 : 1, kWarps = D <= 128 ? 4 : 8, kThreads = kWarps * 32, kPair = D <= 128 ? 2 : 1;
    static constexpr int kTile = 2 * kQuantTokens * D + 16;
    static constexpr int kSlots = D <= 64 ? kCtas == 3 ? 6 : 8 : D <= 128 ? 4 : 2;           // of a warp
    static constexpr int kMergeDims = D < 128 ? D : 128;                      // merged at a time
    // floats between rows in the merge buffer: lanes 4 g + t store at banks 8 g + 2 t (8 rows: 8 t + g)
    static constexpr int kMergeStride = kMergeDims + (R == 16 ? 8 : 4);
    static constexpr int kRowThreads = kThreads / R, kStep = 4 * kRowThreads; // threads that load and store a row, four dims each; dims between theirs
    static constexpr size_t kMerge = size_t(kWarps) * kSlots * kTile, kStats = kMerge + size_t(kWarps) * R * kMergeStride * 4;
    static constexpr size_t kBars = kStats + 3 * kWarps * kRows * 4, kWords = kBars + kWarps * kSlots * 8, kPlaces = kWords + 96 + 3 * kRows * 4;
    static constexpr size_t kPending = kPlaces + kWarps * kPlaceBytes; // fragments of tiles that other CTAs have parts of: at most two
    static constexpr size_t kRaw = kPending + 256;                     // the next tile's query rows as they are
    static constexpr size_t kQuery = kMerge; // query rows as fragments, 2 R bytes a dim, twice; the merge comes after their last use
    static constexpr size_t bytes(bool wide) { return kRaw + R * D * (wide ? 4 : 2); }
    static_assert(2 * 2 * R * D <= kWarps * R * kMergeStride * 4 && kStats % 16 == 0 && bytes(true) <= 227 / kCtas * 1024 && kRaw % 16 == 0, "");
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
    int32_t overlap;  // the launch may begin under the kernel in front of it
    int32_t out_wide; // four outputs of a row can be stored at once
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
    return kTileUnits * tile + floor_sum_from(tile, g.c_hi, p.group) - (g.gaps ? floor_sum_from(tile, g.c_gap, p.group) : 0);
}

__device__ __forceinline__ int tile_blocks(const QuantParams &p, const SeqGeom &g, int tile, int &gap) {
    gap = g.gaps && tile + g.c_gap > 0 ? (tile + g.c_gap) / p.group : 0;
    return (tile + g.c_hi > 0 ? (tile + g.c_hi) / p.group : 0) - gap;
}

struct Fragment {
    int a, q_start, off, tokens; // of the sequence
    int row0, rows, kvh;         // first packed row of the tile, live rows
    int b0, b1;                  // blocks of the row tile, counted without its gap; b0 = b1: none
    int kept, gap;               // gap blocks are left out behind the first `kept`
    bool begins, ends;           // whether the row tile's first and last blocks are in it
    int blocks;                  // of the row tile
    int64_t first;               // the tile's first unit on the line
};
// Place on the line: a row tile and kv head, and how far the piece goes.
struct Walker {
    int a, tile, kvh, blocks, gap;
    int64_t first, pos, end;
    SeqGeom g;
};
__device__ __forceinline__ int snap_of(int blocks) { return min(kSnap, blocks / 2); }
// where in a row tile a border lies that is x units behind its first
__device__ __forceinline__ int snapped(int64_t x, int blocks) {
    const int near = snap_of(blocks);
    return x <= near ? 0 : x >= blocks - near ? blocks + kTileUnits : int(x);
}
__device__ __forceinline__ bool next_fragment(const QuantParams &p, Walker &w, Fragment &f) {
    while (w.pos < w.end) {
        while (w.pos >= w.first + w.blocks + kTileUnits) {
            w.first += w.blocks + kTileUnits;
            if (++w.kvh == p.kv.nkvh) {
                w.kvh = 0;
                ++w.tile;
                while (w.tile >= w.g.tiles) {
                    if (++w.a >= p.n_seqs) {
                        return false;
                    }
                    w.tile = 0;
                    w.g = seq_geom(p, w.a);
                }
                w.blocks = tile_blocks(p, w.g, w.tile, w.gap);
            }
        }
        const int span = w.blocks + kTileUnits, at = snapped(w.pos - w.first, w.blocks), to = snapped(w.end - w.first, w.blocks);
        w.pos = w.first + span;
        if (at >= to) {
            continue; // the neighbours' pieces take it
        }
        f.a = w.a;
        f.q_start = w.g.q_start;
        f.off = w.g.off;
        f.tokens = w.g.tokens;
        f.row0 = w.tile * kRows;
        f.rows = min(kRows, w.g.q_len * p.group - f.row0);
        f.kvh = w.kvh;
        f.b0 = at;
        // (a last tile of fewer than 16 rows is counted as a full one, whose rows would see keys behind the sequence)
        f.b1 = max(min(min(to, w.blocks), (w.g.tokens + kQuantTokens - 1) / kQuantTokens - w.gap), at);
        f.gap = w.gap;
        f.kept = w.gap > 0 ? (p.keep_first + kQuantTokens - 1) / kQuantTokens : 0;
        f.begins = at == 0;
        f.ends = to == span;
        f.blocks = w.blocks;
        f.first = w.first;
        return true;
    }
    return false;
}

// Four codes (a word) as two pairs of f16. Integers lie in the pool as u = c + 128. 0x6400 | u is 1024 + u, so 1152 less is c; the bits of u
// alone are u 2^-24, exactly, which saves the subtraction where the caller makes good for it (kBiased).
template <bool kF8, bool kBiased>
__device__ __forceinline__ void widen(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if constexpr (kF8) {
        const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xffffu), __NV_E4M3);
        const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3);
        lo = uint32_t(a.x) | (uint32_t(a.y) << 16);
        hi = uint32_t(b.x) | (uint32_t(b.y) << 16);
    } else if constexpr (kBiased) {
        lo = __byte_perm(w, 0, 0x4140);
        hi = __byte_perm(w, 0, 0x4342);
    } else {
        const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
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
// The blocks of a fragment that are a warp's: the warps take kPair neighbours each, in turn. Lanes hold the tiles' places, 32 blocks at a time
// and the next 32 ahead.
struct Feed {
    int row; // of the table; -1: no such sequence
    int count, first, kept, gap, kvh;
    int now, next;
};
// What a warp keeps in shared memory, off the registers of its loop over blocks.
struct Place {
    Walker walker;
    Fragment ahead;
    Feed feed; // of the fragment ahead; now and next of the lanes beside it
    int now[32], next[32];
};
// The sequence of a piece's first unit, that sequence's first unit, and what is known of it.
struct Start {
    int64_t begin;
    int a, seq;
    SeqGeom g;
};
static_assert(sizeof(Start) <= 72, "shared memory");
static_assert(sizeof(Place) <= kPlaceBytes && alignof(Place) == 8 && 2 * sizeof(Fragment) <= 256, "shared memory");
template <typename S>
__device__ __forceinline__ int tile_place(const QuantParams &p, const Feed &f, int k) { // -1: no page
    if (k >= f.count) {
        return -1;
    }
    int block = f.first + S::kWarps * (k - k % S::kPair) + k % S::kPair;
    block = block < f.kept ? block : block + f.gap;
    const int entry = p.kv.blocks_per_page == 1 ? block : block / p.kv.blocks_per_page;
    const int page = p.kv.block_table[int64_t(max(f.row, 0)) * p.kv.table_stride + min(entry, p.kv.table_stride - 1)]; // (in the table whatever comes of it)
    const int what = f.row < 0 ? kErrBadSeq : entry >= p.kv.table_stride ? kErrBadPosition : page < 0 || page >= p.kv.num_pages ? kErrBadPage : 0;
    if (what != 0) {
        atomicOr(p.error_flag, what);
        return -1;
    }
    return (page * p.kv.blocks_per_page + block - entry * p.kv.blocks_per_page) * p.kv.nkvh + f.kvh;
}
// first: the first of the fragment's blocks that is the warp's
template <typename S>
__device__ __forceinline__ Feed open_feed(const QuantParams &p, const Fragment &f, int seq, int first, int lane) {
    Feed feed;
    const int blocks = f.b1 - f.b0 - first, sweep = S::kPair * S::kWarps;
    feed.row = seq >= 0 && seq < p.kv.table_rows ? seq : -1;
    feed.first = f.b0 + first;
    feed.count = blocks <= 0 ? 0 : blocks / sweep * S::kPair + min(blocks % sweep, S::kPair);
    feed.kept = f.kept;
    feed.gap = f.gap;
    feed.kvh = f.kvh;
    feed.now = tile_place<S>(p, feed, lane);
    feed.next = tile_place<S>(p, feed, 32 + lane);
    return feed;
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
// d = a b, sums that begin at zero.
__device__ __forceinline__ void mma_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// Four neighbouring elements of a query row in shared memory.
template <bool kWide>
__device__ __forceinline__ float4 load4(const unsigned char *q, int at, bool bf16) {
    if constexpr (kWide) {
        return *reinterpret_cast<const float4 *>(q + 4 * at);
    } else {
        const uint2 w = *reinterpret_cast<const uint2 *>(q + 2 * at);
        if (bf16) {
            return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                               __uint_as_float(w.y & 0xffff0000u));
        }
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&w.y));
        return make_float4(a.x, a.y, b.x, b.y);
    }
}

// Four outputs of a row.
template <bool kWide>
__device__ __forceinline__ void store4(const QuantParams &p, int64_t at, float4 v) {
    if constexpr (kWide) {
        float *to = static_cast<float *>(p.out) + at;
        if (p.out_wide) {
            *reinterpret_cast<float4 *>(to) = v;
        } else {
            to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
        }
    } else {
        uint2 w;
        if (p.bf16) {
            const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
            w = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
        } else {
            w = make_uint2(pack_half2(v.x, v.y), pack_half2(v.z, v.w));
        }
        unsigned short *to = static_cast<unsigned short *>(p.out) + at;
        if (p.out_wide) {
            *reinterpret_cast<uint2 *>(to) = w;
        } else {
            to[0] = static_cast<unsigned short>(w.x), to[1] = static_cast<unsigned short>(w.x >> 16);
            to[2] = static_cast<unsigned short>(w.y), to[3] = static_cast<unsigned short>(w.y >> 16);
        }
    }
}

// Four numbers of a finished row `o` ((query, head)), and a partial result's statistics.
template <bool kWide>
__device__ __forceinline__ void finish(const QuantParams &p, int64_t o, int64_t out_at, int dim, float4 v, float by) {
    v.x *= by, v.y *= by, v.z *= by, v.w *= by;
    if (p.part != nullptr) {
        float *to = p.part + o * (p.kv.d + 2) + dim;
        to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
    } else {
        store4<kWide>(p, out_at + dim, v);
    }
}
__device__ __forceinline__ void finish_stats(const QuantParams &p, int64_t o, float m, float l, float top) {
    if (p.part != nullptr) {
        float *to = p.part + o * (p.kv.d + 2) + p.kv.d;
        to[0] = top * kLn2;
        to[1] = top == -INFINITY ? l : l * fast_exp2(m - kShift - top);
    }
}

// What lanes 4 g + t hold of an 8 x 8 matrix of pairs' halves, turned round.
__device__ __forceinline__ uint32_t turned(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}

// D: head dims, or (kExact false) the next of 64, 128 and 256 above them; kWide: 32-bit activations.
// R 16: rows are the products' 16 rows, S = Q K^T and O = P V. R 8 (one query of up to 8 heads a tile): rows are their 8 columns, S^T = K Q^T and
// O^T = V^T P^T -- the two B operands of a step of K, and of two words of V, are one A operand in the same registers -- half the products, exponentials
// and accumulators, for two turns of P a block.
template <int D, bool kExact, bool kF8, bool kWide, int R>
__global__ void __launch_bounds__(Shape<D, R>::kThreads, Shape<D, R>::kCtas) attention_quant_kernel(QuantParams p) {
    using S = Shape<D, R>;
    constexpr int kScoreTiles = R / 8, kAccs = R / 4 * (D / 32), kOfRow = R / 4; // 16 tokens' scores, accumulators, scores of a row in a block: a lane's share
    constexpr int kWarps = S::kWarps, kThreads = S::kThreads, kPair = S::kPair;
    constexpr int kVecs = D / 32, kSteps = D / 16, kParts = kWide ? 2 : 1;
    constexpr bool kQueryRegs = !kWide && D <= 128;
    // Integers of 16-bit activations are multiplied as u 2^-24: scores lack 128 sum q, outputs 128 sum w, both of the rounded numbers, and
    // that is taken off in f32: 2^-23 of the largest score or value in error, which 32-bit activations do not accept.
    constexpr bool kBiased = !kF8 && !kWide;
    extern __shared__ __align__(128) unsigned char smem[];
    float *s_merge = reinterpret_cast<float *>(smem + S::kMerge), *s_m = reinterpret_cast<float *>(smem + S::kStats);
    float *s_l = s_m + kWarps * kRows, *s_top = s_l + kWarps * kRows;
    Start *s_start = reinterpret_cast<Start *>(smem + S::kWords);
    int *s_last = reinterpret_cast<int *>(smem + S::kWords + 72); // [2]
    float *s_factor = reinterpret_cast<float *>(smem + S::kWords + 96), *s_lack = s_factor + kRows; // of the tile's rows
    int *s_pos = reinterpret_cast<int *>(s_lack + kRows);
    uint32_t *s_query = reinterpret_cast<uint32_t *>(smem + S::kQuery); // [part][step][lane][4]
    const uint32_t query_u32 = smem_u32(s_query);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int d = kExact ? D : p.kv.d, vecs = d >> 5, tile_bytes = 2 * kQuantTokens * d + 16;
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
        // (launched programmatically: all but the set-up waits for the kernel in front; with overlap its index arrays are older than that kernel. The kernel
        // behind is let go only when the one in front has ended, whose results it may then count on without a wait of its own.)
        if (!p.overlap) {
            grid_dependency_wait();
            grid_launch_dependents();
        }
        int64_t *sums = reinterpret_cast<int64_t *>(s_merge);
        const int per = (p.n_seqs + kThreads - 1) / kThreads, a0 = min(tid * per, p.n_seqs), a1 = min(a0 + per, p.n_seqs);
        int64_t mine = 0;
        const int seq0 = p.seq_ids[min(a0, p.n_seqs - 1)]; // (on its way with the lengths)
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
        for (int i = 0; i < kWarps; ++i) {
            before += i < warp ? sums[i] : 0;
            line += sums[i];
        }
        piece = max((line + gridDim.x - 1) / gridDim.x, int64_t(kMinPiece));
        w.pos = min(piece * blockIdx.x, line);
        w.end = min(w.pos + piece, line);
        if (w.pos >= w.end) { // (the whole CTA)
            if (p.overlap) { // where nobody has work the launch still ends behind the kernel in front
                grid_dependency_wait();
            }
            return;
        }
        int64_t begin = before + upto - mine;
        if (begin <= w.pos && w.pos < begin + mine) {
            for (int a = a0; a < a1; ++a) {
                const SeqGeom g = seq_geom(p, a);
                const int64_t n = units_before(p, g, g.tiles) * p.kv.nkvh;
                if (w.pos < begin + n) {
                    *s_start = Start{begin, a, a == a0 ? seq0 : p.seq_ids[a], g};
                    break;
                }
                begin += n;
            }
        }
        __syncthreads();
        w.a = s_start->a;
        w.g = s_start->g;
        const int64_t x = w.pos - s_start->begin;
        int lo = 0, hi = w.g.tiles - 1; // last row tile whose first unit is not behind x
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (units_before(p, w.g, mid) * p.kv.nkvh <= x) {
                lo = mid;
            } else {
                hi = mid - 1;
            }
        }
        w.tile = lo;
        w.blocks = tile_blocks(p, w.g, lo, w.gap);
        const int64_t in_front = units_before(p, w.g, lo) * p.kv.nkvh;
        w.kvh = int((x - in_front) / (w.blocks + kTileUnits));
        w.first = s_start->begin + in_front + int64_t(w.kvh) * (w.blocks + kTileUnits);
    }
    Place &place = *reinterpret_cast<Place *>(smem + S::kPlaces + warp * kPlaceBytes);
    Feed feed;
    uint32_t n = 0;                // pairs of this CTA's fragments so far: the warps take them in turn
    uint32_t asked = 0, taken = 0; // blocks of this warp: block c lies in slot c % kSlots
    Fragment *s_pending = reinterpret_cast<Fragment *>(smem + S::kPending);
    int pending = 0;
    uint32_t found = 0;            // bit s: the page of the block in slot s exists
    bool dead = false;             // a wait ran out
    bool more, fed_ahead = false;  // whether there is a fragment ahead, and whether the feed is its
    int k_feed = 0;                // blocks of the feed that were asked for
    const int g = lane >> 2, t = lane & 3;
    // this lane's two rows, and which of the two element c of a product is in
    auto row_at = [&](int h) { return R == 16 ? g + 8 * h : 2 * t + h; };
    auto row_of = [](int c) { return R == 16 ? c >> 1 : c & 1; };
    // over the lanes that share their rows
    auto most_of = [](float x) {
#pragma unroll
        for (int o = R == 16 ? 1 : 4; o < (R == 16 ? 4 : 32); o <<= 1) {
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
        }
        return x;
    };
    auto sum_of = [](float x) {
#pragma unroll
        for (int o = R == 16 ? 1 : 4; o < (R == 16 ? 4 : 32); o <<= 1) {
            x += __shfl_xor_sync(0xffffffffu, x, o);
        }
        return x;
    };
    const int my_row = tid / S::kRowThreads, my_part = tid % S::kRowThreads; // the row of a tile that this thread loads and stores a share of
    unsigned char *s_raw = smem + S::kRaw;
    // steps to the next fragment and leaves it, with its feed, in the warp's place; its queries are on their way
    auto step = [&]() {
        Fragment ahead;
        const bool is = next_fragment(p, w, ahead);
        if (is) {
            constexpr int kElem = kWide ? 4 : 2;
            if (my_row < ahead.rows) {
                const int packed = ahead.row0 + my_row, query = packed / p.group, head = ahead.kvh * p.group + packed - query * p.group;
                const unsigned char *from = static_cast<const unsigned char *>(p.q) + (int64_t(ahead.q_start + query) * p.nh + head) * d * kElem;
                for (int at = 16 * my_part; at < d * kElem; at += 16 * S::kRowThreads) {
                    cp_async_16(smem_u32(s_raw) + my_row * D * kElem + at, from + at, 16);
                }
            }
            cp_async_commit();
            const Feed next = open_feed<S>(p, ahead, ahead.a == s_start->a ? s_start->seq : p.seq_ids[ahead.a], kPair * int((uint32_t(warp) - n) & (kWarps - 1u)), lane);
            place.now[lane] = next.now;
            place.next[lane] = next.next;
            if (lane == 0) {
                place.walker = w;
                place.ahead = ahead;
                place.feed = next;
            }
        }
        __syncwarp();
        return is;
    };
    // asks for blocks as far as there are slots
    auto ask = [&]() {
        while (asked - taken < uint32_t(S::kSlots) && !dead) {
            if (k_feed >= feed.count) {
                if (fed_ahead || !more) {
                    break;
                }
                feed = place.feed;
                feed.now = place.now[lane];
                feed.next = place.next[lane];
                fed_ahead = true;
                k_feed = 0;
                continue;
            }
            const int where = __shfl_sync(0xffffffffu, feed.now, k_feed & 31);
            const uint32_t slot = asked % S::kSlots;
            found = where >= 0 ? found | (1u << slot) : found & ~(1u << slot);
            if (lane == 0) {
                if (where >= 0) {
                    mbar_arrive_expect_tx(bars + 8 * slot, uint32_t(tile_bytes));
                    bulk_load(ring + slot * S::kTile, p.kv.base + int64_t(where) * tile_bytes, uint32_t(tile_bytes), bars + 8 * slot);
                } else {
                    mbar_arrive(bars + 8 * slot);
                }
            }
            ++asked;
            if ((++k_feed & 31) == 0) {
                feed.now = feed.next;
                feed.next = tile_place<S>(p, feed, k_feed + 32 + lane);
            }
        }
    };
    feed.count = 0;
    if (p.overlap) {
        grid_dependency_wait();
        grid_launch_dependents();
    }
    more = step();
    __syncthreads(); // the sums' place is the queries'
    while (more) {
        const Fragment f = place.ahead;
        if (!fed_ahead) {
            feed = place.feed;
            feed.now = place.now[lane];
            feed.next = place.next[lane];
            k_feed = 0;
        }
        const int blocks = place.feed.count, block0 = place.feed.first; // of this warp
        fed_ahead = false;
        n += uint32_t(f.b1 - f.b0 + kPair - 1) / kPair;

        // ---- the tile's queries, by all threads
        const int my_packed = f.row0 + my_row, my_query = my_packed / p.group, my_head = f.kvh * p.group + my_packed - my_query * p.group;
        const int64_t my_o = int64_t(f.q_start + my_query) * p.nh + my_head; // (query, head) as a row of out
        {
            more = false;
            ask(); // (none of the fragment behind this one)
            cp_async_wait<0>();
            __syncthreads();
            constexpr int kPieces = D / S::kStep;
            float4 x[kPieces];
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int dim = 4 * my_part + S::kStep * i;
                x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (my_row < f.rows && dim < d) {
                    x[i] = load4<kWide>(s_raw, my_row * D + dim, p.bf16);
                }
                most = fmaxf(most, fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))));
            }
#pragma unroll
            for (int o = S::kRowThreads / 2; o > 0; o >>= 1) {
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            }
            const int e = max(-100, min(127, (__float_as_int(most) >> 23) - 127));
            const float up = power_of_two(14 - e);
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int dim = 4 * my_part + S::kStep * i;
                const float4 y = make_float4(x[i].x * up, x[i].y * up, x[i].z * up, x[i].w * up);
                const uint32_t lo = pack_half2(y.x, y.y), hi = pack_half2(y.z, y.w);
                const float2 a = rest_of(lo, y.x, y.y), b = rest_of(hi, y.z, y.w);
                constexpr int kWords = R / 4; // of a lane and step
                uint32_t *to = s_query + ((dim >> 4) * 32 + 4 * (my_row & 7) + ((dim >> 2) & 3)) * kWords + (my_row >> 3);
                to[0] = lo;
                to[kWords / 2] = hi;
                if constexpr (kWide) {
                    to[kSteps * 32 * kWords] = pack_half2(a.x, a.y);
                    to[kSteps * 32 * kWords + kWords / 2] = pack_half2(b.x, b.y);
                }
                if constexpr (kBiased) {
                    sum += (y.x - a.x) + (y.y - a.y) + (y.z - b.x) + (y.w - b.y);
                }
            }
            const float factor = power_of_two(max(e - 14, -126)) * p.scale_log2;
            if constexpr (kBiased) {
#pragma unroll
                for (int o = S::kRowThreads / 2; o > 0; o >>= 1) {
                    sum += __shfl_xor_sync(0xffffffffu, sum, o);
                }
            }
            if (my_part == 0) {
                s_factor[my_row] = factor;
                s_lack[my_row] = 128.f * sum; // (times the factor it need not be a number where the scores are)
                s_pos[my_row] = min(my_packed, f.row0 + f.rows - 1) / p.group + f.off;
            }
        }
        __syncthreads();
        float factor[2], lack[2];
        int pos[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            factor[h] = s_factor[row_at(h)];
            lack[h] = s_lack[row_at(h)];
            pos[h] = s_pos[row_at(h)];
        }
        // blocks that all of the tile's rows see all of
        const int whole_to = min(s_pos[0], f.tokens - 1) - (kQuantTokens - 1);
        const int whole_from = p.window > 0 ? s_pos[R - 1] - p.window + 1 : 0;
        auto load_query = [&](int step, uint32_t (&to)[R / 4]) {
            if constexpr (R == 16) {
                const uint4 x = lds128(query_u32 + 16 * (step * 32 + lane));
                to[0] = x.x, to[1] = x.y, to[2] = x.z, to[3] = x.w;
            } else {
                asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];\n" : "=r"(to[0]), "=r"(to[1]) : "r"(query_u32 + 8 * (step * 32 + lane)));
            }
        };
        uint32_t qf[kQueryRegs ? kSteps : 1][R / 4];
        if constexpr (kQueryRegs) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                load_query(i, qf[i]);
            }
        }
        w = place.walker;
        __syncwarp();
        more = step();

        // ---- its blocks
        float acc[kAccs][4]; // R 16: dims 8 i + 2 t and + 1 of row g, of row g + 8; R 8: dim 16 i + g of rows 2 t and + 1, dim 16 i + 8 + g
#pragma unroll
        for (int i = 0; i < kAccs; ++i) {
            acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
        }
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, top[2] = {-INFINITY, -INFINITY}, weights[4] = {};
        for (int i = 0; i < blocks && !dead; i += kPair) {
            float s[kPair][kScoreTiles][4], mantissa[kPair], down[kPair], fe[kPair];
            uint32_t slot[kPair]; // (the block behind the last one is the last one again, with nothing seen of it: no branch between the two)
            bool live[kPair];
#pragma unroll
            for (int b = 0; b < kPair; ++b) {
                live[b] = i + b < blocks;
                slot[b] = (taken + (live[b] ? b : 0)) % S::kSlots;
                dead = dead || !mbar_wait_bounded(bars + 8 * slot[b], ((taken + (live[b] ? b : 0)) / S::kSlots) & 1, p.kv.wait_limit);
            }
            if (__any_sync(0xffffffffu, dead)) {
                dead = true;
                // what else is on its way lands before the CTA ends
                for (uint32_t c = taken; c != asked; ++c) {
                    mbar_wait_bounded(bars + 8 * (c % S::kSlots), (c / S::kSlots) & 1, kDrainLimit);
                }
                if (lane == 0) {
                    atomicOr(p.error_flag, kErrTimeout);
                }
                break;
            }
            bool whole = true;
            int token0[kPair];
#pragma unroll
            for (int b = 0; b < kPair; ++b) {
                int block = block0 + i * kWarps + b;
                block = block < f.kept ? block : block + f.gap;
                token0[b] = block * kQuantTokens;
                if ((found >> slot[b] & 1) == 0) { // no page: nothing seen of it, and nothing odd in its place
                    live[b] = false;
                    for (int at = 16 * lane; at < tile_bytes; at += 512) {
                        *reinterpret_cast<uint4 *>(my_ring + slot[b] * S::kTile + at) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem(); // before the slot's next copy
                    __syncwarp();
                }
                whole = whole && live[b] && token0[b] <= whole_to && (token0[b] >= whole_from || token0[b] + kQuantTokens <= p.keep_first);
            }
#pragma unroll
            for (int b = 0; b < kPair; ++b) {
#pragma unroll
                for (int j = 0; j < kScoreTiles; ++j) {
                    s[b][j][0] = s[b][j][1] = s[b][j][2] = s[b][j][3] = 0.f;
                }
            }
#pragma unroll
            for (int v = 0; v < kVecs; ++v) {
                if (v < vecs) {
                    uint32_t u[kPair][4];
#pragma unroll
                    for (int b = 0; b < kPair; ++b) {
                        const uint4 words = lds128(ring + slot[b] * S::kTile + 16 * (32 * v + lane));
                        u[b][0] = words.x, u[b][1] = words.y, u[b][2] = words.z, u[b][3] = words.w;
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        uint32_t q[kParts][R / 4];
#pragma unroll
                        for (int part = 0; part < kParts; ++part) {
                            if constexpr (kQueryRegs) {
#pragma unroll
                                for (int k = 0; k < R / 4; ++k) {
                                    q[part][k] = qf[2 * v + j][k];
                                }
                            } else {
                                load_query(part * kSteps + 2 * v + j, q[part]);
                            }
                        }
#pragma unroll
                        for (int b = 0; b < kPair; ++b) {
                            uint32_t lo[2], hi[2];
                            widen<kF8, kBiased>(u[b][2 * j], lo[0], hi[0]);
                            widen<kF8, kBiased>(u[b][2 * j + 1], lo[1], hi[1]);
                            if constexpr (R == 8) {
                                const uint32_t tokens[4] = {lo[0], lo[1], hi[0], hi[1]};
                                if constexpr (kWide) {
                                    float x[4];
                                    mma_zero(x, tokens, q[1][0], q[1][1]);
                                    mma_16816<false>(x, tokens, q[0][0], q[0][1]);
#pragma unroll
                                    for (int c = 0; c < 4; ++c) {
                                        s[b][0][c] += x[c];
                                    }
                                } else {
                                    mma_16816<false>(s[b][0], tokens, q[0][0], q[0][1]);
                                }
                            } else if constexpr (kWide) { // (the tensor cores cut their sums: short ones, added up with rounding)
                                float x[2][4];
#pragma unroll
                                for (int tile = 0; tile < 2; ++tile) {
                                    mma_zero(x[tile], q[1], lo[tile], hi[tile]);
                                    mma_16816<false>(x[tile], q[0], lo[tile], hi[tile]);
#pragma unroll
                                    for (int c = 0; c < 4; ++c) {
                                        s[b][tile][c] += x[tile][c];
                                    }
                                }
                            } else {
                                mma_16816<false>(s[b][0], q[0], lo[0], hi[0]);
                                mma_16816<false>(s[b][1], q[0], lo[1], hi[1]);
                            }
                        }
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < kPair; ++b) { // scores in log2 units
                const float2 scales = *reinterpret_cast<const float2 *>(my_ring + slot[b] * S::kTile + quant_scales_at(d));
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float unit = factor[h] * scales.x, by = unit * (kBiased ? 0x1p24f : 1.f), less = kBiased ? -lack[h] * unit : 0.f;
#pragma unroll
                    for (int k = 0; k < kOfRow; ++k) {
                        float &x = R == 16 ? s[b][k >> 1][2 * h + (k & 1)] : s[b][0][2 * k + h];
                        x = fmaf(x, by, less);
                    }
                }
                const int e = max(kLeastPower, min(126, ((__float_as_int(scales.y) >> 23) & 255) - 127));
                fe[b] = float(e);
                down[b] = power_of_two(-e);
                mantissa[b] = scales.y * down[b];
            }
            if (!whole) {
#pragma unroll
                for (int b = 0; b < kPair; ++b) {
#pragma unroll
                    for (int j = 0; j < kScoreTiles; ++j) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const int token = token0[b] + (R == 16 ? 4 * t + 2 * j + (c & 1) : 4 * (g >> 1) + 2 * (c >> 1) + (g & 1)), at = pos[row_of(c)];
                            const bool seen = live[b] && token <= at && token < f.tokens && (p.window == 0 || at - token < p.window || token < p.keep_first);
                            s[b][j][c] = seen ? s[b][j][c] : -INFINITY;
                        }
                    }
                }
            }
            uint32_t pf[kPair][kParts][R / 4];
            float alpha[2], x[kPair][2][kOfRow]; // weights of the lane's two rows
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float most = -INFINITY;
#pragma unroll
                for (int b = 0; b < kPair; ++b) {
#pragma unroll
                    for (int k = 0; k < kOfRow; ++k) {
                        x[b][h][k] = R == 16 ? s[b][k >> 1][2 * h + (k & 1)] : s[b][0][2 * k + h];
                    }
                    float here = fmaxf(x[b][h][0], x[b][h][1]);
                    if constexpr (R == 16) {
                        here = fmaxf(here, fmaxf(x[b][h][2], x[b][h][3]));
                    }
                    top[h] = fmaxf(top[h], here);
                    most = fmaxf(most, here + fe[b]);
                }
                most = most_of(most);
                const float m_new = fmaxf(m[h], most), base = m_new == -INFINITY ? 0.f : m_new - kShift;
                alpha[h] = m_new == -INFINITY ? 1.f : fast_exp2(m[h] - m_new);
                m[h] = m_new;
                l[h] *= alpha[h];
#pragma unroll
                for (int b = 0; b < kPair; ++b) {
                    const float from = base - fe[b];
                    float sum = 0.f;
#pragma unroll
                    for (int k = 0; k < kOfRow; ++k) {
                        const float score = x[b][h][k];
                        x[b][h][k] = fast_exp2(score - from);
                        sum += x[b][h][k];
                        x[b][h][k] *= mantissa[b];
                        if (!whole) { // a lost block's NaN stays where it is seen
                            x[b][h][k] = score == -INFINITY ? 0.f : x[b][h][k];
                        }
                    }
                    l[h] = fmaf(sum, down[b], l[h]);
                }
            }
#pragma unroll
            for (int b = 0; b < kPair; ++b) {
#pragma unroll
                for (int k = 0; k < R / 4; ++k) { // two tokens of a row, or (8 rows) a token of two rows, turned round to two tokens of a row
                    const float from = R == 16 ? x[b][k & 1][k & 2] : x[b][0][k], to = R == 16 ? x[b][k & 1][(k & 2) + 1] : x[b][1][k];
                    const uint32_t w = pack_half2(from, to);
                    pf[b][0][k] = R == 16 ? w : turned(w);
                    if constexpr (kWide) {
                        const float2 rest = rest_of(w, from, to);
                        const uint32_t w2 = pack_half2(rest.x, rest.y);
                        pf[b][1][k] = R == 16 ? w2 : turned(w2);
                    }
                }
            }
            if constexpr (kWide) {
                // the pair's values in sums of their own, added to the others with one rounding
#pragma unroll
                for (int v = 0; v < kVecs; ++v) {
                    if (v < vecs) {
                        uint32_t u[kPair][4];
#pragma unroll
                        for (int b = 0; b < kPair; ++b) {
                            const uint4 words = lds128(ring + slot[b] * S::kTile + kQuantTokens * d + 16 * (32 * v + lane));
                            u[b][0] = words.x, u[b][1] = words.y, u[b][2] = words.z, u[b][3] = words.w;
                        }
#pragma unroll
                        for (int j = 0; j < R / 4; ++j) {
                            float y[4];
#pragma unroll
                            for (int b = 0; b < kPair; ++b) {
                                if constexpr (R == 16) {
                                    uint32_t lo, hi;
                                    widen<kF8, kBiased>(u[b][j], lo, hi);
                                    if (b == 0) {
                                        mma_zero(y, pf[b][1], lo, hi);
                                    } else {
                                        mma_16816<false>(y, pf[b][1], lo, hi);
                                    }
                                    mma_16816<false>(y, pf[b][0], lo, hi);
                                } else {
                                    uint32_t dims[4];
                                    widen<kF8, kBiased>(u[b][2 * j], dims[0], dims[2]);
                                    widen<kF8, kBiased>(u[b][2 * j + 1], dims[1], dims[3]);
                                    if (b == 0) {
                                        mma_zero(y, dims, pf[b][1][0], pf[b][1][1]);
                                    } else {
                                        mma_16816<false>(y, dims, pf[b][1][0], pf[b][1][1]);
                                    }
                                    mma_16816<false>(y, dims, pf[b][0][0], pf[b][0][1]);
                                }
                            }
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                acc[R / 4 * v + j][c] = fmaf(acc[R / 4 * v + j][c], alpha[row_of(c)], y[c]);
                            }
                        }
                    }
                }
            } else {
                if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
                    for (int i = 0; i < kAccs; ++i) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            acc[i][c] *= alpha[row_of(c)];
                        }
                    }
                    weights[0] *= alpha[0];
                    weights[R == 16 ? 2 : 1] *= alpha[1];
                }
#pragma unroll
                for (int b = 0; b < kPair; ++b) {
                    if constexpr (kBiased) {
                        constexpr uint32_t kOnes = 0x3c003c00u, ones[4] = {kOnes, kOnes, kOnes, kOnes}; // sums of the rounded weights
                        if constexpr (R == 16) {
                            mma_16816<false>(weights, pf[b][0], kOnes, kOnes);
                        } else {
                            mma_16816<false>(weights, ones, pf[b][0][0], pf[b][0][1]);
                        }
                    }
#pragma unroll
                    for (int v = 0; v < kVecs; ++v) {
                        if (v < vecs) {
                            const uint4 words = lds128(ring + slot[b] * S::kTile + kQuantTokens * d + 16 * (32 * v + lane));
                            const uint32_t u[4] = {words.x, words.y, words.z, words.w};
#pragma unroll
                            for (int j = 0; j < R / 4; ++j) {
                                if constexpr (R == 16) {
                                    uint32_t lo, hi;
                                    widen<kF8, kBiased>(u[j], lo, hi);
                                    mma_16816<false>(acc[4 * v + j], pf[b][0], lo, hi);
                                } else {
                                    uint32_t dims[4];
                                    widen<kF8, kBiased>(u[2 * j], dims[0], dims[2]);
                                    widen<kF8, kBiased>(u[2 * j + 1], dims[1], dims[3]);
                                    mma_16816<false>(acc[2 * v + j], dims, pf[b][0][0], pf[b][0][1]);
                                }
                            }
                        }
                    }
                }
            }
            if constexpr (kBiased) {
                if ((i & (kFold - 1)) == kFold - kPair) {
#pragma unroll
                    for (int a = 0; a < kAccs; ++a) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            acc[a][c] = fmaf(-128.f * 0x1p-24f, weights[R == 16 ? c & 2 : c & 1], acc[a][c]);
                        }
                    }
                    weights[0] = weights[R == 16 ? 2 : 1] = 0.f;
                }
            }
            __syncwarp();
            taken += uint32_t(min(kPair, blocks - i));
            ask();
        }

        // ---- the warps' sums
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] = sum_of(l[h]);
            if (p.part != nullptr) {
                top[h] = most_of(top[h]);
            }
            if ((R == 16 ? t : g) == 0) {
                s_m[warp * kRows + row_at(h)] = m[h];
                s_l[warp * kRows + row_at(h)] = l[h];
                s_top[warp * kRows + row_at(h)] = top[h];
            }
        }
        __syncthreads();
        float share[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float all = -INFINITY;
#pragma unroll
            for (int i = 0; i < kWarps; ++i) {
                all = fmaxf(all, s_m[i * kRows + row_at(h)]);
            }
            share[h] = all == -INFINITY ? 1.f : fast_exp2(m[h] - all);
        }
        float m_all = -INFINITY, l_all = 0.f, top_all = -INFINITY; // of the row that this thread stores
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
            m_all = fmaxf(m_all, s_m[i * kRows + my_row]);
            top_all = fmaxf(top_all, s_top[i * kRows + my_row]);
        }
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
            l_all += s_l[i * kRows + my_row] * (m_all == -INFINITY ? 1.f : fast_exp2(s_m[i * kRows + my_row] - m_all));
        }
        const bool whole_tile = f.begins && f.ends;
        float *slot_of_mine = p.partials + (int64_t(blockIdx.x) * 2 + (f.begins ? 1 : 0)) * partial_floats(d);
        const float gate = p.row_scale != nullptr && my_row < f.rows && p.part == nullptr ? p.row_scale[my_o] : 1.f;
        const int64_t my_out = int64_t(f.q_start + my_query) * p.out_stride + int64_t(my_head) * d;
        const float by = (l_all == 0.f ? 0.f : 1.f / l_all) * gate;
#pragma unroll
        for (int c0 = 0; c0 < D; c0 += S::kMergeDims) {
            if (c0 < d) {
#pragma unroll
                for (int i = 0; i < S::kMergeDims * R / 128; ++i) {
                    float y[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        y[c] = acc[c0 * R / 128 + i][c];
                        if constexpr (kBiased) {
                            y[c] = fmaf(y[c], 0x1p24f, -128.f * weights[R == 16 ? c & 2 : c & 1]);
                        }
                        y[c] *= share[row_of(c)];
                    }
                    if constexpr (R == 16) {
                        float *at = s_merge + (warp * R + g) * S::kMergeStride + 8 * i + 2 * t;
                        *reinterpret_cast<float2 *>(at) = make_float2(y[0], y[1]);
                        *reinterpret_cast<float2 *>(at + 8 * S::kMergeStride) = make_float2(y[2], y[3]);
                    } else {
                        float *at = s_merge + (warp * R + 2 * t) * S::kMergeStride + 16 * i + g;
                        at[0] = y[0];
                        at[S::kMergeStride] = y[1];
                        at[8] = y[2];
                        at[S::kMergeStride + 8] = y[3];
                    }
                }
                __syncthreads();
#pragma unroll
                for (int i = 0; i < S::kMergeDims / S::kStep; ++i) {
                    const int dim = S::kStep * i + 4 * my_part;
                    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int k = 0; k < kWarps; ++k) {
                        const float4 x = *reinterpret_cast<const float4 *>(s_merge + (k * R + my_row) * S::kMergeStride + dim);
                        sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
                    }
                    if (c0 + dim < d) {
                        if (!whole_tile) {
                            __stcg(reinterpret_cast<float4 *>(slot_of_mine + my_row * d + c0 + dim), sum);
                        } else if (my_row < f.rows) {
                            finish<kWide>(p, my_o, my_out, c0 + dim, sum, by);
                        }
                    }
                }
                __syncthreads(); // the buffer is free again
            }
        }
        if (whole_tile) {
            if (my_part == 0 && my_row < f.rows) {
                finish_stats(p, my_o, m_all, l_all, top_all);
            }
        } else {
            if (my_part == 0) {
                float *stats = slot_of_mine + kRows * d;
                __stcg(stats + my_row, m_all);
                __stcg(stats + kRows + my_row, l_all);
                __stcg(stats + 2 * kRows + my_row, top_all);
            }
            if (tid == 0) {
                s_pending[pending] = f;
            }
            ++pending;
        }
    }

    // ---- tiles that other CTAs have parts of: whoever comes last puts the parts together, in the order of the CTAs
    const auto first_of = [&](const Fragment &f) { return int((f.first + snap_of(f.blocks)) / piece); };
    const auto last_of = [&](const Fragment &f) { return int((f.first + f.blocks - snap_of(f.blocks) - 1) / piece); };
    __syncthreads();
    if (lane == 0 && warp < pending) { // (one release for everybody's parts: the barrier made them this thread's to publish)
        const Fragment f = s_pending[warp];
        int *counter = p.counters + first_of(f), seen;
        asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;\n" : "=r"(seen) : "l"(counter) : "memory");
        const bool last = seen == last_of(f) - first_of(f);
        if (last) {
            *counter = 0;
        }
        s_last[warp] = last;
    }
    __syncthreads();
    for (int k = 0; k < pending; ++k) {
        if (!s_last[k]) {
            continue;
        }
        const Fragment f = s_pending[k];
        const int c_first = first_of(f), c_last = last_of(f);
        const int my_packed = f.row0 + my_row, my_query = my_packed / p.group, my_head = f.kvh * p.group + my_packed - my_query * p.group;
        const int64_t my_o = int64_t(f.q_start + my_query) * p.nh + my_head, my_out = int64_t(f.q_start + my_query) * p.out_stride + int64_t(my_head) * d;
        // one pass, two parts' loads at a time
        float m_tile = -INFINITY, l_tile = 0.f, top_tile = -INFINITY;
        float4 sum[D / S::kStep] = {};
        for (int c = c_first; c <= c_last; c += 2) {
            float m_part[2], l_part[2];
            float4 x[2][D / S::kStep];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                m_part[u] = -INFINITY;
                l_part[u] = 0.f;
                if (c + u <= c_last) {
                    const float *from = p.partials + (int64_t(c + u) * 2 + (c + u == c_first ? 1 : 0)) * partial_floats(d), *stats = from + kRows * d;
                    m_part[u] = __ldcg(stats + my_row);
                    l_part[u] = __ldcg(stats + kRows + my_row);
                    top_tile = fmaxf(top_tile, __ldcg(stats + 2 * kRows + my_row));
#pragma unroll
                    for (int i = 0; i < D / S::kStep; ++i) {
                        const int dim = S::kStep * i + 4 * my_part;
                        x[u][i] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (dim < d) {
                            x[u][i] = __ldcg(reinterpret_cast<const float4 *>(from + my_row * d + dim));
                        }
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if (c + u > c_last) {
                    continue;
                }
                const float m_new = fmaxf(m_tile, m_part[u]);
                const float had = m_tile == m_new ? 1.f : fast_exp2(m_tile - m_new), adds = m_part[u] == m_new ? 1.f : fast_exp2(m_part[u] - m_new);
                m_tile = m_new;
                l_tile = l_tile * had + l_part[u] * adds;
#pragma unroll
                for (int i = 0; i < D / S::kStep; ++i) {
                    sum[i].x = sum[i].x * had + x[u][i].x * adds, sum[i].y = sum[i].y * had + x[u][i].y * adds;
                    sum[i].z = sum[i].z * had + x[u][i].z * adds, sum[i].w = sum[i].w * had + x[u][i].w * adds;
                }
            }
        }
        if (my_row < f.rows) {
            const float by = (l_tile == 0.f ? 0.f : 1.f / l_tile) * (p.row_scale != nullptr && p.part == nullptr ? p.row_scale[my_o] : 1.f);
#pragma unroll
            for (int i = 0; i < D / S::kStep; ++i) {
                if (S::kStep * i + 4 * my_part < d) {
                    finish<kWide>(p, my_o, my_out, S::kStep * i + 4 * my_part, sum[i], by);
                }
            }
            if (my_part == 0) {
                finish_stats(p, my_o, m_tile, l_tile, top_tile);
            }
        }
    }
}

} // namespace

void attention_quant_scratch(int32_t d, size_t *floats, size_t *counters) {
    const size_t ctas = size_t(device_sms()) * (d <= 64 ? Shape<64, 8>::kCtas : d <= 128 ? Shape<128, 8>::kCtas : Shape<256, 8>::kCtas);
    *floats = ctas * 2 * partial_floats(d);
    *counters = ctas;
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
    p.out_wide = reinterpret_cast<uintptr_t>(out.out) % (dtype == LLAISYS_DTYPE_F32 ? 16 : 8) == 0 && p.out_stride % 4 == 0;
    p.overlap = kv.overlap_launch;
    p.partials = scratch.partials;
    p.counters = scratch.counters;
    p.error_flag = scratch.error_flag;
    CHECK_ARGUMENT(aligned16(q), "attention: queries must be 16-byte aligned");
    CHECK_ARGUMENT(int64_t(batch.total_q) * p.group <= 0x7fffffff - kRows && batch.n_seqs <= 1 << 30 &&
                       int64_t(kv.table_stride) * kv.blocks_per_page * p.group <= 1 << 30,
                   "attention: too many rows or tokens for one launch");
    size_t floats, counters;
    attention_quant_scratch(kv.d, &floats, &counters);
    CHECK_ARGUMENT(scratch.partials_floats >= floats && scratch.counters_len >= counters, "attention: workspace too small");
    auto launch = [&](auto d, auto r) {
        constexpr int D = decltype(d)::value, R = decltype(r)::value;
        auto start = [&](auto kernel) {
            const size_t bytes = Shape<D, R>::bytes(dtype == LLAISYS_DTYPE_F32);
            LLAISYS_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)));
            launch_programmatic_smem(kernel, dim3(unsigned(device_sms() * Shape<D, R>::kCtas)), unsigned(Shape<D, R>::kThreads), bytes, static_cast<cudaStream_t>(stream), p);
        };
        auto pick = [&](auto exact) {
            constexpr bool kExact = decltype(exact)::value;
            if (dtype == LLAISYS_DTYPE_F32) {
                start(kv.f8 ? attention_quant_kernel<D, kExact, true, true, R> : attention_quant_kernel<D, kExact, false, true, R>);
            } else {
                start(kv.f8 ? attention_quant_kernel<D, kExact, true, false, R> : attention_quant_kernel<D, kExact, false, false, R>);
            }
        };
        if (kv.d == D) {
            pick(std::true_type{});
        } else {
            pick(std::false_type{});
        }
    };
    // 8 rows a tile where every tile is one query of at most 8 heads (16 and 8 rows, us: 64 sequences of 4096 tokens, 12 / 2 heads of 128: 37.2 and 33.0;
    // windows of 2000 tokens of 24 sequences, 32 / 8 heads of 64 in 32 bits: 29.7 and 26.4; one of 777: 11.6 and 10.3)
    auto rows = [&](auto d) {
        if (batch.q_starts == nullptr && p.group <= 8) {
            launch(d, std::integral_constant<int, 8>{});
        } else {
            launch(d, std::integral_constant<int, 16>{});
        }
    };
    if (kv.d <= 64) {
        rows(std::integral_constant<int, 64>{});
    } else if (kv.d <= 128) {
        rows(std::integral_constant<int, 128>{});
    } else {
        rows(std::integral_constant<int, 256>{});
    }
    check_launch("attention_quant");
}

} // namespace llaisys::kernels
