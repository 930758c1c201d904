// Attention of chunks over a page pool held in 8 bits on the 5th-generation tensor cores: the chunk kernel of attention_prefill_tc.cu (its line of
// blocks, roles, tensor memory, turns and merge) with operands that four warps make of the codes.
//
// Mathematics. Codes (integers to 127, e4m3 numbers) are exact in f16 and go into the products as they are; queries are scaled by a power of two,
// row by row, to below 2^15. With the raw score S of a key whose block has the scales s_k and s_v,
//     y = S (f s_k) + log2 s_v   (f: the query's factor and the call's scale, in log2 units),   w = 2^(y - m + 7),   m = a running maximum of y,
//     out = sum w v8 / sum w / s_v
// so that one multiply-add per score brings both scales in, the f16 weights stay between 2^7 and (where m lags) 2^15 for the largest whatever the
// values' scales, and the sums of the weights are divided by s_v once per block of 16 keys.
//
// Bound: the tensor pipe (2048 clocks for 256 rows x 128 keys of 128 dims), the exponentials (2048) and, beside them, shared memory: the products read
// 192 KiB per such block and the widened operands are 64 KiB more, 2048 clocks of its 128 bytes in all. Codes come from L2 straight to registers,
// 16 bytes a lane in the order of the tile (quant_tile.cuh), a stage ahead; every word becomes 8 bytes of an operand row, K as [key][dims], V as
// [dim][keys], both K-major in the 128-byte swizzle. Lanes whose rows would meet in the same banks take their words in another order: K's odd tokens
// 16 dims apart from the even ones, V's odd dims from the second of two blocks that lie 32 keys apart.
//
// Measured, 12 / 2 heads of 128: eight chunks of 512 tokens behind up to 8192, integers, 149 us (776 TFLOP/s); a prompt of 5000, 32 / 8 heads,
// e4m3, 280 us (730); 16-bit pages take the other kernel 113 and 199. With operands that nobody widens (a probe) it is 2 and 9 us less: what bounds a block
// is the chain scores -> scale -> maximum -> exponentials -> products of a half. (Loads of codes under a condition, for tiles that may not exist: 155 us.)
//
// Roles: warps 0-3 and 4-7 softmax of the halves, 8 and 9 MMA issue, 10-13 the operands: two blocks of 16 keys each, of K, then of V, of every block of
// 128. Waits are bounded as in the other kernel; nothing asynchronous is left behind but MMAs, which the issuers see through.
#include "chunk_line.cuh"
#include "kernels.hpp"
#include "launch_utils.cuh"
#include "mma_utils.cuh"
#include "quant_tile.cuh"
#include "tcgen05_utils.cuh"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace llaisys::kernels {

namespace {

constexpr int kSoftmaxThreads = 128, kMmaWarp = 8, kWidenWarp = 10, kWidenWarps = 4, kGuideWarp = kWidenWarp + kWidenWarps, kThreads = 512;
// Registers a thread: 512 x 128 at launch, then 256 softmax threads take 200 and the other eight warps (two of them idle) keep 56. (Fourteen warps
// would be launched with 128 as well: a quarter of the SM holds four of them.)
constexpr int kSoftmaxRegs = 200, kOtherRegs = 56;
static_assert(256 * kSoftmaxRegs + 256 * kOtherRegs <= kThreads * 128, "no more than the CTA was launched with");
constexpr int kWarpsOfCta = kThreads / 32, kSchedInts = 3 * kWarpsOfCta + 8, kPlaceInts = 25;
static_assert(sizeof(Place) <= kPlaceInts * sizeof(int), "a warp's words");
constexpr int kErrTimeout = 8;
constexpr float kRescaleThreshold = 8.f; // log2 units
constexpr float kShift = 7.f;            // weights are 2^7 times what they stand for: at most 2^15 with a maximum that lags by the threshold
// A row's sum is kept as 2^-18 of itself: it has 2^15 / s_v for a token, and 2^30 tokens of the smallest scale, 2^-100 (values all zero, say), stay below 2^128.
constexpr float kSumUnit = 0x1p-18f;
constexpr int kFeedSlots = 4;            // blocks whose tiles the guide has found ahead of the operand warps
constexpr int kPlaces = 11;              // warps that keep a place on the line: all but the operand warps and the last one
constexpr int kScaleSlots = 4;           // blocks whose scales are kept: a block's slot is written again when its turn has passed twice over
constexpr float kMergeCostBlocks = 1.5f;
constexpr int kMergeCost = 5;

template <int D>
struct Shape {
    static constexpr int kStages = 5, kStageBytes = kKeys * D * 2;
    static constexpr int kKPiece = kKeys * 128, kVPiece = D * 128, kQPiece = kHalf * 128, kQBytes = kHalf * D * 2;
    static constexpr int kTmemCols = 512, kColS = 0, kColO = 2 * kKeys; // scores of half h at 128 h, accumulators behind them
    static constexpr int kPartialFloats = kHalf * D + 2 * kHalf;
    static constexpr int kBars = 2 * kStages + 14 + 2 * kFeedSlots;
    static constexpr size_t kScales = 2 * size_t(kQBytes) + kStages * size_t(kStageBytes), kFactors = kScales + kScaleSlots * kPagesPerBlock * 16;
    static constexpr size_t kBarsAt = kFactors + 2 * kRows, kSched = kBarsAt + kBars * 8 + 8;
    static constexpr size_t kFeed = kSched + (kSchedInts + kPlaces * kPlaceInts) * sizeof(int), kBytes = kFeed + kFeedSlots * kPagesPerBlock * 12;
    static_assert(kBytes <= 227 * 1024, "shared memory of an SM");
};

struct QuantChunkParams {
    static constexpr bool kQueriesMayLead = true;
    QuantView kv;
    const int32_t *seq_ids, *kv_lens, *q_starts;
    int32_t table_stride; // of the block table, in blocks of 16 tokens
    int32_t contiguous, const_q_len, const_kv_len; // (of the other kernel's line: always a pool here)
    int32_t n_seqs, total_q, nkvh, group, nh;
    uint32_t group_inverse; // ceil(2^32 / group)
    const void *q;
    void *out;
    float scale_log2;
    int32_t *error_flag;
    float *partials;   // [gridDim.x][tile begins here: 0, 1][half][kPartialFloats]
    int32_t *counters; // [gridDim.x][half], zero between launches
    int32_t window, keep_first;
    long long out_stride;
    const float *row_scale;
    int32_t bf16, out_wide;
};

// Four codes (a word) as two pairs of f16; integers lie in the pool as c + 128, and 0x6400 | u is 1024 + u.
template <bool kF8>
__device__ __forceinline__ uint2 widen(uint32_t w) {
    if constexpr (kF8) {
        const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xffffu), __NV_E4M3);
        const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3);
        return make_uint2(uint32_t(a.x) | (uint32_t(a.y) << 16), uint32_t(b.x) | (uint32_t(b.y) << 16));
    } else {
        const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&a), off), y = __hsub2(*reinterpret_cast<const __half2 *>(&b), off);
        return make_uint2(*reinterpret_cast<const uint32_t *>(&x), *reinterpret_cast<const uint32_t *>(&y));
    }
}
__device__ __forceinline__ void sts64(uint32_t addr, uint2 v) { asm volatile("st.shared.v2.u32 [%0], {%1, %2};\n" ::"r"(addr), "r"(v.x), "r"(v.y) : "memory"); }
// 8 columns of this thread's TMEM lane, raw words.
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&w)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"r"(taddr), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                 "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack_out(float a, float b, bool bf16) {
    if (bf16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    return pack_half2(a, b);
}
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }

template <int D, bool kF8, bool kWin, bool kShortWaits = false>
__global__ void __launch_bounds__(kThreads, 1) attention_quant_tc_kernel(QuantChunkParams p) {
    using S = Shape<D>;
    constexpr int kStages = S::kStages, kStageBytes = S::kStageBytes, kQBytes = S::kQBytes, kQPiece = S::kQPiece, kKPiece = S::kKPiece,
                  kVPiece = S::kVPiece, kPartialFloats = S::kPartialFloats, kColS = S::kColS, kColO = S::kColO;
    enum : int {
        kBarFull = 0,                   // [kStages] operand warps (one arrival each) -> MMA: the stage is written
        kBarEmpty = kBarFull + kStages, // [kStages] softmax (one thread per half; issuer of a half without rows) -> operand warps: the stage has been read
        kBarS = kBarEmpty + kStages,    // [2] MMA (commit) -> softmax of a half: [P V of the block before, Q K^T of this one] are done
        kBarO = kBarS + 2,              // [2] MMA (commit) -> softmax: the last product of the fragment is done
        kBarTurn = kBarO + 2,           // [2] issuer of the other half -> issuer of this half: its batch is issued, the next one is yours
        kBarDrain = kBarTurn + 2,       // [2] MMA (commit) -> the issuer itself: everything it issued has finished
        kBarP = kBarDrain + 2,          // [2][2] softmax (128) -> MMA: this part of P is in tensor memory (and the accumulator rescaled)
        kBarQ = kBarP + 4,              // [2] softmax (128) -> MMA: the next fragment's Q rows are in shared memory
        kBarFound = kBarQ + 2,               // [kFeedSlots] guide -> operand warps: the tiles of a block are known
        kBarRead = kBarFound + kFeedSlots,   // [kFeedSlots] operand warps (one arrival each) -> guide: and have been read
        kNumBars = kBarRead + kFeedSlots
    };
    static_assert(kNumBars == S::kBars, "barriers");
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const uint32_t base_u32 = smem_u32(smem_raw);
    unsigned char *base = smem_raw;
    if ((base_u32 & 1023u) != 0) { // swizzled operands need the alignment that is asked for above; there is no room to round up
        if (threadIdx.x == 0) {
            atomicOr(p.error_flag, kErrTimeout);
        }
        return;
    }
    const uint32_t ring_u32 = base_u32 + 2 * kQBytes;
    float4 *s_scales = reinterpret_cast<float4 *>(base + S::kScales); // [slot][block of 16 keys]: s_k, log2 s_v, kSumUnit / s_v
    signed char *s_power = reinterpret_cast<signed char *>(base + S::kFactors); // [fragments in turn][row of the tile]: raw scores are 2^-power of what they stand for
    uint64_t *bars = reinterpret_cast<uint64_t *>(base + S::kBarsAt);
    const uint32_t bars_u32 = smem_u32(bars);
    uint32_t *s_tmem_base = reinterpret_cast<uint32_t *>(bars + kNumBars);
    volatile int *s_abort = reinterpret_cast<volatile int *>(s_tmem_base + 1);
    int *s_sched = reinterpret_cast<int *>(base + S::kSched); // [kSchedInts]

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int kWarps = kThreads / 32;

    // ---- this CTA's piece of the line ----------------------------------------------------------------------------
    // (every CTA sums the sequences' units itself: a few loads per sequence, no launch in front of this one)
    int line_units = 0, longest_tile = 0, tiles = 0;
    {
        int mine = 0, mine_max = 0, mine_tiles = 0;
        for (int a = tid; a < p.n_seqs; a += kThreads) {
            const SeqGeom g = seq_geom(p, a);
            mine += seq_units(p, g, false);
            mine_tiles += seq_units(p, g, true);
            // (with a window: what a tile can reach, it only sizes the pieces)
            const int reach = g.window > 0 ? (g.window + kRows / g.group + kKeys) / kKeys + 1 + g.kept_blocks : 1 << 30;
            mine_max = max(mine_max, g.n_qb > 0 ? min((g.kv_len + kKeys - 1) / kKeys, reach) : 0);
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            mine += __shfl_xor_sync(0xffffffffu, mine, d);
            mine_max = max(mine_max, __shfl_xor_sync(0xffffffffu, mine_max, d));
            mine_tiles += __shfl_xor_sync(0xffffffffu, mine_tiles, d);
        }
        if (lane == 0) {
            s_sched[warp] = mine;
            s_sched[kWarps + warp] = mine_max;
            s_sched[2 * kWarps + warp] = mine_tiles;
        }
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) {
            line_units += s_sched[w];
            longest_tile = max(longest_tile, s_sched[kWarps + w]);
            tiles += s_sched[2 * kWarps + w];
        }
    }
    const int n_slots = int(gridDim.x);
    const int min_piece = int(ceilf(sqrtf(kMergeCostBlocks * float(longest_tile))));
    int piece = max((line_units + n_slots - 1) / n_slots, max(min_piece, kTileCost + 1)); // units per CTA
    // A cut costs its second CTA what a tile costs, and the merge: where no CTA has more to do with whole tiles alone, there are no cuts.
    // (24 chunks of 100 tokens behind 200, 12 / 2 heads, are 144 tiles of three blocks: cut into equal pieces nearly every CTA had parts of two
    // tiles, 35 us a layer; whole 22.)
    const int tiles_each = (tiles + n_slots - 1) / n_slots;
    const bool whole = (long long)tiles_each * (longest_tile + kTileCost) <= piece + kTileCost + kMergeCost;
    if (whole) {
        piece = tiles_each;
        line_units = tiles;
    }
    const int slot = int(blockIdx.x);
    const int piece_begin = slot * piece;
    if (piece_begin >= line_units) {
        return; // uniform over the CTA, before any mbarrier or TMEM allocation
    }
    const int piece_end = min(line_units, piece_begin + piece);
    volatile int *s_line = s_sched + 3 * kWarps + 4; // units per piece, end of this one (kept there for the same reason as a warp's place)
    if (tid == 0) {
        s_line[0] = piece;
        s_line[1] = piece_end;
    }
    {
        // the sequence that holds unit piece_begin, by a block-wide scan over kThreads sequences at a time
        __syncthreads();
        int before = 0; // units of the sequences in front of this pass's
        for (int a0 = 0; a0 < p.n_seqs; a0 += kThreads) {
            const int a = a0 + tid;
            const int w_a = a < p.n_seqs ? seq_units(p, seq_geom(p, a), whole) : 0;
            int incl = w_a;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, incl, d);
                incl += lane >= d ? up : 0;
            }
            if (lane == 31) {
                s_sched[warp] = incl;
            }
            __syncthreads();
            int warps_before = 0, round_total = 0;
            for (int w = 0; w < kWarps; ++w) {
                warps_before += w < warp ? s_sched[w] : 0;
                round_total += s_sched[w];
            }
            const int excl = before + warps_before + incl - w_a;
            if (w_a > 0 && excl <= piece_begin && piece_begin < excl + w_a) {
                s_sched[3 * kWarps] = a;
                s_sched[3 * kWarps + 1] = excl;
            }
            before += round_total;
            __syncthreads();
            if (before > piece_begin) {
                break;
            }
        }
    }
    Walker walker;
    walker.a = s_sched[3 * kWarps];
    walker.seq_begin = s_sched[3 * kWarps + 1];
    walker.g = seq_geom(p, walker.a);
    walker.whole = whole;
    walker.n_units = seq_units(p, walker.g, whole);
    {
        // the last row block that starts at or before the piece: by bisection, a long chunk has hundreds
        int lo = 0, hi = walker.g.n_qb - 1;
        const int at = piece_begin - walker.seq_begin;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (units_before(walker.g, mid, whole) * p.nkvh <= at) {
                lo = mid;
            } else {
                hi = mid - 1;
            }
        }
        walker.qb = lo;
        walker.qb_begin = units_before(walker.g, lo, whole) * p.nkvh;
    }
    {
        Walker first = walker;
        Fragment f;
        int pos0 = piece_begin;
        if (!locate(p, first, pos0, piece_end, f)) {
            return; // the piece holds no block (the line's last units): uniform over the CTA, nothing set up yet
        }
    }

    // ---- set-up: barriers, TMEM ----------------------------------------------------------------------------------
    if (tid == 0) {
        for (int i = 0; i < kNumBars; ++i) {
            mbar_init(bars_u32 + i * 8, i >= kBarRead || i < kBarEmpty ? kWidenWarps : i >= kBarFound ? 1 : i >= kBarP ? kSoftmaxThreads : i < kBarS ? 2 : 1);
        }
        *s_abort = 0;
        mbar_init_fence();
    }
    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32(s_tmem_base), S::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *s_tmem_base;

    auto bar = [&](int which) { return bars_u32 + uint32_t(which) * 8; };
    // False when the wait ran out here or somewhere else in the CTA (lanes may disagree on that); raises the flag that ends the others.
    auto wait = [&](int which, uint32_t parity) {
        const bool ok = wait_or_abort(bar(which), parity & 1u, s_abort, kShortWaits ? p.kv.wait_limit : kMbarWaitLimit);
        if (!ok) {
            *s_abort = 1;
        }
        return ok;
    };
    // For what is on its way in any case: not cut short by another warp's failure.
    auto drain = [&](int which, uint32_t parity) {
        if (!mbar_wait_bounded(bar(which), parity & 1u, kMbarWaitLimit)) {
            *s_abort = 1;
        }
        __syncwarp();
    };
    // A warp's place on the line waits in shared memory while its blocks run: a register that is spilled there is fetched from L2 (the
    // operands leave no L1), and a dozen such loads per block cost as much as the block.
    Place *place = reinterpret_cast<Place *>(s_sched + kSchedInts + min(warp < kWidenWarp ? warp : warp - kWidenWarps, kPlaces - 1) * kPlaceInts);
    auto keep_place = [&](const Walker &w, const Fragment &f, int pos) {
        __syncwarp();
        if (lane == 0) {
            place->w = w;
            place->f = f;
            place->pos = pos;
        }
        __syncwarp();
    };
    if (warp < kWidenWarp || warp == kGuideWarp) {
        keep_place(walker, Fragment{}, piece_begin);
    }
    // The next fragment of the piece, in this warp's place.
    auto next_fragment = [&](Walker &w, Fragment &f) {
        int pos = place->pos;
        w = place->w;
        const bool found = locate(p, w, pos, s_line[1], f);
        keep_place(w, f, pos + (found ? f.units : 0));
        return found;
    };

    // (setmaxnreg inside each branch: where they met again the compiler would keep to the smaller count)
    if (warp >= kMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kOtherRegs));
        // What the guide tells the operand warps of a block of 16 keys: its tile's place in the pool (kNone: there is none, kEnd: no more blocks) and scales.
        struct Found {
            int place;
            float s_k, s_v;
        };
        constexpr int kNone = -1, kEnd = -2;
        Found *s_feed = reinterpret_cast<Found *>(base + S::kFeed); // [kFeedSlots][kPagesPerBlock]
        if (warp == kGuideWarp) {
            // ================================ guide: where the blocks' tiles are =====================================
            // Pages come 4 blocks (32 blocks of 16 keys, a lane each) at a time, the group behind a group early. Behind a tile's last block its last
            // block comes again: hidden keys have weight 0, and what they are multiplied by is then always of this sequence.
            constexpr int kGroup = 32 / kPagesPerBlock;
            uint32_t told = 0; // blocks
            auto tell = [&](const Found &found, int from) { // lanes from, ..., from + 7
                const int at = told % kFeedSlots;
                if (told >= kFeedSlots && !__all_sync(0xffffffffu, wait(kBarRead + at, told / kFeedSlots - 1))) {
                    return false;
                }
                if (lane >= from && lane < from + kPagesPerBlock) {
                    s_feed[at * kPagesPerBlock + lane - from] = found;
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(bar(kBarFound + at));
                }
                ++told;
                return true;
            };
            bool alive = true;
            while (alive) {
                Fragment f;
                Walker w;
                if (!next_fragment(w, f)) {
                    break;
                }
                const int n = f.b1 - f.b0, seq = p.seq_ids[f.a];
                const int last = (min(tile_kv_hi(w.g, f.qb), min(max(p.kv_lens[f.a], 0), p.table_stride * kPage)) + kPage - 1) / kPage - 1;
                const bool known = seq >= 0 && seq < p.kv.table_rows;
                if (!known && last >= 0) {
                    atomicOr(p.error_flag, kErrBadSeq);
                }
                const int32_t *table = p.kv.block_table + (long long)(known ? seq : 0) * p.kv.table_stride;
                auto find = [&](int blk0) {
                    const int b = blk0 + lane / kPagesPerBlock;
                    const int at = min((kWin && b >= w.g.kept_blocks ? b + f.gap : b) * kPagesPerBlock + lane % kPagesPerBlock, last);
                    // (what is loaded lies in the table and in the pool whatever comes of it: where there is no token, no sequence or no page, page 0's)
                    const int in_table = max(at, 0), entry = p.kv.blocks_per_page == 1 ? in_table : in_table / p.kv.blocks_per_page, page = table[entry];
                    const bool named = at >= 0 && known, there = named && page >= 0 && page < p.kv.num_pages;
                    const int place = ((there ? page : 0) * p.kv.blocks_per_page + in_table - entry * p.kv.blocks_per_page) * p.kv.nkvh + f.kvh;
                    const float2 scales = __ldcg(reinterpret_cast<const float2 *>(p.kv.base + (long long)place * p.kv.tile_bytes + quant_scales_at(D)));
                    if (named && !there) {
                        atomicOr(p.error_flag, kErrBadPage);
                    }
                    return there ? Found{place, scales.x, scales.y} : Found{kNone, 0.f, 0.f};
                };
                Found group = find(f.b0), next_group = find(f.b0 + kGroup);
                for (int i = 0; i < n && alive; ++i) {
                    if (i > 0 && i % kGroup == 0) {
                        group = next_group;
                        next_group = find(f.b0 + i + kGroup);
                    }
                    alive = tell(group, i % kGroup * kPagesPerBlock);
                }
            }
            if (alive) {
                tell(Found{kEnd, 0.f, 0.f}, 0);
            }
        } else if (warp > kGuideWarp) {
            // (idle)
        } else if (warp >= kWidenWarp) {
            // ================================ operands: codes to f16 =================================================
            constexpr int kVecs = D / 32;
            const int ww = warp - kWidenWarp, block_a = (ww >> 1) * 4 + (ww & 1); // this warp's blocks of 16 keys: block_a and block_a + 2
            const int g = lane >> 2, t = lane & 3, odd = g & 1;
            const int tile_bytes = p.kv.tile_bytes;
            // Where a lane's words go, from the start of a stage. K, word j of vector v: token 4 (g / 2) + 2 (j & 1) + odd, dims 32 v + 16 ((j >> 1) ^ odd) + 4 t.
            const uint32_t k_at = uint32_t((block_a * kPage + 4 * (g >> 1) + odd) * 128 +
                                           ((((odd << 1) | (t >> 1)) ^ ((((g >> 1) & 1) << 2) | odd)) << 4) + (t & 1) * 8);
            // V, word k of vector v of the block `other` (0: a, 1: the one 32 keys on): dim 32 v + 8 k + g, tokens 4 t; lanes of odd g begin with the other block
            const uint32_t v_at = uint32_t((block_a >> 2) * kVPiece + g * 128 + (((((block_a & 3) << 1) | (t >> 1)) ^ (odd << 2) ^ g) << 4) + (t & 1) * 8);
            // The registers of these warps hold one UNIT of codes, 16 words a lane: K of one block of 16 keys, or the low or high half of the dims of V of
            // both. As soon as a word is read its register is asked to bring the next unit's. (Two units would be a stage, and spill: what is spilled
            // here comes back from L2, the operands leave no L1.)
            int tiles[2] = {kNone, kNone}; // places of the two tiles of the units that are asked for
            uint32_t heard = 0;            // blocks
            bool more = true, ok = true;
            auto step = [&]() { // to the next block: its tiles
                const int at = heard % kFeedSlots;
                ok = __all_sync(0xffffffffu, wait(kBarFound + at, heard / kFeedSlots)) && ok;
                tiles[0] = ok ? s_feed[at * kPagesPerBlock + block_a].place : kNone; // (where the wait ran out nobody may have written there yet)
                tiles[1] = ok ? s_feed[at * kPagesPerBlock + block_a + 2].place : kNone;
                more = ok && tiles[0] != kEnd;
            };
            constexpr int kHalfVecs = kVecs / 2; // 16-byte loads of a unit of V from either tile
            uint4 raw[2 * kHalfVecs];
            // Where the next unit's words come from: the low half of `raw` from one place on, the high half from another. Where there is no tile the pool's
            // first one stands in: codes are numbers, and whoever they are multiplied with has the weight 0 (and, behind the last block, nobody asks).
            const uint4 *from[2];
            auto tile_of = [&](int b) { return reinterpret_cast<const uint4 *>(p.kv.base + (long long)max(tiles[b], 0) * tile_bytes) + lane; };
            auto point_k = [&](int b) {
                from[0] = tile_of(b);
                from[1] = from[0] + 32 * kHalfVecs;
            };
            auto point_v = [&](int half) {
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    from[b] = tile_of(b) + kQuantTokens * D / 16 + 32 * kHalfVecs * half;
                }
            };
            auto fetch = [&](int k) { raw[k] = __ldcg(from[k / kHalfVecs] + 32 * (k % kHalfVecs)); };
            int stage = 0;
            uint32_t turn = 0;
            auto take_stage = [&]() {
                if (turn > 0) {
                    ok = __all_sync(0xffffffffu, wait(kBarEmpty + stage, turn - 1)) && ok;
                }
                return ring_u32 + stage * kStageBytes;
            };
            auto give_stage = [&]() {
                fence_proxy_async_smem(); // read by the MMAs
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(bar(kBarFull + stage));
                }
                if (++stage == kStages) {
                    stage = 0;
                    ++turn;
                }
            };
            // K of a block, vector v
            auto put_k = [&](uint32_t to, int v, const uint4 &x) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t u = j == 0 ? (odd ? x.z : x.x) : j == 1 ? (odd ? x.w : x.y) : j == 2 ? (odd ? x.x : x.z) : (odd ? x.y : x.w);
                    // (bits 4 to 6 of a row's place are swizzled: 32 dims are bit 6, 16 dims bit 5, two tokens bit 5 and a row of 256 bytes on)
                    sts64(to + (v >> 1) * kKPiece + (j & 1) * 256 + (k_at ^ uint32_t(((v & 1) << 6) | (((j >> 1) ^ (j & 1)) << 5))),
                          widen<kF8>(u));
                }
            };
            step();
            point_k(0);
#pragma unroll
            for (int v = 0; v < kVecs; ++v) {
                fetch(v);
            }
            while (more && ok) {
                // ---- K of the block
                uint32_t to = take_stage();
                if (!ok) {
                    break;
                }
                if (lane < 2) {
                    const int b = heard % kFeedSlots * kPagesPerBlock + block_a + 2 * lane;
                    // (a block never written to has no scale; the NaN of a lost one is in the logarithm, and so in the weights of whoever sees it, and not in
                    // what the sums of all others are multiplied by; what has no page is hidden)
                    const float s_v = s_feed[b].s_v < kQuantFloor ? kQuantFloor : s_feed[b].s_v;
                    s_scales[heard % kScaleSlots * kPagesPerBlock + block_a + 2 * lane] =
                        make_float4(s_feed[b].s_k, s_feed[b].place < 0 ? -INFINITY : fast_log2(s_v), isnan(s_v) ? 0.f : kSumUnit / s_v, 0.f);
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(bar(kBarRead + heard % kFeedSlots));
                }
                ++heard;
#pragma unroll 1
                for (int b = 0; b < 2; ++b) { // (the code of these warps shares the SM's instruction cache with the softmax: units in loops)
                    if (b == 0) {
                        point_k(1);
                    } else {
                        point_v(0);
                    }
#pragma unroll
                    for (int v = 0; v < kVecs; ++v) {
                        put_k(to + b * 32 * 128, v, raw[v]);
                        fetch(v);
                    }
                }
                give_stage();
                // ---- V of the block
                to = take_stage();
                if (!ok) {
                    break;
                }
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    if (half == 0) {
                        point_v(1);
                    } else {
                        step(); // (V is asked for; K of the next block comes next)
                        point_k(0);
                    }
#pragma unroll
                    for (int v = 0; v < kHalfVecs; ++v) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint4 &a = raw[v], &c = raw[kHalfVecs + v];
                            const uint32_t x = j == 0 ? a.x : j == 1 ? a.y : j == 2 ? a.z : a.w, y = j == 0 ? c.x : j == 1 ? c.y : j == 2 ? c.z : c.w;
                            const uint32_t row = to + half * (32 * kHalfVecs * 128) + (32 * v + 8 * j) * 128;
                            sts64(row + v_at, widen<kF8>(odd ? y : x));
                            sts64(row + (v_at ^ 64u), widen<kF8>(odd ? x : y));
                        }
                        fetch(v);
                        fetch(kHalfVecs + v);
                    }
                }
                give_stage();
            }
        } else if (warp <= kMmaWarp + 1) {
            // ================================ MMA issuers, one warp per half ========================================
            // tcgen05.mma is accepted at the pace of the tensor pipe, a few instructions ahead: with one warp for both halves the pipe stood idle
            // through every wait, commit and loop step between batches (2100 of a block's 4200 clocks). With two, one half's batch runs under the
            // other's waits. The whole warp walks the blocks and one lane issues: descriptors then come from uniform registers.
            // A lane whose wait ran out issues nothing any more and skips its later waits, but walks on: the warp stays together without a vote per
            // wait (with one, a prompt of 8192 took 587 instead of 558 us).
            const int h = __shfl_sync(0xffffffffu, warp, 0) - kMmaWarp;
            constexpr uint32_t idesc_qk = make_idesc(false, false, kHalf, kKeys), idesc_pv = make_idesc(false, false, kHalf, D);
            const uint32_t tmem_s = __shfl_sync(0xffffffffu, tmem_base, 0) + kColS + h * kKeys, tmem_o = __shfl_sync(0xffffffffu, tmem_base, 0) + kColO + h * D;
            const uint64_t q_desc = smem_desc_sw128(base_u32 + h * kQBytes, 0, 1024), k_desc = smem_desc_sw128(ring_u32, 0, 1024),
                           v_desc = k_desc;
            const bool leader = elect_one();
            bool ok = true;
            int stage = 0;
            uint32_t turn = 0, p_turn = 0, q_turn = 0, my_turn = 0;
            // Where both halves have rows their batches alternate: left to themselves they fall into step, both softmaxes at once (and short of
            // exponentials), then both halves' MMAs (3600 clocks a block against 3050).
            bool two = false;
            auto take_turn = [&]() {
                if (two && (h == 1 || my_turn > 0)) {
                    ok = ok && wait(kBarTurn + h, h == 1 ? my_turn : my_turn - 1);
                }
                my_turn += two ? 1u : 0u;
            };
            auto take_stage = [&]() { // the next stage of the ring, once it has landed
                const int s = stage;
                ok = ok && wait(kBarFull + s, turn);
                stage = s + 1 == kStages ? 0 : s + 1;
                turn += s + 1 == kStages ? 1u : 0u;
                return s;
            };
            auto issue_qk = [&](int s) {
                const uint64_t k = k_desc + uint64_t(s * (kStageBytes >> 4));
                if (leader && ok) {
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks) {
                        umma_f16(tmem_s, q_desc + uint64_t(((ks >> 2) * kQPiece + (ks & 3) * 32) >> 4), k + uint64_t(((ks >> 2) * kKPiece + (ks & 3) * 32) >> 4),
                                 idesc_qk, ks > 0 ? 1u : 0u);
                    }
                }
            };
            auto commit = [&](int which) {
                if (leader && ok) {
                    umma_commit(bar(which));
                    if (two) {
                        mbar_arrive(bar(kBarTurn + 1 - h));
                    }
                }
                __syncwarp();
            };
            for (;;) {
                Fragment f;
                {
                    Walker w;
                    if (!next_fragment(w, f)) {
                        break;
                    }
                }
                const int n = __shfl_sync(0xffffffffu, f.b1 - f.b0, 0);
                two = __shfl_sync(0xffffffffu, f.rows, 0) > kHalf;
                if (h == 1 && !two) { // no rows: see the stages pass (every phase in order) and free them
                    for (int i = 0; i < 2 * n; ++i) {
                        const int s = take_stage();
                        if (ok && lane == 0) {
                            mbar_arrive(bar(kBarEmpty + s));
                        }
                    }
                    continue;
                }
                const int k0 = take_stage();
                ok = ok && wait(kBarQ + h, q_turn++);
                take_turn();
                issue_qk(k0);
                commit(kBarS + h);
                for (int i = 0; i < n; ++i) {
                    const bool more = i + 1 < n;
                    const int v_at = take_stage(), k_at = more ? take_stage() : 0;
                    const uint64_t v = v_desc + uint64_t(v_at * (kStageBytes >> 4));
#pragma unroll
                    for (int part = 0; part < 2; ++part) {
                        ok = ok && wait(kBarP + h * 2 + part, p_turn);
                        if (part == 0) {
                            take_turn();
                        }
                        tc_fence_after();
                        if (leader && ok) {
#pragma unroll
                            for (int k4 = 0; k4 < kPagesPerBlock / 2; ++k4) {
                                // B = 16 keys x D dims of V, K-major: 64 keys are a row of 128 bytes. A = P rows x 16 keys from tensor memory: 8 columns
                                // of packed pairs per step
                                const int kk = part * (kPagesPerBlock / 2) + k4;
                                umma_f16_ts(tmem_o, tmem_s + kk * 8, v + uint64_t(((kk >> 2) * kVPiece + (kk & 3) * 32) >> 4), idesc_pv, i > 0 || kk > 0 ? 1u : 0u);
                            }
                        }
                    }
                    ++p_turn;
                    if (more) {
                        issue_qk(k_at);
                    }
                    commit((more ? kBarS : kBarO) + h);
                }
            }
            if (leader) {
                umma_commit(bar(kBarDrain + h));
            }
            __syncwarp();
            drain(kBarDrain + h, 0);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kSoftmaxRegs));
        // ================================ softmax: one row per thread ===========================================
        const int h = warp >> 2, row = tid & (kHalf - 1); // half of the tile, TMEM lane
        const uint32_t lane_base = tmem_base + (uint32_t((warp & 3) * 32) << 16);
        const uint32_t tmem_s = lane_base + kColS + h * kKeys, tmem_o = lane_base + kColO + h * D;
        const uint32_t q_u32 = base_u32 + h * kQBytes;
        auto per_group = [&](int x) { return p.group == 1 ? x : int(__umulhi(uint32_t(x), p.group_inverse)); };
        // Q rows of this half, scaled by a power of two to below 2^15, 16 bytes per store, into the K-major 128-byte-swizzled layout; rows past the chunk
        // are zero. All loads first, then all stores: the stores are volatile asm, which no load may pass.
        int q_loads = 0;
        auto load_q = [&](const Fragment &f, const SeqGeom &g) {
            constexpr int kRowLanes = D / 8, kAtOnce = kSoftmaxThreads / kRowLanes, kIter = kHalf / kAtOnce; // lanes of a row, rows at once
            uint4 vals[kIter];
#pragma unroll
            for (int it = 0; it < kIter; ++it) {
                const int r = row / kRowLanes + it * kAtOnce, cc = row % kRowLanes, x = f.qb * kRows + h * kHalf + r, t = per_group(x);
                const uint4 had = *reinterpret_cast<const uint4 *>(static_cast<const char *>(p.q) + cc * 16 + // (rows past the chunk: its last one)
                                                                   ((long long)(g.q_start + min(t, g.q_len - 1)) * p.nh + f.kvh * p.group + (x - t * p.group)) * (D * 2));
                vals[it] = t < g.q_len ? had : make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int it = 0; it < kIter; ++it) {
                const int r = row / kRowLanes + it * kAtOnce, cc = row % kRowLanes;
                uint32_t words[4] = {vals[it].x, vals[it].y, vals[it].z, vals[it].w};
                float2 v[4];
                float most = 0.f;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    v[k] = p.bf16 ? make_float2(__uint_as_float(words[k] << 16), __uint_as_float(words[k] & 0xffff0000u))
                                  : __half22float2(*reinterpret_cast<const __half2 *>(&words[k]));
                    most = fmaxf(most, fmaxf(fabsf(v[k].x), fabsf(v[k].y)));
                }
#pragma unroll
                for (int o = kRowLanes / 2; o > 0; o >>= 1) {
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                }
                const int e = max(-100, min(127, (__float_as_int(most) >> 23) - 127));
                const float up = power_of_two(14 - e);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    words[k] = pack_half2(v[k].x * up, v[k].y * up);
                }
                if (cc == 0) {
                    s_power[(q_loads & 1) * kRows + h * kHalf + r] = static_cast<signed char>(e - 14);
                }
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};\n" ::"r"(q_u32 + (cc >> 3) * kQPiece + r * 128 + (((cc & 7) ^ (r & 7)) << 4)),
                             "r"(words[0]), "r"(words[1]), "r"(words[2]), "r"(words[3])
                             : "memory");
            }
            ++q_loads;
            fence_proxy_async_smem(); // read by the async proxy
            mbar_arrive(bar(kBarQ + h));
        };
        // A lane whose wait ran out goes on with what it finds, so that the warp stays together (without a vote per block, which took 2 % of
        // a prompt, and with one flag less in the block loop) and the named barrier and the arrival counts below see all 128 threads every
        // time. Nothing of a fragment is stored once the CTA has given up.
        uint32_t s_turn = 0, o_turn = 0;
        // stages that this half has seen read: K of block b is load 2 b of the CTA, V load 2 b + 1
        int done = 0; // blocks of earlier fragments
        auto free_stage = [&](int load) {
            if (row == 0) {
                mbar_arrive(bar(kBarEmpty + load % kStages));
            }
        };
        bool more = false;
        auto move_on = [&]() { // to the next fragment that has rows for this half: Q rows loaded
            Walker w;
            Fragment f;
            while ((more = next_fragment(w, f)) && h == 1 && f.rows <= kHalf) {
                done += f.b1 - f.b0;
            }
            if (more) {
                load_q(f, w.g);
            }
        };
        move_on();
        while (more) {
            Fragment f = place->f;
            SeqGeom g = place->w.g;
            const int n = f.b1 - f.b0;
            // (the line counts a chunk that is longer than what the sequence holds as if it held it; here its first queries see nothing)
            const int tokens = min(max(p.kv_lens[f.a], 0), p.table_stride * kPage);
            const int last_visible = per_group(f.qb * kRows + h * kHalf + row) + tokens - g.q_len; // keys j <= last_visible take part
            const int n_seen = min(last_visible + 1, tokens);
            float m_used = -INFINITY, l = 0.f;
            named_barrier_sync(1 + h, kSoftmaxThreads); // the factors of all rows are there
            const float factor = power_of_two(s_power[((q_loads - 1) & 1) * kRows + h * kHalf + row]) * p.scale_log2;
            for (int i = 0; i < n; ++i) {
                wait(kBarS + h, s_turn++);
                tc_fence_after();
                free_stage(2 * (done + i));
                if (i >= 1) {
                    free_stage(2 * (done + i) - 1);
                }
                const int j0 = (f.b0 + i + (kWin && f.b0 + i >= g.kept_blocks ? f.gap : 0)) * kKeys;
                const int n_ok = min(n_seen - j0, kKeys);                     // visible columns are [0, n_ok)
                const int n_lo = kWin ? last_visible - p.window + 1 - j0 : 0; // columns below n_lo lie before the row's window,
                const int n_kept = kWin ? p.keep_first - j0 : 0;              // those below n_kept are seen all the same
                uint32_t sr[kKeys / 32][32];
#pragma unroll
                for (int c = 0; c < kKeys / 32; ++c) {
                    tmem_ld32_nowait(tmem_s + c * 32, sr[c]);
                }
                tmem_wait_ld();
                // scores in log2 units, and what the values' scales add to them
                const float4 *block_scales = s_scales + (uint32_t(done + i) % kScaleSlots) * kPagesPerBlock;
#pragma unroll
                for (int b = 0; b < kPagesPerBlock; ++b) {
                    const float4 sc = block_scales[b];
                    const float by = factor * sc.x;
#pragma unroll
                    for (int k = 0; k < 16; k += 2) {
                        float x0, x1;
                        fma2(x0, x1, __uint_as_float(sr[b >> 1][(b & 1) * 16 + k]), __uint_as_float(sr[b >> 1][(b & 1) * 16 + k + 1]), by, sc.y);
                        sr[b >> 1][(b & 1) * 16 + k] = __float_as_uint(x0);
                        sr[b >> 1][(b & 1) * 16 + k + 1] = __float_as_uint(x1);
                    }
                }
                // Most blocks lie wholly below the diagonal: the whole warp then skips the mask (warp-uniform choice), and otherwise the 32-column
                // pieces that every row of the warp sees. Hidden scores become -inf: 2^(-inf * scale - m) = 0.
                if (!__all_sync(0xffffffffu, n_ok >= kKeys && (!kWin || n_lo <= 0 || n_kept >= kKeys))) {
                    auto below = [](int n) { return n <= 0 ? 0u : 0xffffffffu >> (32 - min(n, 32)); }; // bits 0 .. n - 1
#pragma unroll
                    for (int c = 0; c < kKeys / 32; ++c) {
                        uint32_t seen = below(n_ok - c * 32);
                        if constexpr (kWin) {
                            seen &= ~below(n_lo - c * 32) | below(n_kept - c * 32);
                        }
                        if (!__all_sync(0xffffffffu, seen == 0xffffffffu)) {
#pragma unroll
                            for (int k = 0; k < 32; ++k) {
                                sr[c][k] = (seen >> k) & 1u ? sr[c][k] : 0xff800000u;
                            }
                        }
                    }
                }
                // row maximum as four independent chains
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < kKeys / 32; ++c) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        mx4[k & 3] = max3(mx4[k & 3], __uint_as_float(sr[c][k]), __uint_as_float(sr[c][k + 16]));
                    }
                }
                const float mx = fmaxf(max3(mx4[0], mx4[1], mx4[2]), mx4[3]);
                // The running max only moves when it grew by more than 2^8: P and the row sum both use m_used, so the result is exact
                // either way, and O is rescaled rarely. (The scores' arrival says that the product of the block before is done.)
                float alpha = 1.f;
                const bool grow = mx > m_used + kRescaleThreshold;
                if (grow) {
                    alpha = fast_exp2(m_used - mx); // 0 on the fragment's first visible block
                    m_used = mx;
                }
                l *= alpha;
                if (i >= 1 && __any_sync(0xffffffffu, grow)) { // (the first product of a fragment overwrites O)
#pragma unroll 1
                    for (int c = 0; c < D / 16; ++c) { // (16 columns at a time: 32 beside the scores would spill)
                        float v[16];
                        tmem_ld16(tmem_o + c * 16, v);
                        tmem_wait_ld();
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            v[k] *= alpha;
                        }
                        tmem_st16(tmem_o + c * 16, v);
                    }
                }
                const float neg_m = m_used == -INFINITY ? 0.f : kShift - m_used;
#pragma unroll
                for (int b = 0; b < kPagesPerBlock; ++b) { // 16 keys = 8 columns of packed pairs over the scores
                    uint32_t packed[8];
                    float l0 = 0.f, l1 = 0.f;
#pragma unroll
                    for (int k = 0; k < 16; k += 2) {
                        float x0 = __uint_as_float(sr[b >> 1][(b & 1) * 16 + k]), x1 = __uint_as_float(sr[b >> 1][(b & 1) * 16 + k + 1]);
                        add2(x0, x1, neg_m, neg_m);
                        const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
                        add2(l0, l1, p0, p1);
                        packed[k >> 1] = pack_half2(p0, p1);
                    }
                    l = fmaf(l0 + l1, block_scales[b].z, l);
                    tmem_st8(tmem_s + b * 8, packed);
                    if ((b & 3) == 3) {
                        tmem_wait_st();
                        tc_fence_before();
                        mbar_arrive(bar(kBarP + h * 2 + (b >> 2)));
                    }
                }
            }
            // ---- Q rows of the next fragment: every Q K^T of this one has finished (its last scores were read above) ----------
            asm volatile("" ::: "memory");
            f = place->f;
            g = place->w.g;
            const int x = f.qb * kRows + h * kHalf + row, t = per_group(x), head = f.kvh * p.group + (x - t * p.group);
            const int last_load = 2 * (done + n) - 1; // V of the last block
            done += n;
            move_on();
            // ---- epilogue of the fragment ---------------------------------------------------------------------------
            wait(kBarO + h, o_turn++);
            tc_fence_after();
            free_stage(last_load);
            const bool dead = __any_sync(0xffffffffu, *s_abort != 0) != 0;
            const bool whole = f.b0 == 0 && f.b1 == f.tile_nblk;
            bool store_rows = whole;
            float w_own = 1.f, l_all = l, m_all = m_used;
            const int piece = s_line[0], first_slot = f.tile_begin / piece, last_slot = (f.tile_begin + f.tile_nblk - 1) / piece;
            auto part_of = [&](int s2) { // a fragment's place in the workspace: 1 for the one that begins its tile (and goes on in the next CTA)
                return p.partials + ((long long)(s2 * 2 + (s2 * piece <= f.tile_begin ? 1 : 0)) * 2 + h) * kPartialFloats;
            };
            if (!whole) {
                float *part = p.partials + ((long long)(slot * 2 + (f.b0 == 0 ? 1 : 0)) * 2 + h) * kPartialFloats;
                if (!dead) {
#pragma unroll
                    for (int c4 = 0; c4 < D / 32; ++c4) {
                        float v[32];
                        tmem_ld32(tmem_o + c4 * 32, v);
#pragma unroll
                        for (int q8 = 0; q8 < 8; ++q8) {
                            reinterpret_cast<float4 *>(part)[(c4 * 8 + q8) * kHalf + row] = make_float4(v[q8 * 4], v[q8 * 4 + 1], v[q8 * 4 + 2], v[q8 * 4 + 3]);
                        }
                    }
                    part[kHalf * D + row] = m_used;
                    part[kHalf * D + kHalf + row] = l;
                }
                named_barrier_sync(1 + h, kSoftmaxThreads);
                if (row == 0) { // (one release for all of the half's stores: the barrier made them this thread's to publish)
                    int before;
                    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;\n" : "=r"(before) : "l"(p.counters + first_slot * 2 + h) : "memory");
                    const bool last = before == last_slot - first_slot;
                    if (last) {
                        p.counters[first_slot * 2 + h] = 0; // ready for the next launch
                    }
                    s_sched[3 * kWarps + 2 + h] = last ? 1 : 0;
                }
                named_barrier_sync(1 + h, kSoftmaxThreads);
                store_rows = s_sched[3 * kWarps + 2 + h] != 0;
                if (store_rows && !dead) {
                    // weights 2^(m_i - m); sums run over the fragments in the order of their CTAs, this one's terms in its place: the
                    // result does not depend on which fragment happened to arrive last
                    for (int s2 = first_slot; s2 <= last_slot; ++s2) {
                        if (s2 != slot) {
                            m_all = fmaxf(m_all, __ldcg(part_of(s2) + kHalf * D + row));
                        }
                    }
                    w_own = m_used == -INFINITY ? 0.f : fast_exp2(m_used - m_all);
                    l_all = 0.f;
                    for (int s2 = first_slot; s2 <= last_slot; ++s2) {
                        const float m2 = s2 == slot ? m_used : __ldcg(part_of(s2) + kHalf * D + row);
                        const float l2 = s2 == slot ? l : __ldcg(part_of(s2) + kHalf * D + kHalf + row);
                        l_all = fmaf(l2, m2 == -INFINITY ? 0.f : fast_exp2(m2 - m_all), l_all);
                    }
                }
            }
            if (store_rows && !dead) {
                float inv = l_all > 0.f ? kSumUnit / l_all : 0.f;
                if (p.row_scale != nullptr && t < g.q_len) {
                    inv *= p.row_scale[(long long)(g.q_start + t) * p.nh + head];
                }
                char *out_row = static_cast<char *>(p.out) + ((long long)(g.q_start + t) * p.out_stride + head * D) * 2;
#pragma unroll
                for (int c2 = 0; c2 < D / 64; ++c2) { // 64 columns at a time
                    float v[64];
                    auto own = [&](bool first, float w) { // this fragment's columns
                        float o[32];
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            tmem_ld32(tmem_o + c2 * 64 + c * 32, o);
#pragma unroll
                            for (int k = 0; k < 32; ++k) {
                                v[c * 32 + k] = first ? o[k] : fmaf(o[k], w, v[c * 32 + k]);
                            }
                        }
                    };
                    if (whole) {
                        own(true, 1.f);
                    } else {
#pragma unroll
                        for (int k = 0; k < 64; ++k) {
                            v[k] = 0.f;
                        }
                        for (int s2 = first_slot; s2 <= last_slot; ++s2) {
                            if (s2 == slot) {
                                own(false, w_own);
                                continue;
                            }
                            const float *other = part_of(s2);
                            const float m2 = __ldcg(other + kHalf * D + row);
                            const float w2 = m2 == -INFINITY ? 0.f : fast_exp2(m2 - m_all);
#pragma unroll
                            for (int q16 = 0; q16 < 16; ++q16) {
                                const float4 o = __ldcg(reinterpret_cast<const float4 *>(other) + (c2 * 16 + q16) * kHalf + row);
                                v[q16 * 4] = fmaf(o.x, w2, v[q16 * 4]);
                                v[q16 * 4 + 1] = fmaf(o.y, w2, v[q16 * 4 + 1]);
                                v[q16 * 4 + 2] = fmaf(o.z, w2, v[q16 * 4 + 2]);
                                v[q16 * 4 + 3] = fmaf(o.w, w2, v[q16 * 4 + 3]);
                            }
                        }
                    }
                    if (t < g.q_len && p.out_wide) {
                        // a thread owns a row: a 16-byte store fills half a 32-byte sector and the other half comes with the next
                        // instruction; 32-byte stores halve the write transactions of the epilogue
#pragma unroll
                        for (int q4 = 0; q4 < 4; ++q4) {
                            uint32_t w[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                w[e] = pack_out(v[q4 * 16 + 2 * e] * inv, v[q4 * 16 + 2 * e + 1] * inv, p.bf16 != 0);
                            }
                            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(out_row + c2 * 128 + q4 * 32),
                                         "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                                         : "memory");
                        }
                    } else if (t < g.q_len) {
#pragma unroll
                        for (int q8 = 0; q8 < 8; ++q8) {
                            uint4 w;
                            w.x = pack_out(v[q8 * 8 + 0] * inv, v[q8 * 8 + 1] * inv, p.bf16 != 0);
                            w.y = pack_out(v[q8 * 8 + 2] * inv, v[q8 * 8 + 3] * inv, p.bf16 != 0);
                            w.z = pack_out(v[q8 * 8 + 4] * inv, v[q8 * 8 + 5] * inv, p.bf16 != 0);
                            w.w = pack_out(v[q8 * 8 + 6] * inv, v[q8 * 8 + 7] * inv, p.bf16 != 0);
                            *reinterpret_cast<uint4 *>(out_row + c2 * 128 + q8 * 16) = w;
                        }
                    }
                }
            }
            tc_fence_before(); // the O reads above come before the next fragment's P arrival in program order
        }
    }

    // ---- teardown: everyone is done with TMEM before the allocating warp frees it ----------------------------------
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && *s_abort != 0) {
        atomicOr(p.error_flag, kErrTimeout);
    }
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem_base, S::kTmemCols);
    }
}

// Whether this kernel is the faster one for a call, of what the host knows of it (sums and the longest lengths). Microseconds on an SM; the
// other kernel works on 16 rows x 16 keys at a time (0.23 a CTA of two on an SM, a tile of rows costs about 20 of them besides), this one on 256 x
// 128 (3.5, pieces of no less than sqrt(1.5 longest tile) blocks). Measured, 12 / 2 heads of 128, us there and here: 64 chunks of 8 behind 4000
// tokens 90 and 109, of 16 162 and 110; 8 of 16 behind 4000 35 and 40, of 32 53 and 44; one of 64 behind 300 15 and 22; 32 / 8 heads, 64 chunks of 4
// behind 300 23 and 64, of 16 72 and 66.
bool wide_tiles_pay(const AttnBatch &batch, int nkvh, int group) {
    const double sms = device_sms(), rows = double(batch.total_q) * group;
    const double seen = batch.window > 0 ? std::min(double(batch.max_kv_len), double(batch.window) + batch.keep_first + 256) : double(batch.max_kv_len);
    const double small = (0.5 * batch.n_seqs + rows / 16) * nkvh, large = (batch.n_seqs + rows / 256) * nkvh, longest = std::ceil(seen / kKeys);
    const double there = 8 + 0.23 * std::max(small * (seen / 16 + 20) / (2 * sms), 16.0);
    const double here = 7 + 3.5 * std::max(large * (longest + 2) / sms, std::min(longest, std::max(3.0, std::sqrt(1.5 * longest))));
    return here < there;
}

} // namespace

void attention_quant_tc_scratch(int32_t d, size_t *floats, size_t *counters) {
    const size_t sms = size_t(device_sms());
    *floats = 4 * sms * size_t(d == 64 ? Shape<64>::kPartialFloats : Shape<128>::kPartialFloats);
    *counters = 2 * sms;
}

bool attention_quant_tc(stream_t stream, llaisysDataType_t dtype, const QuantView &kv, const AttnBatch &batch, const void *q, float scale,
                        const AttnOut &out, const AttnScratch &scratch) {
    const bool bf16 = dtype == LLAISYS_DTYPE_BF16;
    const int group = batch.nh / kv.nkvh;
    // the line's units, whatever lengths the arrays hold, and its geometry are counted in 32 bits
    const int64_t longest = std::max(int64_t(kv.table_stride) * kv.blocks_per_page * kPage, int64_t(batch.total_q));
    const int64_t most_tiles = int64_t(batch.total_q) * group / kRows + batch.n_seqs;
    if (!(bf16 || dtype == LLAISYS_DTYPE_F16) || (kv.d != 64 && kv.d != 128) || batch.q_starts == nullptr || out.out == nullptr || out.part != nullptr ||
        group > 32 || int64_t(batch.total_q) * group >= int64_t(1) << 26 || !aligned16(q) || !aligned16(out.out) || out.row_stride % 8 != 0 ||
        longest * group >= int64_t(1) << 30 || most_tiles > (int64_t(1) << 30) / ((longest / kKeys + 1 + kTileCost) * kv.nkvh) || !wide_tiles_pay(batch, kv.nkvh, group)) {
        return false;
    }
    size_t floats, counters;
    attention_quant_tc_scratch(kv.d, &floats, &counters);
    if (scratch.partials == nullptr || scratch.partials_floats < floats || scratch.counters_len < counters) {
        return false;
    }
    QuantChunkParams p{};
    p.kv = kv;
    p.seq_ids = batch.seq_ids;
    p.kv_lens = batch.kv_lens;
    p.q_starts = batch.q_starts;
    p.table_stride = kv.table_stride * kv.blocks_per_page;
    p.n_seqs = batch.n_seqs;
    p.total_q = batch.total_q;
    p.nkvh = kv.nkvh;
    p.group = group;
    p.nh = batch.nh;
    p.group_inverse = uint32_t(((uint64_t(1) << 32) + uint64_t(group) - 1) / uint64_t(group));
    p.q = q;
    p.out = out.out;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.error_flag = scratch.error_flag;
    p.partials = scratch.partials;
    p.counters = scratch.counters;
    p.window = batch.window;
    p.keep_first = batch.window > 0 ? batch.keep_first : 0;
    p.out_stride = out.row_stride != 0 ? out.row_stride : (long long)batch.nh * kv.d;
    p.row_scale = out.row_scale;
    p.bf16 = bf16;
    p.out_wide = reinterpret_cast<uintptr_t>(out.out) % 32 == 0 && p.out_stride % 16 == 0;
    auto start = [&](auto kernel, size_t bytes) {
        LLAISYS_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)));
        kernel<<<unsigned(device_sms()), kThreads, bytes, static_cast<cudaStream_t>(stream)>>>(p);
    };
    auto launch = [&](auto d) {
        constexpr int D = decltype(d)::value;
        if (D == 128 && kv.wait_limit != kMbarWaitLimit && !kv.f8 && batch.window == 0) { // (a limit that tests set)
            start(attention_quant_tc_kernel<128, false, false, true>, Shape<128>::kBytes);
        } else if (batch.window > 0) {
            start(kv.f8 ? attention_quant_tc_kernel<D, true, true> : attention_quant_tc_kernel<D, false, true>, Shape<D>::kBytes);
        } else {
            start(kv.f8 ? attention_quant_tc_kernel<D, true, false> : attention_quant_tc_kernel<D, false, false>, Shape<D>::kBytes);
        }
    };
    if (kv.d == 64) {
        launch(std::integral_constant<int, 64>{});
    } else {
        launch(std::integral_constant<int, 128>{});
    }
    check_launch("attention_quant_tc");
    return true;
}

} // namespace llaisys::kernels
