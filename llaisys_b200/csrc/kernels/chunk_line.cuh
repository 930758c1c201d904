// The line of key blocks that the tcgen05 chunk kernels cut over the SMs, and the packed arithmetic of their softmax rows.
//
// Rows are packed over queries and the heads of a group, 256 of a sequence and kv head are a tile, and a tile visits its visible keys 128 at a
// time. P, the parameters of a kernel, names: kv_lens, q_starts, n_seqs, nkvh, group, window, keep_first, table_stride (pages of 16 tokens),
// contiguous, const_q_len, const_kv_len; kQueriesMayLead: chunks may be longer than what their sequence holds, and end with total_q.
#pragma once

#include "device_utils.cuh"

namespace llaisys::kernels {

namespace {

constexpr int kPage = 16;
constexpr int kHalf = 128, kRows = 2 * kHalf; // packed rows of a half and of a tile
constexpr int kKeys = 128, kPagesPerBlock = kKeys / kPage;
// What a tile costs besides its blocks (loading Q, draining the pipeline, storing its rows: about 11500 clocks), in units of a block's time.
constexpr int kTileCost = 4;

// ---- the line of blocks ------------------------------------------------------------------------------------------

struct SeqGeom {
    int q_start, q_len, kv_len, off, n_qb; // query t sees keys j <= t + off
    int group, window, kept_blocks;        // window 0: none; kept_blocks: blocks that hold the first tokens a window keeps
};

template <typename P>
__device__ __forceinline__ SeqGeom seq_geom(const P &p, int a) {
    SeqGeom g;
    if (p.contiguous) {
        g.q_start = 0;
        g.q_len = p.const_q_len;
        g.kv_len = max(p.const_kv_len, g.q_len);
    } else {
        g.q_start = p.q_starts[a];
        g.q_len = p.q_starts[a + 1] - g.q_start;
        if constexpr (P::kQueriesMayLead) {
            g.q_start = max(g.q_start, 0);
            g.q_len = max(min(p.q_starts[a + 1], p.total_q) - g.q_start, 0);
            g.kv_len = max(min(p.kv_lens[a], p.table_stride * kPage), g.q_len);
        } else {
            g.kv_len = min(max(p.kv_lens[a], g.q_len), p.table_stride * kPage);
        }
    }
    g.q_len = min(g.q_len, g.kv_len); // (a chunk longer than the tables can hold: flagged elsewhere, never off the end here)
    g.off = g.kv_len - g.q_len;
    g.n_qb = (g.q_len * p.group + kRows - 1) / kRows;
    g.group = p.group;
    // (a chunk longer than what its sequence holds, where a kernel allows it: no window on the line, so that none of its blocks is left out)
    g.window = P::kQueriesMayLead && p.kv_lens[a] < g.q_len ? 0 : p.window;
    g.kept_blocks = (p.keep_first + kKeys - 1) / kKeys;
    return g;
}

// keys any row of row block qb can see
__device__ __forceinline__ int tile_kv_hi(const SeqGeom &g, int qb) { return min(g.kv_len, (qb * kRows + kRows - 1) / g.group + 1 + g.off); }
// key blocks that no row of the row block sees, between the blocks of the kept first tokens and the one where the window of its first
// row begins; a tile's blocks are counted without them
__device__ __forceinline__ int tile_gap(const SeqGeom &g, int qb) {
    return g.window > 0 ? max(qb * kRows / g.group + g.off - g.window + 1 - g.kept_blocks * kKeys, 0) / kKeys : 0;
}
__device__ __forceinline__ int tile_blocks(const SeqGeom &g, int qb) { return (tile_kv_hi(g, qb) + kKeys - 1) / kKeys - tile_gap(g, qb); }

// sum of floor((2 i + b) / m) over i < n, for 0 <= b and m <= 32. Callers see to it that the sum fits 32 bits; n (n - 1) may not where a / m is 0, and
// counts for nothing there.
__device__ __forceinline__ int floor_sum(int n, int m, int b) {
    int sum = 0, a = 2;
    while (n > 0) {
        sum += (a >= m ? n * (n - 1) / 2 * (a / m) : 0) + n * (b / m);
        a %= m;
        b %= m;
        const int y = a * n + b;
        if (y < m) {
            break;
        }
        n = y / m;
        b = y % m;
        const int t = m;
        m = a;
        a = t;
    }
    return sum;
}
// Units of the line in front of row block qb of a sequence (qb < n_qb), per kv head. Whole tiles: one each. Else the tiles' blocks in closed
// form -- tile i ends at key floor((256 i + 255) / group) + 1 + off, so it has floor((2 i + B) / group) blocks, and its gap is such a term too -- and kTileCost each
__device__ __forceinline__ int units_before(const SeqGeom &g, int qb, bool whole) {
    static_assert(kRows == 2 * kKeys, "row blocks advance two key blocks over the group's heads");
    if (whole) {
        return qb;
    }
    int units = qb * kTileCost + floor_sum(qb, g.group, (kRows - 1 + g.group * (g.off + kKeys)) >> 7);
    if (g.window > 0) {
        const int c = g.group * (g.off - g.window + 1 - g.kept_blocks * kKeys), q0 = c >= 0 ? 0 : (-c + kRows - 1) / kRows;
        if (q0 < qb) {
            units -= floor_sum(qb - q0, g.group, 2 * q0 + (c >> 7)); // (an arithmetic shift: floor)
        }
    }
    return units;
}
// units of a whole sequence
template <typename P>
__device__ __forceinline__ int seq_units(const P &p, const SeqGeom &g, bool whole) {
    if (whole || g.n_qb == 0) {
        return g.n_qb * p.nkvh;
    }
    return (units_before(g, g.n_qb - 1, false) + tile_blocks(g, g.n_qb - 1) + kTileCost) * p.nkvh;
}

// Position on the line: every role of the CTA walks the same fragments with one of these.
struct Walker {
    int a;         // sequence
    int seq_begin; // index on the line of its first unit
    int n_units;   // its units (all kv heads)
    SeqGeom g;
    int qb, qb_begin; // the row block of the last position asked for, and its first unit inside the sequence (positions only move forward)
    bool whole;       // a unit is a whole tile
};

struct Fragment {
    int a, qb, kvh;
    int b0, b1;     // key blocks [b0, b1) of the tile, counted without its gap
    int gap;        // tile_gap
    int tile_nblk;  // blocks of the whole tile
    int tile_begin; // index on the line of the tile's block 0
    int rows;       // live rows of the tile
    int units;      // from its first unit to the position behind it
};
struct Place {
    Walker w;
    Fragment f;
    int pos; // on the line, behind the fragment
};

// The fragment that starts at or after unit `pos` of the line and before piece_end: `pos` moves on to its first block (over the units
// at a tile's end that stand for no block). False when the piece holds no further block.
template <typename P>
__device__ __forceinline__ bool locate(const P &p, Walker &w, int &pos, int piece_end, Fragment &f) {
    while (pos < piece_end) {
        while (pos >= w.seq_begin + w.n_units && w.a + 1 < p.n_seqs) {
            w.seq_begin += w.n_units;
            ++w.a;
            w.g = seq_geom(p, w.a);
            w.n_units = seq_units(p, w.g, w.whole);
            w.qb = w.qb_begin = 0;
        }
        int x = pos - w.seq_begin - w.qb_begin, nb = tile_blocks(w.g, w.qb), span = w.whole ? 1 : nb + kTileCost;
        while (x >= span * p.nkvh && w.qb + 1 < w.g.n_qb) {
            x -= span * p.nkvh;
            w.qb_begin += span * p.nkvh;
            nb = tile_blocks(w.g, ++w.qb);
            span = w.whole ? 1 : nb + kTileCost;
        }
        const int kvh = min(x / span, p.nkvh - 1), b0 = x - kvh * span;
        if (b0 >= span) {
            return false; // (past the end of the line: no caller asks)
        }
        if (b0 >= nb) { // behind the tile's last block: on to the next tile
            pos += span - b0;
            continue;
        }
        f.a = w.a;
        f.qb = w.qb;
        f.kvh = kvh;
        f.b0 = b0;
        f.tile_nblk = nb;
        f.gap = tile_gap(w.g, w.qb);
        f.b1 = w.whole ? nb : min(nb, b0 + (piece_end - pos));
        f.units = w.whole ? 1 : f.b1 - b0;
        f.tile_begin = pos - b0;
        f.rows = min(kRows, w.g.q_len * w.g.group - w.qb * kRows);
        return true;
    }
    return false;
}

// Blackwell's wider scalar arithmetic for the softmax rows: a three-input maximum and two-wide f32 multiply-add / add
// (one instruction for two scores: these warps are short of issue slots, not of pipe throughput).
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void fma2(float &x0, float &x1, float a0, float a1, float b, float c) { // x = a * b + c
    asm("{\n"
        ".reg .b64 ra, rb, rc, rd;\n"
        "mov.b64 ra, {%2, %3};\n"
        "mov.b64 rb, {%4, %4};\n"
        "mov.b64 rc, {%5, %5};\n"
        "fma.rn.f32x2 rd, ra, rb, rc;\n"
        "mov.b64 {%0, %1}, rd;\n"
        "}\n"
        : "=f"(x0), "=f"(x1)
        : "f"(a0), "f"(a1), "f"(b), "f"(c));
}
__device__ __forceinline__ void add2(float &s0, float &s1, float a0, float a1) { // s += a
    asm("{\n"
        ".reg .b64 rs, ra;\n"
        "mov.b64 rs, {%0, %1};\n"
        "mov.b64 ra, {%2, %3};\n"
        "add.rn.f32x2 rs, rs, ra;\n"
        "mov.b64 {%0, %1}, rs;\n"
        "}\n"
        : "+f"(s0), "+f"(s1)
        : "f"(a0), "f"(a1));
}

} // namespace

} // namespace llaisys::kernels
