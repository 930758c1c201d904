// Rows into a page pool held in 8 bits, and back.
//
// Append. Rows that go to one block of 16 tokens are neighbours in the call: a RUN. With x the run's numbers of one kv head (K and V apart),
//     s' = max(s, max|x| / M, 2^-100),  c = round(x (1 / s')),  tokens in front of the run, where s' > s: c = round(c (s (1 / s')))
// One warp per run, head and K or V: nobody else touches those codes or that scale, so there is nothing to order.
//
// Bound: bytes, rows in and codes out (and back the other way); for a token per sequence the chain of loads row -> table -> tile. A warp copies a
// run to shared memory between the maximum and the rounding (asynchronously, while its place is looked up), so that rows are read once, and stores
// codes 16 bytes a lane in the order of the tile (quant_tile.cuh): a lane of K takes the four neighbours that make a word of its own; one of V takes
// four tokens of four dims, turns its 4 x 4 codes round and passes them on through shared memory.
// Measured: 65536 rows of 2 heads of 128 in bf16, integers, in 21.9 us and back out 20.1 (101 MB each way: 4.6 and 5.0 TB/s; the append
// issues in 68 % of the cycles -- a number costs its maximum, a product, a rounding and its share of the byte moves -- and waits for its copies a third of a
// warp's time); 64 rows of 64 sequences 4.0 and 3.5 us. (Rows held in registers over both passes of
// an append 55 us with the way back, through shared memory with scalar arithmetic 37 + 21.)
#include "kernels.hpp"
#include "launch_utils.cuh"
#include "mma_utils.cuh"
#include "quant_tile.cuh"

#include <algorithm>
#include <type_traits>

namespace llaisys::kernels {

namespace {

constexpr int kWarps = 4;
constexpr int kChunk = 16; // rows a warp looks for runs in, where there are many

// Four neighbouring numbers of a row as they are.
template <typename T>
struct Four {
    typename std::conditional<sizeof(T) == 4, uint4, uint2>::type raw;
};
__device__ __forceinline__ float4 widened(const Four<float> &v) {
    return make_float4(__uint_as_float(v.raw.x), __uint_as_float(v.raw.y), __uint_as_float(v.raw.z), __uint_as_float(v.raw.w));
}
__device__ __forceinline__ float4 widened(const Four<__half> &v) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&v.raw.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&v.raw.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 widened(const Four<__nv_bfloat16> &v) {
    return make_float4(__uint_as_float(v.raw.x << 16), __uint_as_float(v.raw.x & 0xffff0000u), __uint_as_float(v.raw.y << 16),
                       __uint_as_float(v.raw.y & 0xffff0000u));
}
__device__ __forceinline__ void narrow(float4 v, Four<float> &to) {
    to.raw = make_uint4(__float_as_uint(v.x), __float_as_uint(v.y), __float_as_uint(v.z), __float_as_uint(v.w));
}
__device__ __forceinline__ void narrow(float4 v, Four<__half> &to) {
    const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    to.raw = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}
__device__ __forceinline__ void narrow(float4 v, Four<__nv_bfloat16> &to) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    to.raw = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}

// Two products and two sums at a time, each rounded once.
__device__ __forceinline__ float2 mul2(float2 a, float b) {
    float2 d;
    asm("{\n"
        ".reg .b64 x, y, z;\n"
        "mov.b64 x, {%2, %3};\n"
        "mov.b64 y, {%4, %4};\n"
        "mul.rn.f32x2 z, x, y;\n"
        "mov.b64 {%0, %1}, z;\n"
        "}\n"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float b) {
    float2 d;
    asm("{\n"
        ".reg .b64 x, y, z;\n"
        "mov.b64 x, {%2, %3};\n"
        "mov.b64 y, {%4, %4};\n"
        "add.rn.f32x2 z, x, y;\n"
        "mov.b64 {%0, %1}, z;\n"
        "}\n"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b));
    return d;
}
// Codes of four numbers times `by` (and so at most M, up to a rounding), packed. Integers: 1.5 * 2^23 + 128 more than x, rounded to nearest even,
// has c + 128 in its low byte.
template <bool kF8>
__device__ __forceinline__ uint32_t codes_times(float4 v, float by) {
    const float2 x = mul2(make_float2(v.x, v.y), by), y = mul2(make_float2(v.z, v.w), by);
    if constexpr (kF8) {
        const uint32_t a = __nv_cvt_float2_to_fp8x2(x, __NV_SATFINITE, __NV_E4M3), b = __nv_cvt_float2_to_fp8x2(y, __NV_SATFINITE, __NV_E4M3);
        return a | (b << 16);
    } else {
        constexpr float kMagic = 12582912.f + 128.f;
        // (one at a time: the packed product and sum come out of the assembler as one operation, and the product unrounded)
        const auto of = [](float a) { return __float_as_uint(__fadd_rn(a, kMagic)); };
        return __byte_perm(__byte_perm(of(x.x), of(x.y), 0x0040), __byte_perm(of(y.x), of(y.y), 0x0040), 0x5410);
    }
}
template <bool kF8>
__device__ __forceinline__ float4 worth_of(uint32_t w) {
    if constexpr (kF8) {
        const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xffffu), __NV_E4M3);
        const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3);
        const float2 x = __half22float2(__half2(a)), y = __half22float2(__half2(b));
        return make_float4(x.x, x.y, y.x, y.y);
    } else { // 0x4b000000 | u is 2^23 + u
        const float2 x = add2(make_float2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440)), __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7441))),
                              -8388736.f);
        const float2 y = add2(make_float2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7442)), __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7443))),
                              -8388736.f);
        return make_float4(x.x, x.y, y.x, y.y);
    }
}
// Byte k of the four words -> word k.
__device__ __forceinline__ void turn(uint32_t (&w)[4]) {
    const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[2], w[3], 0x5140); // bytes 0 and 1 of two words, side by side
    const uint32_t c = __byte_perm(w[0], w[1], 0x7362), e = __byte_perm(w[2], w[3], 0x7362); // bytes 2 and 3
    w[0] = __byte_perm(a, b, 0x5410);
    w[1] = __byte_perm(a, b, 0x7632);
    w[2] = __byte_perm(c, e, 0x5410);
    w[3] = __byte_perm(c, e, 0x7632);
}

// A run: `count` tokens from slot `slot` of a block on, rows `row` ... of the call.
struct Run {
    int row, slot, count;
    unsigned char *tile; // of the head
};

// fetch(row, count), then body(run) where the run has a place in the pool and lost() where it has none, for every run that begins among the warp's rows
// [row0, row0 + rows). Rows are read 32 at a time: a run that begins among the first 16 ends among them. seq_ids null: rows are tokens 0, 1, ... of
// sequence seq_row.
template <typename Fetch, typename Body, typename Lost>
__device__ __forceinline__ void for_runs(const QuantView &kv, const int32_t *seq_ids, const int32_t *positions, int seq_row, int row0, int rows, int n_rows,
                                         int head, bool skip_none, int32_t *error_flag, Fetch &&fetch, Body &&body, Lost &&lost) {
    const int lane = threadIdx.x & 31;
    const bool in = int64_t(row0) + lane < n_rows;
    const int seq = !in ? -2 : seq_ids ? seq_ids[row0 + lane] : seq_row, pos = !in ? -2 : seq_ids ? positions[row0 + lane] : row0 + lane;
    int seq_up = __shfl_up_sync(0xffffffffu, seq, 1), pos_up = __shfl_up_sync(0xffffffffu, pos, 1);
    if (lane == 0) {
        seq_up = row0 == 0 ? -2 : seq_ids ? seq_ids[row0 - 1] : seq_row;
        pos_up = row0 == 0 ? -2 : seq_ids ? positions[row0 - 1] : row0 - 1;
    }
    const bool joined = in && pos > 0 && pos % kQuantTokens != 0 && seq_up == seq && pos_up == pos - 1; // to the row in front of it
    const unsigned joins = __ballot_sync(0xffffffffu, joined);
    unsigned leaders = __ballot_sync(0xffffffffu, in && !joined && lane < rows);
    for (; leaders != 0; leaders &= leaders - 1) {
        const int from = __ffs(leaders) - 1;
        const int its_seq = __shfl_sync(0xffffffffu, seq, from), its_pos = __shfl_sync(0xffffffffu, pos, from);
        if (skip_none && its_seq == -1) {
            continue; // no token
        }
        if (its_pos < 0) {
            if (lane == 0) {
                atomicOr(error_flag, kErrBadPosition);
            }
            continue;
        }
        Run run;
        const unsigned behind = from < 31 ? joins >> (from + 1) : 0u;
        run.row = row0 + from;
        run.slot = its_pos % kQuantTokens;
        run.count = __ffs(~behind); // the leader and the rows joined to it
        fetch(run.row, run.count);
        if (!quant_tile_of(kv, its_seq, its_pos / kQuantTokens, error_flag, run.tile)) {
            lost();
            continue;
        }
        run.tile += int64_t(head) * kv.tile_bytes;
        body(run);
    }
}

// The places of a lane's words in a tile: of word u = 4 v + k of K, its token and first dim; of V, see below.
__device__ __forceinline__ int k_token(int lane, int k) { return 4 * (lane >> 3) + 2 * (k & 1) + ((lane >> 2) & 1); }
__device__ __forceinline__ int k_dim(int lane, int v, int k) { return 32 * v + 16 * (k >> 1) + 4 * (lane & 3); }
// A lane's share of V in vector v: tokens 4 (lane % 4) ..+3 of dims 32 v + 4 (lane / 4) ..+3. Turned round, word b of it (dim + b) is word lane / 8 of
// lane 16 (lane / 4 % 2) + 4 b + lane % 4.
__device__ __forceinline__ int v_word(int lane, int b) { return 4 * (16 * ((lane >> 2) & 1) + 4 * b + (lane & 3)) + (lane >> 3); }

// Four tokens' or words' places: word k of vector v of a lane's share, as an offset from the lane's first number of the run's block in rows.
template <bool kV>
__device__ __forceinline__ int share_token(int lane, int k) {
    return kV ? 4 * (lane & 3) + k : k_token(lane, k);
}
template <bool kV>
__device__ __forceinline__ int share_dim(int lane, int v, int k) {
    return kV ? 32 * v + 4 * (lane >> 2) : k_dim(lane, v, k);
}

// The largest magnitude of the numbers fed to it, by the bits without their sign: infinities and NaN come out above every number.
template <typename T>
struct Largest {
    uint32_t bits = 0;
    __device__ __forceinline__ void take(uint4 v) {
        if constexpr (sizeof(T) == 4) {
            bits = __vimax3_u32(__vimax3_u32(bits, v.x & 0x7fffffffu, v.y & 0x7fffffffu), v.z & 0x7fffffffu, v.w & 0x7fffffffu);
        } else { // two at a time
            bits = __vimax3_u16x2(__vimax3_u16x2(bits, v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), v.z & 0x7fff7fffu, v.w & 0x7fff7fffu);
        }
    }
    __device__ __forceinline__ float over_warp() { // not below infinity: something was not finite
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(min(__reduce_max_sync(0xffffffffu, bits), 0x7f800000u));
        } else {
            const uint32_t most = __reduce_max_sync(0xffffffffu, max(bits & 0xffffu, bits >> 16));
            if constexpr (std::is_same<T, __half>::value) {
                return most >= 0x7c00u ? INFINITY : __half2float(__ushort_as_half(static_cast<unsigned short>(most)));
            } else {
                return most >= 0x7f80u ? INFINITY : __uint_as_float(most << 16);
            }
        }
    }
};

// Shared memory of a warp that appends: 16 rows (16 bytes apart more than they are long: a lane's neighbours in tokens lie in other banks), the tile's
// half as it was, and the place where V is turned.
constexpr int kPad = 16;
__host__ __device__ __forceinline__ int append_smem(int d, int elem) { return kQuantTokens * (d * elem + kPad) + kQuantTokens * d + 512; }

// body(row, piece) for this lane's share of `rows` rows of `pieces` times 16 bytes.
template <typename Body>
__device__ __forceinline__ void for_pieces(int pieces, int rows, Body &&body) {
    const int lane = threadIdx.x & 31;
    if (pieces <= 32 && (pieces & (pieces - 1)) == 0) { // whole rows at a time
        const int log = 31 - __clz(pieces), step = 32 >> log, c = lane & (pieces - 1);
        int r = lane >> log;
        if (rows == kQuantTokens && step <= 2) {
#pragma unroll
            for (int k = 0; k < kQuantTokens / 2; ++k) { // (two rows a step, or one and as many again)
                body(r, c);
                r += step;
            }
            if (step == 2) {
                return;
            }
        }
        for (; r < rows; r += step) {
            body(r, c);
        }
        return;
    }
    for (int r = 0; r < rows; ++r) {
        for (int c = lane; c < pieces; c += 32) {
            body(r, c);
        }
    }
}

template <typename T, bool kF8, bool kV, bool kAll>
__device__ __forceinline__ void append_run(const QuantView &kv, const Run &run, unsigned char *smem) {
    constexpr float kMost = kF8 ? 448.f : 127.f;
    const int lane = threadIdx.x & 31, d = kv.d, row_bytes = d * int(sizeof(T)), stride = row_bytes + kPad;
    unsigned char *s_tile = smem + kQuantTokens * stride;
    uint4 *s_turn = reinterpret_cast<uint4 *>(s_tile + kQuantTokens * d);
    float *scale_at = reinterpret_cast<float *>(run.tile + quant_scales_at(d)) + (kV ? 1 : 0);
    uint4 *codes = reinterpret_cast<uint4 *>(run.tile + (kV ? kQuantTokens * d : 0)) + lane;
    if constexpr (!kAll) {
        for (int v = 0; v < d >> 5; ++v) {
            cp_async_16(smem_u32(s_tile) + 16 * (32 * v + lane), codes + 32 * v, 16);
        }
        cp_async_commit();
    }
    const float old = !kAll && run.slot > 0 ? *scale_at : 0.f;
    cp_async_wait<0>();
    __syncwarp();
    Largest<T> largest;
    for_pieces(row_bytes / 16, run.count, [&](int r, int c) { largest.take(*reinterpret_cast<const uint4 *>(smem + r * stride + 16 * c)); });
    const float most = largest.over_warp();
    const bool finite = most < INFINITY && !isnan(old);
    const float scale = finite ? fmaxf(fmaxf(old, most / kMost), kQuantFloor) : NAN, inverse = finite ? 1.f / scale : 0.f;
    const bool grows = !kAll && run.slot > 0 && scale > old;
    const float factor = __fmul_rn(old, inverse);
    const unsigned char *at[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        at[k] = smem + (share_token<kV>(lane, k) - run.slot) * stride + share_dim<kV>(lane, 0, k) * int(sizeof(T));
    }
#pragma unroll 2
    for (int v = 0; v < d >> 5; ++v) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int token = share_token<kV>(lane, k) - run.slot;
            w[k] = 0;
            if (kAll || (token >= 0 && token < run.count)) {
                w[k] = codes_times<kF8>(widened(*reinterpret_cast<const Four<T> *>(at[k] + 32 * v * int(sizeof(T)))), inverse);
            }
            w[k] = finite ? w[k] : kF8 ? 0u : 0x80808080u;
        }
        if constexpr (kV) {
            turn(w);
            __syncwarp();
            uint32_t *to = reinterpret_cast<uint32_t *>(s_turn);
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                to[v_word(lane, b)] = w[b];
            }
            __syncwarp();
            const uint4 y = s_turn[lane];
            w[0] = y.x, w[1] = y.y, w[2] = y.z, w[3] = y.w;
        }
        if constexpr (!kAll) {
            const uint4 had = *reinterpret_cast<const uint4 *>(s_tile + 16 * (32 * v + lane));
            const uint32_t h[4] = {had.x, had.y, had.z, had.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t kept = grows ? codes_times<kF8>(worth_of<kF8>(h[k]), factor) : h[k];
                if constexpr (kV) { // a word is tokens 4 (lane % 4) ..+3
                    uint32_t front = 0, fresh = 0;
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const int token = 4 * (lane & 3) + b - run.slot;
                        front |= token < 0 ? 0xffu << (8 * b) : 0u;
                        fresh |= token >= 0 && token < run.count ? 0xffu << (8 * b) : 0u;
                    }
                    w[k] = (w[k] & fresh) | (kept & front) | (h[k] & ~(fresh | front));
                } else {
                    const int token = k_token(lane, k) - run.slot;
                    w[k] = token < 0 ? kept : token < run.count ? w[k] : h[k];
                }
            }
        }
        codes[32 * v] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (lane == 0) {
        *scale_at = scale;
    }
    __syncwarp(); // the rows' place is the next run's
}

template <typename T, bool kF8>
__global__ void __launch_bounds__(kWarps * 32, 8) quant_append_kernel(QuantView kv, const T *__restrict__ k_rows, const T *__restrict__ v_rows,
                                                                   const int32_t *__restrict__ seq_ids, const int32_t *__restrict__ positions,
                                                                   int32_t n_rows, int32_t chunk, int32_t *error_flag) {
    extern __shared__ __align__(16) unsigned char smem_all[];
    const int warp = threadIdx.x >> 5, parts = 2 * kv.nkvh, row_bytes = kv.d * int(sizeof(T));
    unsigned char *smem = smem_all + warp * append_smem(kv.d, sizeof(T));
    const int64_t unit = int64_t(blockIdx.x) * kWarps + warp;
    const int head = int(unit % parts) >> 1;
    const bool is_v = unit & 1;
    const int64_t row0 = unit / parts * chunk;
    if (row0 >= n_rows) {
        return;
    }
    grid_dependency_wait(); // (launched programmatically: under the tail of the kernel in front)
    grid_launch_dependents();
    const unsigned char *rows = reinterpret_cast<const unsigned char *>((is_v ? v_rows : k_rows) + int64_t(head) * kv.d);
    const int64_t row_step = int64_t(kv.nkvh) * row_bytes;
    // the rows are on their way before their place in the pool is looked up
    const auto fetch = [&](int row, int count) {
        const uint32_t to = smem_u32(smem);
        for_pieces(row_bytes / 16, count, [&](int r, int c) {
            cp_async_16(to + r * (row_bytes + kPad) + 16 * c, rows + (int64_t(row) + r) * row_step + 16 * c, 16);
        });
        cp_async_commit();
    };
    for_runs(kv, seq_ids, positions, 0, int(row0), chunk, n_rows, head, true, error_flag, fetch, [&](const Run &run) {
        const bool all = run.count == kQuantTokens;
        if (is_v) {
            all ? append_run<T, kF8, true, true>(kv, run, smem) : append_run<T, kF8, true, false>(kv, run, smem);
        } else {
            all ? append_run<T, kF8, false, true>(kv, run, smem) : append_run<T, kF8, false, false>(kv, run, smem);
        }
    }, [] { // the rows are on their way to where the next run's will lie: copies have no order among themselves
        cp_async_wait<0>();
        __syncwarp();
    });
}

template <typename T, bool kF8, int kVecs, bool kV, bool kAll>
__device__ __forceinline__ void gather_run(const QuantView &kv, const Run &run, T *rows, int64_t row_step, uint4 *s_turn) {
    const int lane = threadIdx.x & 31, d = kv.d, vecs = d >> 5;
    const float scale = reinterpret_cast<const float *>(run.tile + quant_scales_at(d))[kV ? 1 : 0];
    const uint4 *codes = reinterpret_cast<const uint4 *>(run.tile + (kV ? kQuantTokens * d : 0)) + lane;
    const auto in = [&](int token) { return kAll || (token >= run.slot && token < run.slot + run.count); };
    const int low = share_token<kV>(lane, 0);
    const bool mine = kAll ? true : kV ? low + 3 >= run.slot && low < run.slot + run.count : in(low) || in(low + 2); // any of the lane's tokens
    T *at[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        at[k] = rows + (int64_t(run.row - run.slot) + share_token<kV>(lane, k)) * row_step + share_dim<kV>(lane, 0, k);
    }
    uint4 had[kVecs];
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
        had[v] = make_uint4(0, 0, 0, 0);
        if (v < vecs && mine) {
            had[v] = codes[32 * v];
        }
    }
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
        if (v < vecs) {
            uint32_t w[4] = {had[v].x, had[v].y, had[v].z, had[v].w};
            if constexpr (kV) {
                __syncwarp();
                s_turn[lane] = had[v];
                __syncwarp();
                const uint32_t *from = reinterpret_cast<const uint32_t *>(s_turn);
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    w[b] = from[v_word(lane, b)];
                }
                turn(w);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (in(share_token<kV>(lane, k))) {
                    const float4 y = worth_of<kF8>(w[k]);
                    const float2 a = mul2(make_float2(y.x, y.y), scale), b = mul2(make_float2(y.z, y.w), scale);
                    Four<T> to;
                    narrow(make_float4(a.x, a.y, b.x, b.y), to);
                    *reinterpret_cast<Four<T> *>(at[k] + 32 * v) = to;
                }
            }
        }
    }
}

template <typename T, bool kF8, int kVecs>
__global__ void __launch_bounds__(kWarps * 32, kVecs > 4 ? 6 : 10) quant_gather_kernel(QuantView kv, const int32_t *__restrict__ seq_ids,
                                                                   const int32_t *__restrict__ positions, int32_t seq_row, int32_t n_rows, int32_t chunk,
                                                                   T *__restrict__ k_out, T *__restrict__ v_out, int32_t *error_flag) {
    __shared__ uint4 s_turn[kWarps][32];
    const int warp = threadIdx.x >> 5, parts = 2 * kv.nkvh;
    const int64_t unit = int64_t(blockIdx.x) * kWarps + warp;
    const int head = int(unit % parts) >> 1;
    const bool is_v = unit & 1;
    const int64_t row0 = unit / parts * chunk;
    if (row0 >= n_rows) {
        return;
    }
    T *rows = (is_v ? v_out : k_out) + int64_t(head) * kv.d;
    const int64_t row_step = int64_t(kv.nkvh) * kv.d;
    for_runs(kv, seq_ids, positions, seq_row, int(row0), chunk, n_rows, head, false, error_flag, [](int, int) {}, [&](const Run &run) {
        const bool all = run.count == kQuantTokens;
        if (is_v) {
            all ? gather_run<T, kF8, kVecs, true, true>(kv, run, rows, row_step, s_turn[warp])
                : gather_run<T, kF8, kVecs, true, false>(kv, run, rows, row_step, s_turn[warp]);
        } else {
            all ? gather_run<T, kF8, kVecs, false, true>(kv, run, rows, row_step, s_turn[warp])
                : gather_run<T, kF8, kVecs, false, false>(kv, run, rows, row_step, s_turn[warp]);
        }
    }, [] {});
}

// body(T{}, kF8, kVecs)
template <typename Body>
void pick(llaisysDataType_t dtype, const QuantView &kv, Body &&body) {
    dispatch(dtype, [&](auto t) {
        auto with = [&](auto f8) {
            if (kv.d <= 64) {
                body(t, f8, std::integral_constant<int, 2>{});
            } else if (kv.d <= 128) {
                body(t, f8, std::integral_constant<int, 4>{});
            } else {
                body(t, f8, std::integral_constant<int, 8>{});
            }
        };
        if (kv.f8) {
            with(std::true_type{});
        } else {
            with(std::false_type{});
        }
    });
}

// Rows a warp looks at: a run begins at every row where sequences bring one each, and a warp per row then shortens the chain of loads; many rows
// are mostly whole blocks.
int chunk_of(int32_t n_rows, int32_t nkvh) { return int64_t(n_rows) * 2 * nkvh <= int64_t(device_sms()) * 64 ? 1 : kChunk; }
unsigned blocks_of(int32_t n_rows, int32_t nkvh, int chunk) {
    const int64_t units = (int64_t(n_rows) + chunk - 1) / chunk * 2 * nkvh, blocks = (units + kWarps - 1) / kWarps;
    CHECK_ARGUMENT(blocks <= 0x7fffffff, "paged KV: too many rows for one launch");
    return unsigned(blocks);
}

} // namespace

void quant_append(stream_t stream, llaisysDataType_t dtype, const QuantView &kv, const void *k_rows, const void *v_rows,
                  const int32_t *seq_ids, const int32_t *positions, int32_t n_rows, int32_t *error_flag) {
    CHECK_ARGUMENT(aligned16(k_rows) && aligned16(v_rows), "paged KV append: rows must be 16-byte aligned");
    const int chunk = chunk_of(n_rows, kv.nkvh);
    const unsigned blocks = blocks_of(n_rows, kv.nkvh, chunk);
    dispatch(dtype, [&](auto t) {
        using T = decltype(t);
        auto kernel = kv.f8 ? quant_append_kernel<T, true> : quant_append_kernel<T, false>;
        const int bytes = kWarps * append_smem(kv.d, sizeof(T));
        LLAISYS_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        launch_programmatic_smem(kernel, dim3(blocks), kWarps * 32, size_t(bytes), static_cast<cudaStream_t>(stream), kv, static_cast<const T *>(k_rows),
                                 static_cast<const T *>(v_rows), seq_ids, positions, n_rows, chunk, error_flag);
    });
    check_launch("quant_append");
}

void quant_gather(stream_t stream, llaisysDataType_t dtype, const QuantView &kv, const int32_t *seq_ids, const int32_t *positions,
                  int32_t seq_row, int32_t n_rows, void *k_out, void *v_out, int32_t *error_flag) {
    CHECK_ARGUMENT(aligned16(k_out) && aligned16(v_out), "paged KV gather: rows must be 16-byte aligned");
    const int chunk = chunk_of(n_rows, kv.nkvh);
    const unsigned blocks = blocks_of(n_rows, kv.nkvh, chunk);
    pick(dtype, kv, [&](auto t, auto f8, auto vecs) {
        using T = decltype(t);
        quant_gather_kernel<T, decltype(f8)::value, decltype(vecs)::value><<<blocks, kWarps * 32, 0, static_cast<cudaStream_t>(stream)>>>(
            kv, seq_ids, positions, seq_row, n_rows, chunk, static_cast<T *>(k_out), static_cast<T *>(v_out), error_flag);
    });
    check_launch("quant_gather");
}

} // namespace llaisys::kernels
