// Rows into a page pool held in 8 bits, and back.
//
// Append. Rows that go to one block of 16 tokens are neighbours in the call: a RUN. With x the run's numbers of one kv head (K and V apart),
//     s' = max(s, max|x| / M, 2^-100),  c = round(x (1 / s')),  tokens in front of the run, where s' > s: c = round(c (s (1 / s')))
// One warp per run, head and K or V: nobody else touches those codes or that scale, so there is nothing to order.
#include "kernels.hpp"
#include "launch_utils.cuh"
#include "quant_tile.cuh"

#include <algorithm>

namespace llaisys::kernels {

namespace {

template <typename T, bool kF8>
__global__ void __launch_bounds__(128) quant_append_kernel(QuantView kv, const T *__restrict__ k_rows, const T *__restrict__ v_rows,
                                                           const int32_t *__restrict__ seq_ids, const int32_t *__restrict__ positions,
                                                           int32_t n_rows, int32_t *error_flag) {
    constexpr float kMost = kF8 ? 448.f : 127.f;
    const int lane = threadIdx.x & 31, d = kv.d;
    const int64_t units = int64_t(n_rows) * 2 * kv.nkvh, warps = int64_t(gridDim.x) * 4;
    for (int64_t u = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5); u < units; u += warps) {
        const int32_t row = int32_t(u / (2 * kv.nkvh)), part = int32_t(u - int64_t(row) * 2 * kv.nkvh);
        const int head = part >> 1;
        const bool is_v = part & 1;
        const int seq = seq_ids[row], pos = positions[row];
        if (seq == -1 || (row > 0 && pos > 0 && pos % kQuantTokens != 0 && seq_ids[row - 1] == seq && positions[row - 1] == pos - 1)) {
            continue; // no token, or not the first of its run
        }
        unsigned char *tile;
        if (pos < 0) {
            atomicOr(error_flag, kErrBadPosition);
            continue;
        }
        if (!quant_tile_of(kv, seq, pos / kQuantTokens, error_flag, tile)) {
            continue;
        }
        tile += int64_t(head) * kv.tile_bytes;
        const int slot = pos % kQuantTokens;
        const bool mine = lane < kQuantTokens - slot && row + lane < n_rows && seq_ids[row + lane] == seq && positions[row + lane] == pos + lane;
        const int run = __ffs(~__ballot_sync(0xffffffffu, mine)) - 1;

        const T *rows = (is_v ? v_rows : k_rows) + (int64_t(row) * kv.nkvh + head) * d;
        const int64_t row_step = int64_t(kv.nkvh) * d;
        float most = 0.f;
        bool finite = true;
        for (int r = 0; r < run; ++r) {
            for (int x = lane; x < d; x += 32) {
                const float a = fabsf(to_f32(rows[r * row_step + x]));
                finite &= a < INFINITY;
                most = fmaxf(most, a);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        }
        finite = __all_sync(0xffffffffu, finite);
        float *scale_at = reinterpret_cast<float *>(tile + quant_scales_at(d)) + (is_v ? 1 : 0);
        const float old = slot > 0 ? *scale_at : 0.f;
        finite &= !isnan(old);
        const float scale = finite ? fmaxf(fmaxf(old, most / kMost), kQuantFloor) : NAN, inverse = 1.f / scale;
        unsigned char *codes = tile + (is_v ? kQuantTokens * d : 0);
        if (scale > old) {
            const float factor = old * inverse;
            for (int r = 0; r < slot; ++r) {
                for (int x = lane; x < d; x += 32) {
                    unsigned char *c = codes + (is_v ? quant_v_at(r, x) : quant_k_at(r, x));
                    *c = quant_code<kF8>(quant_worth<kF8>(*c) * factor);
                }
            }
        }
        for (int r = 0; r < run; ++r) {
            for (int x = lane; x < d; x += 32) {
                codes[is_v ? quant_v_at(slot + r, x) : quant_k_at(slot + r, x)] =
                    quant_code<kF8>(finite ? to_f32(rows[r * row_step + x]) * inverse : 0.f);
            }
        }
        __syncwarp();
        if (lane == 0) {
            *scale_at = scale;
        }
    }
}

template <typename T, bool kF8>
__global__ void __launch_bounds__(128) quant_gather_kernel(QuantView kv, const int32_t *__restrict__ seq_ids,
                                                           const int32_t *__restrict__ positions, int32_t seq_row, int32_t n_rows,
                                                           T *__restrict__ k_out, T *__restrict__ v_out, int32_t *error_flag) {
    const int lane = threadIdx.x & 31, d = kv.d;
    const int64_t units = int64_t(n_rows) * kv.nkvh, warps = int64_t(gridDim.x) * 4;
    for (int64_t u = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5); u < units; u += warps) {
        const int32_t row = int32_t(u / kv.nkvh), head = int32_t(u - int64_t(row) * kv.nkvh);
        const int seq = seq_ids ? seq_ids[row] : seq_row, pos = seq_ids ? positions[row] : row;
        unsigned char *tile;
        if (pos < 0) {
            atomicOr(error_flag, kErrBadPosition);
            continue;
        }
        if (!quant_tile_of(kv, seq, pos / kQuantTokens, error_flag, tile)) {
            continue;
        }
        tile += int64_t(head) * kv.tile_bytes;
        const float *scales = reinterpret_cast<const float *>(tile + quant_scales_at(d));
        const int token = pos % kQuantTokens;
        for (int x = lane; x < d; x += 32) {
            k_out[u * d + x] = from_f32<T>(quant_worth<kF8>(tile[quant_k_at(token, x)]) * scales[0]);
            v_out[u * d + x] = from_f32<T>(quant_worth<kF8>(tile[kQuantTokens * d + quant_v_at(token, x)]) * scales[1]);
        }
    }
}

} // namespace

void quant_append(stream_t stream, llaisysDataType_t dtype, const QuantView &kv, const void *k_rows, const void *v_rows,
                  const int32_t *seq_ids, const int32_t *positions, int32_t n_rows, int32_t *error_flag) {
    const int64_t units = int64_t(n_rows) * 2 * kv.nkvh;
    const unsigned blocks = unsigned(std::min<int64_t>((units + 3) / 4, 1 << 20));
    dispatch(dtype, [&](auto t) {
        using T = decltype(t);
        auto kernel = kv.f8 ? quant_append_kernel<T, true> : quant_append_kernel<T, false>;
        kernel<<<blocks, 128, 0, static_cast<cudaStream_t>(stream)>>>(kv, static_cast<const T *>(k_rows), static_cast<const T *>(v_rows), seq_ids,
                                                                      positions, n_rows, error_flag);
    });
    check_launch("quant_append");
}

void quant_gather(stream_t stream, llaisysDataType_t dtype, const QuantView &kv, const int32_t *seq_ids, const int32_t *positions,
                  int32_t seq_row, int32_t n_rows, void *k_out, void *v_out, int32_t *error_flag) {
    const int64_t units = int64_t(n_rows) * kv.nkvh;
    const unsigned blocks = unsigned(std::min<int64_t>((units + 3) / 4, 1 << 20));
    dispatch(dtype, [&](auto t) {
        using T = decltype(t);
        auto kernel = kv.f8 ? quant_gather_kernel<T, true> : quant_gather_kernel<T, false>;
        kernel<<<blocks, 128, 0, static_cast<cudaStream_t>(stream)>>>(kv, seq_ids, positions, seq_row, n_rows, static_cast<T *>(k_out),
                                                                      static_cast<T *>(v_out), error_flag);
    });
    check_launch("quant_gather");
}

} // namespace llaisys::kernels
