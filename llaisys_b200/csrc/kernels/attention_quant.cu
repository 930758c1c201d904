// Attention over a page pool held in 8 bits, one CTA of four warps per (query row, query head): keys are dealt to the lanes 32 at a time, a lane
// scores one key with the query in shared memory, a warp folds its scores into a running maximum and sum and adds the values with every
// lane owning every 32nd dim. Codes are multiplied as they are; a block's scale of K multiplies the score, that of V the weight.
#include "kernels.hpp"
#include "launch_utils.cuh"
#include "quant_tile.cuh"

namespace llaisys::kernels {

namespace {

constexpr int kWarps = 4, kMaxDimsPerLane = 8;

template <typename T, bool kF8>
__global__ void __launch_bounds__(kWarps * 32)
    attention_quant_kernel(QuantView kv, AttnBatch batch, const T *__restrict__ q, float scale, T *__restrict__ out, float *__restrict__ part,
                           const float *__restrict__ row_scale, int64_t out_stride, int32_t *error_flag) {
    __shared__ float q_s[256], acc_s[kWarps][256], m_s[kWarps], l_s[kWarps];
    const int d = kv.d, row = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int seq = row, t = 0, q_len = 1;
    if (batch.q_starts != nullptr) {
        int lo = 0, hi = batch.n_seqs - 1;
        while (lo < hi) { // last sequence with q_starts[seq] <= row
            const int mid = (lo + hi + 1) >> 1;
            if (batch.q_starts[mid] <= row) {
                lo = mid;
            } else {
                hi = mid - 1;
            }
        }
        seq = lo;
        t = row - batch.q_starts[seq];
        q_len = batch.q_starts[seq + 1] - batch.q_starts[seq];
        if (t < 0 || t >= q_len) {
            return; // behind the last sequence's rows
        }
    }
    const int kv_len = batch.kv_lens[seq], visible = max(0, min(kv_len, kv_len - q_len + t + 1));
    const int first = batch.window > 0 ? max(0, visible - batch.window) : 0, kept = min(batch.keep_first, first), gap = first - kept;
    const int seq_row = batch.seq_ids[seq], kvh = h / (batch.nh / kv.nkvh);
    const T *q_row = q + (int64_t(row) * batch.nh + h) * d;
    for (int i = threadIdx.x; i < d; i += blockDim.x) {
        q_s[i] = to_f32(q_row[i]) * scale;
    }
    __syncthreads();
    float m = -INFINITY, l = 0.f, acc[kMaxDimsPerLane] = {};
    const int n_keys = visible - gap;
    for (int base = warp * 32; base < n_keys; base += kWarps * 32) {
        const int j = base + lane + (base + lane >= kept ? gap : 0);
        unsigned char *tile = nullptr;
        const bool valid = base + lane < n_keys && quant_tile_of(kv, seq_row, j / kQuantTokens, error_flag, tile);
        const int token = j % kQuantTokens;
        float s = -INFINITY, v_scale = 0.f;
        if (valid) {
            tile += int64_t(kvh) * kv.tile_bytes;
            const float *scales = reinterpret_cast<const float *>(tile + quant_scales_at(d));
            float dot = 0.f;
            for (int i = 0; i < d; ++i) {
                dot = fmaf(q_s[i], quant_worth<kF8>(tile[quant_k_at(token, i)]), dot);
            }
            s = dot * scales[0];
            v_scale = scales[1];
        }
        float mx = s;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        }
        if (!__any_sync(0xffffffffu, s != -INFINITY)) {
            continue;
        }
        const float m_new = fmaxf(m, mx), alpha = expf(m - m_new), p = valid ? expf(s - m_new) : 0.f;
        float p_sum = p;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            p_sum += __shfl_xor_sync(0xffffffffu, p_sum, o);
        }
        l = l * alpha + p_sum;
        m = m_new;
#pragma unroll
        for (int i = 0; i < kMaxDimsPerLane; ++i) {
            acc[i] *= alpha;
        }
        const int n_here = min(32, n_keys - base);
        for (int jj = 0; jj < n_here; ++jj) {
            const float w = __shfl_sync(0xffffffffu, valid ? p * v_scale : 0.f, jj);
            const unsigned char *from = reinterpret_cast<const unsigned char *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(tile), jj));
            const int tok = __shfl_sync(0xffffffffu, token, jj);
            if (from == nullptr) {
                continue;
            }
#pragma unroll
            for (int i = 0; i < kMaxDimsPerLane; ++i) {
                const int dim = lane + 32 * i;
                if (dim < d) {
                    acc[i] = fmaf(w, quant_worth<kF8>(from[kQuantTokens * d + quant_v_at(tok, dim)]), acc[i]);
                }
            }
        }
    }
    if (lane == 0) {
        m_s[warp] = m;
        l_s[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < kMaxDimsPerLane; ++i) {
        acc_s[warp][lane + 32 * i] = acc[i];
    }
    __syncthreads();
    float m_all = -INFINITY, l_all = 0.f, share[kWarps];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        m_all = fmaxf(m_all, m_s[w]);
    }
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        share[w] = m_s[w] == -INFINITY ? (l_s[w] == 0.f ? 0.f : l_s[w]) : expf(m_s[w] - m_all);
        l_all += l_s[w] * share[w];
    }
    const float inv_l = l_all == 0.f ? 0.f : 1.f / l_all;
    const int64_t o_row = int64_t(row) * batch.nh + h;
    const float gate = row_scale != nullptr ? row_scale[o_row] : 1.f;
    for (int dim = threadIdx.x; dim < d; dim += blockDim.x) {
        float o = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            o += acc_s[w][dim] * share[w];
        }
        o *= inv_l;
        if (part != nullptr) {
            part[o_row * (d + 2) + dim] = o;
        } else {
            out[int64_t(row) * out_stride + int64_t(h) * d + dim] = from_f32<T>(o * gate);
        }
    }
    if (part != nullptr && threadIdx.x == 0) {
        part[o_row * (d + 2) + d] = m_all;
        part[o_row * (d + 2) + d + 1] = l_all;
    }
}

} // namespace

void attention_quant(stream_t stream, llaisysDataType_t dtype, const QuantView &kv, const AttnBatch &batch, const void *q, float scale,
                     const AttnOut &out, const AttnScratch &scratch) {
    CHECK_ARGUMENT(batch.nh <= 65535, "attention: too many heads for one launch");
    dispatch(dtype, [&](auto t) {
        using T = decltype(t);
        auto kernel = kv.f8 ? attention_quant_kernel<T, true> : attention_quant_kernel<T, false>;
        kernel<<<dim3(unsigned(batch.total_q), unsigned(batch.nh)), kWarps * 32, 0, static_cast<cudaStream_t>(stream)>>>(
            kv, batch, static_cast<const T *>(q), scale, static_cast<T *>(out.out), out.part, out.row_scale,
            out.row_stride ? out.row_stride : int64_t(batch.nh) * kv.d, scratch.error_flag);
    });
    check_launch("attention_quant");
}

} // namespace llaisys::kernels
