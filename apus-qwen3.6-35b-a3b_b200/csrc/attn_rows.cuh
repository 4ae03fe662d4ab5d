/*
 * attn_rows.cuh — attention of one row and head by one warp, over packed keys: the plainest form of
 *     s_j = scale q . k_j,   p = softmax(s),   o = sum_j p_j v_j,   lse = log sum_j exp(s_j)
 * with a running maximum and sum.
 */
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "attn_view.cuh"
#include "common.cuh"
#include "kv_pages.cuh"

namespace apus {

struct AttnPacked {
    const uint16_t *k, *v;
    long k_stride, v_stride;
    const int32_t *cu_q, *cu_k;
    int rows, seqs, causal;
};

template <int D>
__global__ void __launch_bounds__(256)
attn_rows_kernel(AttnView a, AttnPacked pk) {
    pdl_enter();
    constexpr int N = D / 32;
    const int lane = threadIdx.x & 31;
    const long item = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (item >= (long)a.rows * a.heads) return;
    const int row = (int)(item / a.heads), h = (int)(item % a.heads), kh = h / a.group;
    int begin, count;
    {
        int lo = 0, hi = pk.seqs;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (pk.cu_q[mid + 1] <= row) lo = mid + 1;
            else hi = mid;
        }
        if (lo >= pk.seqs || row < pk.cu_q[lo]) return;
        begin = min(max(pk.cu_k[lo], 0), pk.rows);
        const int end = min(max(pk.cu_k[lo + 1], begin), pk.rows);
        count = end - begin;
        if (pk.causal) count = max(0, min(count, count - (pk.cu_q[lo + 1] - 1 - row)));
    }
    float q[N], o[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        q[i] = bf16_f32(a.q[row * a.q_stride + h * D + lane * N + i]) * a.scale;
        o[i] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int j = 0; j < count; j++) {
        const uint16_t *k = pk.k + (size_t)(begin + j) * pk.k_stride + kh * D;
        const uint16_t *v = pk.v + (size_t)(begin + j) * pk.v_stride + kh * D;
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) t = fmaf(q[i], bf16_f32(k[lane * N + i]), t);
        t = warp_sum(t);
        const float mn = fmaxf(m, t), c = expf(m - mn), e = expf(t - mn);
        m = mn;
        l = l * c + e;
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = fmaf(e, bf16_f32(v[lane * N + i]), o[i] * c);
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        float y = o[i] * inv;
        if (a.gate) y *= sigmoid_f32(bf16_f32(a.gate[row * a.gate_stride + h * D + lane * N + i]));
        a.out[row * a.out_stride + h * D + lane * N + i] = bf16_bits(y);
    }
    if (a.lse && lane == 0) a.lse[(size_t)row * a.heads + h] = l > 0.0f ? m + logf(l) : -INFINITY;
}

}  // namespace apus
