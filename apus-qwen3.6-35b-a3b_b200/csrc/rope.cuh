/*
 * rope.cuh — rotary positions of queries and keys on one or several axes (time, height, width),
 * with the rotated keys and the values written into the pages of a cache on the way.  (The
 * engine rotates one token's heads on the CPU with one axis, c/attn.h.)
 *
 *   pair i of a head (x_i, x_{i + r/2}), i < r/2, turns by  pos[axis(i)] * theta^(-2 i / r);
 *   what lies behind the first r values of a head is passed on.
 *
 * Bound: HBM (each vector read once, written once or twice).  The angles are the same for all
 * heads of a token, so a CTA takes a few tokens, finds their cosines and sines once (in turns,
 * reduced in 64 bits: at position 10^6 a 32-bit angle is off by 0.06) and keeps them in shared
 * memory.  A lane holds 16 bytes of a head; the other half of its pairs is in a lane r/16 away.
 */
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "kv_pages.cuh"

namespace apus {

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_MAX_PAIRS = 128;

struct RopeParams {
    const uint16_t *q, *k, *v;
    uint16_t *q_out, *k_out;
    long q_stride, k_stride, v_stride, q_out_stride, k_out_stride;
    int rows, heads, kv_heads, head_dim, rot;
    const int32_t *pos;                        /* [axes][rows] */
    const int32_t *slot;                       /* [rows] or null: no cache */
    uint16_t *cache_k, *cache_v;               /* of the layer */
    int page_tokens, pages;
    int32_t *status;
    int tokens;                                /* of a CTA */
    double turns[ROPE_MAX_PAIRS];              /* theta^(-2i/r) / 2 pi */
    unsigned char axis[ROPE_MAX_PAIRS];
};

__global__ void __launch_bounds__(ROPE_THREADS)
rope_kernel(const __grid_constant__ RopeParams p) {
    pdl_enter();
    extern __shared__ float2 rope_cs[];                  /* [tokens][rot / 2]: cos, sin */
    const int half = p.rot / 2, t0 = blockIdx.x * p.tokens;
    const int tokens = min(p.tokens, p.rows - t0);
    for (int i = threadIdx.x; i < tokens * half; i += ROPE_THREADS) {
        const int t = i / half, pair = i - t * half;
        const double x = (double)p.pos[(size_t)p.axis[pair] * p.rows + t0 + t] * p.turns[pair];
        float s, c;
        sincospif(2.0f * (float)(x - rint(x)), &s, &c);
        rope_cs[i] = make_float2(c, s);
    }
    __syncthreads();
    const int lanes = p.head_dim / 8;                    /* that share a head: 8, 16 or 32 */
    const int slots_of = 32 / lanes;                     /* heads of a warp at a time */
    const int lane = threadIdx.x & 31, sub = lane / lanes, c8 = lane % lanes;
    const int heads = p.heads + p.kv_heads + (p.slot ? p.kv_heads : 0);
    const int total = tokens * heads;
    const int step = (ROPE_THREADS / 32) * slots_of;
    const bool turned = c8 * 8 < p.rot, upper = c8 * 8 >= half;
    const int mate = turned ? (upper ? lane - half / 8 : lane + half / 8) : lane;
    const int pair0 = turned ? (upper ? c8 * 8 - half : c8 * 8) : 0;
    constexpr int U = 4;                                 /* vectors in flight a lane */
    for (int i0 = (threadIdx.x >> 5) * slots_of + sub; i0 - sub < total; i0 += step * U) {
        uint4 x[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u * step;
            x[u] = make_uint4(0, 0, 0, 0);
            if (i < total) {
                const int t = i / heads, h = i - t * heads;
                const size_t row = (size_t)(t0 + t);
                const uint16_t *from =
                    h < p.heads ? p.q + row * p.q_stride + (size_t)h * p.head_dim
                    : h < p.heads + p.kv_heads
                        ? p.k + row * p.k_stride + (size_t)(h - p.heads) * p.head_dim
                        : p.v + row * p.v_stride +
                              (size_t)(h - p.heads - p.kv_heads) * p.head_dim;
                x[u] = *reinterpret_cast<const uint4 *>(from + c8 * 8);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u * step;
            uint4 y;
            y.x = __shfl_sync(0xffffffffu, x[u].x, mate);
            y.y = __shfl_sync(0xffffffffu, x[u].y, mate);
            y.z = __shfl_sync(0xffffffffu, x[u].z, mate);
            y.w = __shfl_sync(0xffffffffu, x[u].w, mate);
            if (i >= total) continue;
            const int t = i / heads, h = i - t * heads;
            const size_t row = (size_t)(t0 + t);
            const bool is_v = h >= p.heads + p.kv_heads;
            if (turned && !is_v) {
                const float2 *cs = rope_cs + t * half + pair0;
                const uint32_t *a = &x[u].x, *b = &y.x;
                uint32_t r[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float2 c0 = cs[2 * j], c1 = cs[2 * j + 1];
                    const float s0 = upper ? c0.y : -c0.y, s1 = upper ? c1.y : -c1.y;
                    /* the one rounding: fp32 to BF16, once */
                    r[j] = pack_bf16_rn(fmaf(bf16lo(b[j]), s0, bf16lo(a[j]) * c0.x),
                                        fmaf(bf16hi(b[j]), s1, bf16hi(a[j]) * c1.x));
                }
                x[u] = make_uint4(r[0], r[1], r[2], r[3]);
            }
            if (h < p.heads) {
                *reinterpret_cast<uint4 *>(p.q_out + row * p.q_out_stride +
                                           (size_t)h * p.head_dim + c8 * 8) = x[u];
                continue;
            }
            const int kh = is_v ? h - p.heads - p.kv_heads : h - p.heads;
            if (!is_v && p.k_out)
                *reinterpret_cast<uint4 *>(p.k_out + row * p.k_out_stride +
                                           (size_t)kh * p.head_dim + c8 * 8) = x[u];
            if (p.slot) {
                const int at = p.slot[row];
                if (at < 0) continue;
                const int page = at / p.page_tokens;
                if (page >= p.pages) {
                    atomicCAS(p.status, 0, KV_BAD_PAGE);
                    continue;
                }
                const size_t to =
                    (((size_t)page * p.kv_heads + kh) * p.page_tokens + at % p.page_tokens) *
                        p.head_dim + c8 * 8;
                *reinterpret_cast<uint4 *>((is_v ? p.cache_v : p.cache_k) + to) = x[u];
            }
        }
    }
}

}  // namespace apus
