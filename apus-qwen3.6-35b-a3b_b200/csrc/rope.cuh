/*
 * rope.cuh — rotary positions of queries and keys on one or several axes (time, height, width),
 * with the rotated keys and the values written into the pages of a cache on the way.  (The
 * engine rotates one token's heads on the CPU with one axis, c/attn.h.)
 *
 *   pair i of a head (x_i, x_{i + r/2}), i < r/2, turns by  pos[axis(i)] * theta^(-2 i / r);
 *   what lies behind the first r values of a head is passed on.
 *
 * Bound: HBM (each vector read once, written once or twice).  The angles are the same for all
 * heads of a token, so a warp takes a token (or, with few tokens, several warps one): it asks for
 * its first vectors, finds the cosines and sines, a pair to a lane, while they are under way (in
 * turns, reduced in 64 bits: at position 10^6 a 32-bit angle is off by 0.06), and keeps those of
 * its lanes' values in registers.  A lane holds 16 bytes of a head; the other half of its pairs is
 * in a lane r/16 away.  6728 tokens of 16 + 2 + 2 heads of 256: 28 us, 145 MB at 5.2 TB/s.
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
    int split;                                 /* warps of a token */
    double turns[ROPE_MAX_PAIRS];              /* theta^(-2i/r) / 2 pi */
    unsigned char axis[ROPE_MAX_PAIRS];
};

template <int D>
__global__ void __launch_bounds__(ROPE_THREADS)
rope_kernel(const __grid_constant__ RopeParams p) {
    pdl_enter();
    constexpr int LANES = D / 8;                         /* that share a head: 8, 16 or 32 */
    constexpr int AT_ONCE = 32 / LANES;                  /* heads of a warp */
    constexpr int U = 8;                                 /* vectors under way a lane */
    __shared__ float2 angles[ROPE_THREADS / 32][ROPE_MAX_PAIRS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long unit = (long)blockIdx.x * (ROPE_THREADS / 32) + warp;
    const long row = unit / p.split;
    if (row >= p.rows) return;
    const int half = p.rot / 2, sub = lane / LANES, c8 = (lane % LANES) * 8;
    const int heads = p.heads + p.kv_heads + (p.slot ? p.kv_heads : 0);
    const int first = (int)(unit - row * p.split) * AT_ONCE + sub, step = p.split * AT_ONCE;
    const uint16_t *q = p.q + row * p.q_stride + c8, *k = p.k + row * p.k_stride + c8,
                   *v = p.v + row * p.v_stride + c8;
    auto load = [&](int h) {
        const uint16_t *from = h < p.heads                ? q + h * D
                               : h < p.heads + p.kv_heads ? k + (h - p.heads) * D
                                                          : v + (h - p.heads - p.kv_heads) * D;
        return *reinterpret_cast<const uint4 *>(from);
    };
    uint4 x[U];
#pragma unroll
    for (int u = 0; u < U; u++)
        x[u] = first + u * step < heads ? load(first + u * step) : make_uint4(0, 0, 0, 0);
    for (int i = lane; i < half; i += 32) {
        const double t = (double)p.pos[(size_t)p.axis[i] * p.rows + row] * p.turns[i];
        float s, c;
        sincospif(2.0f * (float)(t - rint(t)), &s, &c);
        angles[warp][i] = make_float2(c, s);
    }
    long place = -1;                                     /* in the cache, of head 0 */
    if (p.slot) {
        const int at = p.slot[row], page = at / p.page_tokens;
        if (at >= 0 && page < p.pages)
            place = ((long)page * p.kv_heads * p.page_tokens + at % p.page_tokens) * D + c8;
        else if (at >= 0 && lane == 0)
            atomicCAS(p.status, 0, KV_BAD_PAGE);
    }
    __syncwarp();
    const bool turned = c8 < p.rot, upper = c8 >= half;
    const int mate = turned ? (upper ? lane - half / 8 : lane + half / 8) : lane;
    float c[8], s[8];                                    /* of values that stay: 1 and 0 */
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float2 a = turned ? angles[warp][upper ? c8 - half + i : c8 + i]
                                : make_float2(1.0f, 0.0f);
        c[i] = a.x;
        s[i] = upper ? a.y : -a.y;
    }
    for (int h0 = first;; h0 += U * step) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int h = h0 + u * step;
            if (h - sub >= heads) break;                 /* (the same in all lanes) */
            uint4 y;
            y.x = __shfl_sync(0xffffffffu, x[u].x, mate);
            y.y = __shfl_sync(0xffffffffu, x[u].y, mate);
            y.z = __shfl_sync(0xffffffffu, x[u].z, mate);
            y.w = __shfl_sync(0xffffffffu, x[u].w, mate);
            if (h >= heads) continue;
            const bool is_v = h >= p.heads + p.kv_heads;
            uint4 r = x[u];
            if (turned && !is_v) {
                const uint32_t *a = &x[u].x, *b = &y.x;
                uint32_t *o = &r.x;
#pragma unroll
                for (int j = 0; j < 4; j++)              /* the one rounding: fp32 to BF16 */
                    o[j] = pack_bf16_rn(
                        fmaf(bf16lo(b[j]), s[2 * j], bf16lo(a[j]) * c[2 * j]),
                        fmaf(bf16hi(b[j]), s[2 * j + 1], bf16hi(a[j]) * c[2 * j + 1]));
            }
            if (h < p.heads) {
                *reinterpret_cast<uint4 *>(p.q_out + row * p.q_out_stride + h * D + c8) = r;
                continue;
            }
            const int kh = is_v ? h - p.heads - p.kv_heads : h - p.heads;
            if (!is_v && p.k_out)
                *reinterpret_cast<uint4 *>(p.k_out + row * p.k_out_stride + kh * D + c8) = r;
            if (place >= 0)
                *reinterpret_cast<uint4 *>((is_v ? p.cache_v : p.cache_k) + place +
                                           (long)kh * p.page_tokens * D) = r;
        }
        if (h0 - sub + U * step >= heads) break;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int h = h0 + (U + u) * step;
            if (h < heads) x[u] = load(h);
        }
        __syncwarp();
    }
}

}  // namespace apus
