/*
 * attn_decode.cuh — attention of one new token a sequence over the pages of a cache.
 *
 *   s_j = scale q . k_j over all tokens j of the sequence,  p = softmax(s),
 *   o = (sum_j p_j v_j) * sigmoid(gate),  lse = log sum_j exp(s_j)
 *
 * Bound: HBM, every key and value once: 4 * head_dim bytes a token and key head, against which
 * the products of its heads (at most 16 queries a key) are small.  So the work is split over
 * tokens, not heads: all sequences' tiles of 16 tokens form one line, (row, key head, tile), that
 * is cut into as many equal pieces as there are warps (eight to an SM), whatever the lengths are.  A
 * warp runs along its piece with a running maximum and sum, fed by a ring of its own in shared
 * memory that TMA fills (24 KB a warp, 192 KB an SM, of which about 44 KB in flight would cover the
 * latency), across the ends of sequences.  The heads of one key head are the rows (for the
 * scores) and the columns (for the outputs) of mma.sync tiles of 8: what tcgen05 would do with
 * 128 rows would be 8 or 16 rows here, and mma.sync needs a fifth of its rate to keep up with HBM.
 *
 *   scores   S[heads x 16 tokens] = Q . K^T       A: q in registers, B: ldmatrix of K
 *   outputs  O^T[D x heads] += V^T . P^T          A: ldmatrix.trans of V, B: the scores'
 *                                                 accumulators as they lie, narrowed to BF16
 *
 * (the operand's type beside V's; their sum keeps 32 bits.  Against 64 bits results are off by
 * 1.9e-3 to 2.3e-3 of their norm, 1.6e-3 of it the result's own narrowing.)
 *
 * A piece that holds a sequence's tokens only in part leaves (max, sum, outputs) behind: those of
 * one SM are put together in shared memory, those of several SMs by these SMs, each a share of
 * the values, as they arrive (a cooperative launch: all CTAs run at the same time, and a wait
 * has a limit); always in the same order, so that a result does not depend on timing.
 */
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "attn_tags.h"
#include "attn_view.cuh"
#include "common.cuh"
#include "kv_pages.cuh"
#include "prefill_gemm.cuh"

namespace apus {

constexpr int AD_WARPS = 8;
constexpr int AD_THREADS = AD_WARPS * 32;
constexpr int AD_TILE = 16;                  /* tokens */
constexpr int AD_MAX_ROWS = 1024;            /* of a launch */
constexpr int AD_RING_BYTES = 24 << 10;      /* of a warp */
constexpr int AD_SYNC_ROUND = 0, AD_SYNC_SEEN = 32, AD_SYNC_WORDS = 64;
constexpr int AD_MAX_GROUP = 16;
constexpr int AD_MAX_DIM = 256;
/* one unfinished result: outputs, four floats between heads (the accumulators' lanes then
 * write to 32 banks), then max and sum of each head */
constexpr int AD_PAD = 4;
constexpr int AD_PART_ML = AD_MAX_GROUP * (AD_MAX_DIM + AD_PAD);
constexpr int AD_PART_FLOATS = AD_PART_ML + 2 * AD_MAX_GROUP;

struct DecodeParams {
    AttnView a;
    const int32_t *table, *len, *seq;
    int32_t *status;                         /* the cache's */
    int *wait_status;                        /* the library's */
    int pages, page_tokens, page_tiles, seqs, max_pages, kv_heads;
    int row0, rows;                          /* of this launch */
    int absent;                              /* a CTA that asks for no tile (a test's), or -1 */
    uint2 *shared_parts;                     /* [gridDim][2]: began in an earlier CTA, or here */
    float *parts;                            /* [gridDim][warps]: ends in the warp, began before it */
    int blocks;                              /* CTAs that shared_parts has room for */
    unsigned *sync;                          /* the last round, CTAs that have seen its number */
};

/* a part as other SMs read it: every float beside the number of the round that wrote it, so that
 * it is its own flag (no fence, no second look): (value, round) words, outputs and then a
 * head's max and sum side by side (attn_tags.h: how a number comes again) */
constexpr int AD_SHARED_ML = AD_MAX_GROUP * AD_MAX_DIM;
constexpr int AD_SHARED_WORDS = AD_SHARED_ML + 2 * AD_MAX_GROUP;
inline size_t ad_scratch_bytes(int sms) {
    return (size_t)sms * (2 * AD_SHARED_WORDS * sizeof(uint2) +
                          AD_WARPS * AD_PART_FLOATS * sizeof(float));
}

template <int D>
struct AdShape {
    static constexpr int TILE_BYTES = AD_TILE * D * 2;
    static constexpr int STAGES = AD_RING_BYTES / TILE_BYTES;       /* 3, 6, 12 */
};

struct AdShared {
    long long start[AD_MAX_ROWS + 1];        /* tiles before a row */
    int seq[AD_MAX_ROWS], len[AD_MAX_ROWS];
    uint64_t full[AD_WARPS][12];
    int valid[AD_WARPS][12];                 /* tokens of a stage that count */
    float m[AD_WARPS][2][AD_MAX_GROUP], l[AD_WARPS][2][AD_MAX_GROUP];
    int item[AD_WARPS][2];
    long long scan[AD_WARPS];
    /* the items that parts are of: which parts (bit 2 warp + slot), row, key head, and where the
     * sum of them goes (0: out; else 1 + slot of shared_parts) */
    int items, same[2 * AD_WARPS], item_row[2 * AD_WARPS], item_head[2 * AD_WARPS],
        item_to[2 * AD_WARPS];
    int joint[2], joint_row[2], joint_head[2], joint_first[2];    /* CTAs that hold parts of it */
};
inline int ad_smem_bytes() { return AD_WARPS * AD_RING_BYTES + (int)sizeof(AdShared) + 1024; }

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, int x, int y,
                                            int z, uint64_t *bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::"
        "complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %5}], [%2], %6;" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z),
        "l"(policy)
        : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

/* where a warp is on the line */
struct AdCursor {
    int row, head, tile, tiles;              /* tiles: of the row */
    __device__ __forceinline__ void seek(const AdShared &s, int rows, int kv_heads,
                                         long long at) {
        int lo = 0, hi = rows;               /* the last row that starts at or before it */
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s.start[mid] * kv_heads <= at) lo = mid;
            else hi = mid;
        }
        row = lo;
        tiles = (int)(s.start[row + 1] - s.start[row]);
        const long long in = at - s.start[row] * kv_heads;
        head = 0;
        if (tiles) {                         /* in / tiles, without a 64-bit division */
            head = (int)((double)in / (double)tiles);
            if ((long long)head * tiles > in) head--;
            if ((long long)(head + 1) * tiles <= in) head++;
        }
        tile = tiles ? (int)(in - (long long)head * tiles) : 0;
    }
    __device__ __forceinline__ void next_item(const AdShared &s, int rows, int kv_heads) {
        tile = 0;
        if (++head < kv_heads) return;
        head = 0;
        do
            row++;
        while (row < rows && s.start[row + 1] == s.start[row]);
        tiles = row < rows ? (int)(s.start[row + 1] - s.start[row]) : 0;
    }
};

/* o narrowed once, the gate included (its sigmoid to a few 2^-23: no step of a BF16 result) */
__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float ad_gate(float g) {
    return rcp_fast(1.0f + exp2_fast(-LOG2E * g));
}
/* an 8 x 8 tile of 16-bit values, two to a lane, the other way round */
__device__ __forceinline__ uint32_t ad_transpose(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint2 ad_gate4(const AttnView &a, long row, int at) {
    return a.gate ? __ldg(reinterpret_cast<const uint2 *>(a.gate + row * a.gate_stride + at))
                  : make_uint2(0, 0);
}
/* (top, sum, acc) and another part's: both maxima may be of nothing */
__device__ __forceinline__ void ad_merge(float &top, float &sum, float4 &acc, float pm, float ps,
                                         float4 v) {
    const float t = fmaxf(top, pm), base = t == -INFINITY ? 0.0f : t;
    const float a = exp2_fast(top - base), b = exp2_fast(pm - base);
    top = t;
    sum = a * sum + b * ps;
    acc.x = a * acc.x + b * v.x;
    acc.y = a * acc.y + b * v.y;
    acc.z = a * acc.z + b * v.z;
    acc.w = a * acc.w + b * v.w;
}
/* four values of a head's sums as they leave */
__device__ __forceinline__ void ad_finish4(const AttnView &a, long row, int head, int D, int c,
                                           float4 y, float top, float sum, uint2 gate) {
    const float inv = sum == 0.0f ? 0.0f : __fdividef(1.0f, sum);
    y.x *= inv;
    y.y *= inv;
    y.z *= inv;
    y.w *= inv;
    if (a.gate) {
        y.x *= ad_gate(bf16lo(gate.x));
        y.y *= ad_gate(bf16hi(gate.x));
        y.z *= ad_gate(bf16lo(gate.y));
        y.w *= ad_gate(bf16hi(gate.y));
    }
    if (sum == 0.0f) y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);     /* no key, whatever the gate is */
    *reinterpret_cast<uint2 *>(a.out + row * a.out_stride + head * D + c) =
        make_uint2(pack_bf16_rn(y.x, y.y), pack_bf16_rn(y.z, y.w));
    if (c == 0 && a.lse)
        a.lse[row * a.heads + head] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * LN2;
}
/* Two such words.  Of a vector access each element is whole, not the vector: a value and its round
 * are the halves of one 64-bit element, so that none is seen without the other. */
__device__ __forceinline__ void ad_put2(uint2 *at, float x, float y, unsigned round) {
    const uint64_t tag = (uint64_t)round << 32;
    asm volatile("st.relaxed.gpu.global.v2.b64 [%0], {%1, %2};" ::"l"(at),
                 "l"(tag | __float_as_uint(x)), "l"(tag | __float_as_uint(y))
                 : "memory");
}
__device__ __forceinline__ uint4 ad_look2(const uint2 *at) {
    uint64_t a, b;
    asm volatile("ld.relaxed.gpu.global.v2.b64 {%0, %1}, [%2];" : "=l"(a), "=l"(b)
                 : "l"(at)
                 : "memory");
    return make_uint4((uint32_t)a, (uint32_t)(a >> 32), (uint32_t)b, (uint32_t)(b >> 32));
}
/* A copy's barrier by a whole warp, with one answer: lanes that went on alone would wait for the others
 * in the next shuffle or MMA for good. */
__device__ __forceinline__ bool ad_wait(uint64_t *bar, uint32_t parity) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    return __all_sync(0xffffffffu, mbar_wait(bar, parity)) != 0;
}
/* Four values and a head's max and sum, looked at once already: again until they are this
 * round's, for about a second at most (a look is an L2 round trip, four times a barrier's). */
__device__ __forceinline__ bool ad_get(const uint2 *at, const uint2 *at_ml, unsigned round,
                                       uint4 &a, uint4 &b, uint4 &ml) {
    for (uint32_t i = 0; i < APUS_WAIT_LIMIT / 4; i++) {
        if (a.y == round && a.w == round && b.y == round && b.w == round && ml.y == round &&
            ml.w == round)
            return true;
        a = ad_look2(at);
        b = ad_look2(at + 2);
        ml = ad_look2(at_ml);
        if (i > 64) __nanosleep(64);
    }
    return false;
}
/* place / per (per > 0) */
__device__ __forceinline__ int ad_piece_of(long long place, long long per) {
    if (place < 0x40000000) return (int)((unsigned)place / (unsigned)min(per, 0x7fffffffLL));
    return (int)(place / per);
}

template <int D, int NH>
__global__ void __launch_bounds__(AD_THREADS, 1)
attn_decode_kernel(const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v,
                   const __grid_constant__ DecodeParams p) {
    constexpr int STAGES = AdShape<D>::STAGES, TILE_BYTES = AdShape<D>::TILE_BYTES;
    constexpr int MT = D / 16;                            /* row tiles of O^T, steps of Q . K^T */
    constexpr int NT = NH / 8;                            /* column tiles of O^T */
    extern __shared__ unsigned char ad_raw[];
    unsigned char *ring0 = reinterpret_cast<unsigned char *>(
        (reinterpret_cast<uintptr_t>(ad_raw) + 1023) & ~(uintptr_t)1023);
    AdShared &s = *reinterpret_cast<AdShared *>(ring0 + AD_WARPS * AD_RING_BYTES);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const int group = p.a.group;
    if (lane == 0) {
        for (int i = 0; i < STAGES; i++) mbar_init(&s.full[warp][i], 1);
        mbar_fence_init();
    }
    pdl_enter();
    /* this round's number: no word holds it yet */
    const unsigned round =
        ad_round_after(*reinterpret_cast<volatile unsigned *>(p.sync + AD_SYNC_ROUND));
    /* (this CTA's own words, before it writes any, and those of CTAs that there are not) */
    if (ad_round_clears(round))
        for (int b = blockIdx.x; b < p.blocks; b += gridDim.x)
            for (int i = tid; i < AD_SHARED_WORDS; i += AD_THREADS)
                ad_put2(p.shared_parts + (size_t)b * 2 * AD_SHARED_WORDS + 2 * i, 0.0f, 0.0f, 0);

    /* ---- the line: tiles before every row (each CTA for itself) ---- */
    {
        constexpr int PER = AD_MAX_ROWS / AD_THREADS;
        long long mine[PER], sum = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int r = tid * PER + i;
            int q = -1, n = 0;
            if (r < p.rows) {
                q = p.seq ? p.seq[p.row0 + r] : p.row0 + r;
                if (q >= p.seqs) {
                    if (blockIdx.x == 0) atomicCAS(p.status, 0, KV_BAD_LIST);
                    q = -1;
                }
                if (q >= 0) n = min(max(p.len[q], 0), p.max_pages * p.page_tokens);
                s.seq[r] = q;
                s.len[r] = n;
            }
            mine[i] = sum;
            sum += (n + AD_TILE - 1) / AD_TILE;
        }
        long long x = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) s.scan[warp] = x;
        __syncthreads();
        long long before = x - sum;
        for (int w = 0; w < warp; w++) before += s.scan[w];
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (tid * PER + i <= p.rows) s.start[tid * PER + i] = before + mine[i];
        if (tid == AD_THREADS - 1 && p.rows == AD_MAX_ROWS) s.start[p.rows] = before + sum;
        if (tid < 2 * AD_WARPS) s.item[tid >> 1][tid & 1] = -1;
    }
    __syncthreads();
    /* all of this CTA has the round's number; the CTA that is last in this makes the next one */
    unsigned seen = 0;
    if (tid == 0) seen = atomicInc(p.sync + AD_SYNC_SEEN, gridDim.x - 1);
    const long long total = s.start[p.rows] * p.kv_heads;
    long long per = total < 0x40000000 ? ((unsigned)total + gridDim.x - 1) / gridDim.x
                                       : (total + gridDim.x - 1) / gridDim.x;
    if (per < AD_WARPS) per = AD_WARPS;                   /* one tile to a warp */
    const long long lo = min(total, per * blockIdx.x), hi = min(total, lo + per);
    const long long from = lo + (hi - lo) * warp / AD_WARPS,
                    to = lo + (hi - lo) * (warp + 1) / AD_WARPS;

    /* rows of no token: zeros */
    for (int r = blockIdx.x; r < p.rows; r += gridDim.x) {
        if (s.seq[r] < 0 || s.len[r] > 0) continue;
        const long row = p.row0 + r;
        for (int i = tid; i < p.a.heads * D; i += AD_THREADS)
            p.a.out[row * p.a.out_stride + i] = 0;
        if (p.a.lse)
            for (int h = tid; h < p.a.heads; h += AD_THREADS)
                p.a.lse[row * p.a.heads + h] = -INFINITY;
    }

    /* ---- the warp's piece ---- */
    const uint32_t ring = smem_u32(ring0) + warp * AD_RING_BYTES;
    const float sc = p.a.scale * LOG2E;
    const uint64_t policy = l2_read_once();
    bool alive = true;
    float o[NT][MT][4], m[NT], l[NT];
    uint32_t qa[MT][NT * 2];
    long long issued = from, done = from;                 /* tiles asked for, tiles summed */
    AdCursor ci, cc;
    ci.seek(s, p.rows, p.kv_heads, from);
    cc = ci;
    /* copies: the keys of tile i are copy 2i, its values 2i + 1, each into stage copy % STAGES */
    uint32_t copies = 0, used = 0;
    int page_row = -1, page_base = 0, page_lane = 0;      /* pages of 32 tiles, one to a lane */
    int coord = 0, count = 0;
    auto issue = [&]() {
        const int st = (int)(copies % STAGES);
        const bool keys = !(copies & 1);
        if (keys) {
            if (page_row != ci.row || ci.tile < page_base || ci.tile >= page_base + 32) {
                page_row = ci.row;
                page_base = ci.tile;
                const int tile = page_base + lane;
                page_lane = tile < ci.tiles ? p.table[(size_t)s.seq[ci.row] * p.max_pages +
                                                      (unsigned)tile / (unsigned)p.page_tiles]
                                            : 0;
            }
            int page = __shfl_sync(0xffffffffu, page_lane, ci.tile - page_base);
            count = min(AD_TILE, s.len[ci.row] - ci.tile * AD_TILE);
            if ((unsigned)page >= (unsigned)p.pages) {
                if (lane == 0) atomicCAS(p.status, 0, KV_BAD_PAGE);
                page = 0;
                count = 0;
            }
            coord = (page * p.kv_heads + ci.head) * p.page_tokens +
                    (int)((unsigned)ci.tile % (unsigned)p.page_tiles) * AD_TILE;
        }
        if (lane == 0 && (int)blockIdx.x != p.absent) {
            s.valid[warp][st] = count;
            mbar_expect_tx(&s.full[warp][st], TILE_BYTES);
            tma_load_3d(ring + st * TILE_BYTES, keys ? &map_k : &map_v, 0, coord, 0,
                        &s.full[warp][st], policy);
        }
        copies++;
        if (!keys) {
            issued++;
            if (++ci.tile == ci.tiles) ci.next_item(s, p.rows, p.kv_heads);
        }
    };
    while (copies < STAGES && issued < to) issue();

    auto begin = [&]() {                                  /* q of the item's heads, nothing summed */
        const long row = p.row0 + cc.row;
        const uint16_t *q = p.a.q + row * p.a.q_stride + (size_t)cc.head * group * D;
#pragma unroll
        for (int k = 0; k < MT; k++)
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 2; j++)
                    qa[k][n * 2 + j] =
                        g + 8 * n < group ? *reinterpret_cast<const uint32_t *>(
                                                q + (g + 8 * n) * D + k * 16 + j * 8 + t4 * 2)
                                          : 0u;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            m[n] = -INFINITY;
            l[n] = 0.0f;
#pragma unroll
            for (int k = 0; k < MT; k++)
#pragma unroll
                for (int j = 0; j < 4; j++) o[n][k][j] = 0.0f;
        }
    };
    auto leave_top = [&](int slot) {
        if (t4 == 0)
#pragma unroll
            for (int n = 0; n < NT; n++) {
                s.m[warp][slot][n * 8 + g] = m[n];
                s.l[warp][slot][n * 8 + g] = l[n];
            }
    };
    /* an unfinished result in fp32, times a factor for each head */
    auto leave = [&](float *dst, const float (&f)[NT][2]) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int h = n * 8 + t4 * 2 + (j & 1);
                if (h < group)
#pragma unroll
                    for (int k = 0; k < MT; k++)
                        dst[h * (D + AD_PAD) + k * 16 + (j >> 1) * 8 + g] =
                            o[n][k][j] * f[n][j & 1];
            }
    };
    const size_t warp_part = (size_t)(blockIdx.x * AD_WARPS + warp) * AD_PART_FLOATS;
    bool first = cc.tile > 0;              /* the item began before this piece */
    if (from < to) begin();
    while (alive && done < to) {
        /* ---- scores of 16 tokens ---- */
        int st = (int)(used % STAGES);
        if (!ad_wait(&s.full[warp][st], (used / STAGES) & 1u)) {
            alive = false;
            break;
        }
        const int valid = s.valid[warp][st];
        float sc0[NT][2], sc1[NT][2];                     /* [head tile][token pair] by token tile */
        {
            float c[2][4] = {};
            const uint32_t base = ring + st * TILE_BYTES;
            const int tok = (lane & 7) + (lane >> 4) * 8, ch = (lane >> 3) & 1;
#pragma unroll
            for (int k = 0; k < MT; k++) {
                uint32_t b[4];
                const int chunk = (2 * k + ch) & 7;
                ldmatrix_x4(b, base + (k >> 2) * (AD_TILE * 128) + tok * 128 +
                                   ((chunk ^ (tok & 7)) << 4));
                const uint32_t a[4] = {qa[k][0], NT > 1 ? qa[k][2 * (NT - 1)] : 0u, qa[k][1],
                                       NT > 1 ? qa[k][2 * (NT - 1) + 1] : 0u};
                mma_16x8(c[0], a, b[0], b[1]);
                mma_16x8(c[1], a, b[2], b[3]);
            }
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    sc0[n][j] = t4 * 2 + j < valid ? c[0][n * 2 + j] * sc : -INFINITY;
                    sc1[n][j] = 8 + t4 * 2 + j < valid ? c[1][n * 2 + j] * sc : -INFINITY;
                }
        }
        used++;
        __syncwarp();
        if (issued < to) issue();
        /* ---- running maximum; what has been summed is scaled down only where the maximum
         * has moved by more than 2^8, which fp32 sums and BF16 weights of any size bear ---- */
        float f[NT];
        bool moved = false;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float x = fmaxf(fmaxf(sc0[n][0], sc0[n][1]), fmaxf(sc1[n][0], sc1[n][1]));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
            f[n] = 1.0f;
            if (x > m[n] + 8.0f || (m[n] == -INFINITY && x > -INFINITY)) {
                moved |= m[n] > -INFINITY;               /* (else there is nothing to scale) */
                f[n] = exp2_fast(m[n] - x);
                m[n] = x;
                l[n] *= f[n];
            }
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const float f0 = __shfl_sync(0xffffffffu, f[n], t4 * 8),
                            f1 = __shfl_sync(0xffffffffu, f[n], t4 * 8 + 4);
#pragma unroll
                for (int k = 0; k < MT; k++) {
                    o[n][k][0] *= f0;
                    o[n][k][1] *= f1;
                    o[n][k][2] *= f0;
                    o[n][k][3] *= f1;
                }
            }
        }
        uint32_t pb[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const float mm = m[n] == -INFINITY ? 0.0f : m[n];
            const float p0 = exp2_fast(sc0[n][0] - mm), p1 = exp2_fast(sc0[n][1] - mm),
                        p2 = exp2_fast(sc1[n][0] - mm), p3 = exp2_fast(sc1[n][1] - mm);
            l[n] += (p0 + p1) + (p2 + p3);
            pb[n][0] = pack_bf16_rn(p0, p1);
            pb[n][1] = pack_bf16_rn(p2, p3);
        }
        /* ---- outputs ---- */
        st = (int)(used % STAGES);
        if (!ad_wait(&s.full[warp][st], (used / STAGES) & 1u)) {
            alive = false;
            break;
        }
        {
            const uint32_t base = ring + st * TILE_BYTES;
            const int tok = (lane & 7) + (lane >> 4) * 8, ch = (lane >> 3) & 1;
            /* values of tokens that do not count may be anything: 0 * NaN is not 0 */
            const uint32_t keep0 = (t4 * 2 < valid ? 0xffffu : 0u) |
                                   (t4 * 2 + 1 < valid ? 0xffff0000u : 0u),
                           keep1 = (8 + t4 * 2 < valid ? 0xffffu : 0u) |
                                   (8 + t4 * 2 + 1 < valid ? 0xffff0000u : 0u);
#pragma unroll
            for (int k = 0; k < MT; k++) {
                uint32_t a[4];
                const int chunk = (2 * k + ch) & 7;
                ldmatrix_x4_trans(a, base + (k >> 2) * (AD_TILE * 128) + tok * 128 +
                                         ((chunk ^ (tok & 7)) << 4));
                a[0] &= keep0;
                a[1] &= keep0;
                a[2] &= keep1;
                a[3] &= keep1;
#pragma unroll
                for (int n = 0; n < NT; n++) mma_16x8(o[n][k], a, pb[n][0], pb[n][1]);
            }
        }
        used++;
        __syncwarp();
        if (issued < to) issue();
        done++;
        const bool ends = ++cc.tile == cc.tiles;
        if (!ends && done < to) continue;
        /* ---- the end of the item or of the piece ---- */
#pragma unroll
        for (int n = 0; n < NT; n++) {
            l[n] += __shfl_xor_sync(0xffffffffu, l[n], 1);
            l[n] += __shfl_xor_sync(0xffffffffu, l[n], 2);
        }
        const int item = cc.row * p.kv_heads + cc.head;
        if (ends && !first) {                             /* all of it was here */
            const long row = p.row0 + cc.row;
            const int h0 = cc.head * group;
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const float inv = l[n] == 0.0f ? 0.0f : __fdividef(1.0f, l[n]);
                if (p.a.lse && t4 == 0 && n * 8 + g < group)
                    p.a.lse[row * p.a.heads + h0 + n * 8 + g] =
                        l[n] == 0.0f ? -INFINITY : (m[n] + log2f(l[n])) * LN2;
                const float v0 = __shfl_sync(0xffffffffu, inv, t4 * 8),
                            v1 = __shfl_sync(0xffffffffu, inv, t4 * 8 + 4);
                /* the accumulators hold (value g; heads 2 t, 2 t + 1); memory wants (head g;
                 * values 2 t, 2 t + 1): 8 x 8 transposes, of the gate on its way in */
                const int at = (h0 + n * 8 + g) * D + t4 * 2;
                const bool there = n * 8 + g < group;
                uint32_t gt[2 * MT];
                if (p.a.gate)
#pragma unroll
                    for (int k = 0; k < 2 * MT; k++)
                        gt[k] = there ? __ldg(reinterpret_cast<const uint32_t *>(
                                            p.a.gate + row * p.a.gate_stride + at + k * 8))
                                      : 0u;
#pragma unroll
                for (int k = 0; k < 2 * MT; k++) {
                    float y0 = o[n][k >> 1][(k & 1) * 2] * v0,
                          y1 = o[n][k >> 1][(k & 1) * 2 + 1] * v1;
                    if (p.a.gate) {
                        const uint32_t x = ad_transpose(gt[k]);
                        /* (no key: zero, whatever the gate is) */
                        y0 = v0 == 0.0f ? 0.0f : y0 * ad_gate(bf16lo(x));
                        y1 = v1 == 0.0f ? 0.0f : y1 * ad_gate(bf16hi(x));
                    }
                    const uint32_t y = ad_transpose(pack_bf16_rn(y0, y1));
                    if (there)
                        *reinterpret_cast<uint32_t *>(p.a.out + row * p.a.out_stride + at +
                                                      k * 8) = y;
                }
            }
        } else if (done == to) {                          /* kept until all is through */
            leave_top(1);
            if (lane == 0) s.item[warp][1] = item;
        } else {                                          /* out of the way of what comes */
            float one[NT][2];
#pragma unroll
            for (int n = 0; n < NT; n++) one[n][0] = one[n][1] = 1.0f;
            leave(p.parts + warp_part, one);
            leave_top(0);
            if (lane == 0) s.item[warp][0] = item;
        }
        first = false;
        if (done < to) {
            cc.next_item(s, p.rows, p.kv_heads);
            begin();
        }
    }
    if (!alive) {                                         /* a copy never came: no result, no hang */
        if (lane == 0) set_status(p.wait_status, ST_MBAR_TIMEOUT);
        /* what is under way lands before the CTA leaves (one more limit, not one for each) */
        while (used < copies && ad_wait(&s.full[warp][used % STAGES], (used / STAGES) & 1u)) used++;
    }
    __syncthreads();                                      /* every ring is read to its end */

    /* ---- the SM's unfinished results, put together in the order of the line ----
     * What this takes is mostly instructions that run once, out of L2 at 8 cycles each: few of
     * them, and nothing that an earlier step can say. */
    constexpr int ENTRIES = 2 * AD_WARPS;
    if (tid < 2) s.joint[tid] = 0;
    __syncwarp();
    if (tid < ENTRIES) {                                  /* an entry to a lane */
        const int item = s.item[tid >> 1][tid & 1];
        const unsigned same = __match_any_sync(0xffffu, item);
        const bool leads = item >= 0 && __ffs(same) - 1 == tid;
        const unsigned leaders = __ballot_sync(0xffffu, leads);
        if (tid == 0) s.items = __popc(leaders);
        if (leads) {
            const int i = __popc(leaders & ((1u << tid) - 1));
            const int row = item / p.kv_heads, head = item - row * p.kv_heads;
            const long long tiles = s.start[row + 1] - s.start[row],
                            begin = s.start[row] * p.kv_heads + head * tiles;
            const bool before = begin < lo, after = begin + tiles > hi;
            s.same[i] = same;
            s.item_row[i] = row;
            s.item_head[i] = head;
            s.item_to[i] = before ? 1 : after ? 2 : 0;
            if (before || after) {
                const int j = !before, c0 = ad_piece_of(begin, per);
                s.joint_first[j] = c0;
                s.joint[j] = ad_piece_of(begin + tiles - 1, per) - c0 + 1;
                s.joint_row[j] = row;
                s.joint_head[j] = head;
            }
        }
    }
    const int mine = s.item[warp][1];
    if (mine >= 0) {                                      /* in the ring, against the item's maximum */
        float f[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int h = n * 8 + t4 * 2 + j;
                float top = -INFINITY;
#pragma unroll
                for (int e = 0; e < ENTRIES; e++)
                    if (s.item[e >> 1][e & 1] == mine) top = fmaxf(top, s.m[e >> 1][e & 1][h]);
                f[n][j] = exp2_fast(s.m[warp][1][h] - (top == -INFINITY ? 0.0f : top));
            }
        leave(reinterpret_cast<float *>(ring0 + warp * AD_RING_BYTES), f);
    }
    __syncthreads();
    constexpr int HEAD4 = D / 4;                          /* pieces of 16 bytes of a head */
    const int per_item = group * HEAD4, pieces_here = s.items * per_item;
#pragma unroll 1
    for (int x = tid; x < pieces_here; x += AD_THREADS) {
        int i = 0, in = x;
        for (; in >= per_item; in -= per_item) i++;
        const int h = in / HEAD4, c = (in - h * HEAD4) * 4, at = h * (D + AD_PAD) + c;
        const unsigned same = s.same[i];
        float4 v[AD_WARPS], acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < AD_WARPS; w++) {
            const bool of = same >> (2 * w + 1) & 1;
            v[w] = of ? *reinterpret_cast<const float4 *>(ring0 + w * AD_RING_BYTES + at * 4)
                      : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (of) top = fmaxf(top, s.m[w][1][h]);
        }
        for (unsigned b = same & 0x5555u; b; b &= b - 1)
            top = fmaxf(top, s.m[(__ffs(b) - 1) >> 1][0][h]);
        const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int w = 0; w < AD_WARPS; w++) {
            if (same >> (2 * w + 1) & 1) sum = fmaf(exp2_fast(s.m[w][1][h] - base), s.l[w][1][h], sum);
            acc.x += v[w].x;
            acc.y += v[w].y;
            acc.z += v[w].z;
            acc.w += v[w].w;
        }
        for (unsigned b = same & 0x5555u; b; b &= b - 1) {        /* what ended in a warp */
            const int w = (__ffs(b) - 1) >> 1;
            const float f = exp2_fast(s.m[w][0][h] - base);
            const float4 y = *reinterpret_cast<const float4 *>(
                p.parts + (size_t)(blockIdx.x * AD_WARPS + w) * AD_PART_FLOATS + at);
            sum = fmaf(f, s.l[w][0][h], sum);
            acc.x = fmaf(f, y.x, acc.x);
            acc.y = fmaf(f, y.y, acc.y);
            acc.z = fmaf(f, y.z, acc.z);
            acc.w = fmaf(f, y.w, acc.w);
        }
        const int dest = s.item_to[i];
        if (dest) {
            uint2 *part = p.shared_parts + (size_t)(blockIdx.x * 2 + dest - 1) * AD_SHARED_WORDS;
            ad_put2(part + h * D + c, acc.x, acc.y, round);
            ad_put2(part + h * D + c + 2, acc.z, acc.w, round);
            if (c == 0) ad_put2(part + AD_SHARED_ML + 2 * h, top, sum, round);
        } else {
            const long row = p.row0 + s.item_row[i];
            const int head = s.item_head[i] * group + h;
            ad_finish4(p.a, row, head, D, c, acc, top, sum, ad_gate4(p.a, row, head * D + c));
        }
    }

    /* ---- items that several SMs hold parts of ---- */
    bool gone = false;                                    /* a part never came: ask for no other */
#pragma unroll 1
    for (int j = 0; j < 2; j++) {
        const int n = s.joint[j], c0 = s.joint_first[j];
        if (!n) continue;
        const long row = p.row0 + s.joint_row[j];
        /* every SM that holds a part adds up a share of the pieces: a few lanes to a piece, each
         * some of the parts, then the lanes by shuffles */
        const int share = (per_item + n - 1) / n, first_piece = share * ((int)blockIdx.x - c0);
        const int pieces = min(share, per_item - first_piece);
        if (pieces <= 0) continue;
        int lanes = 32;
        while (lanes > 1 && lanes * pieces > AD_THREADS) lanes >>= 1;
        const int sub = tid & (lanes - 1);
#pragma unroll 1
        for (int x0 = tid / lanes; x0 - tid / lanes < pieces; x0 += AD_THREADS / lanes) {
            const bool real = x0 < pieces;
            const int in = first_piece + (real ? x0 : 0), h = in / HEAD4, c = (in - h * HEAD4) * 4;
            const int head = s.joint_head[j] * group + h;
            const uint2 gate = ad_gate4(p.a, row, head * D + c);      /* beside the wait */
            float top = -INFINITY, sum = 0.0f;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
            for (int e0 = sub; e0 < n && !gone; e0 += 2 * lanes) {
                uint4 a[2], b[2], ml[2];
#pragma unroll
                for (int k = 0; k < 2; k++) {             /* both under way before one is waited for */
                    const int e = min(e0 + k * lanes, n - 1);
                    const uint2 *part =
                        p.shared_parts + (size_t)((c0 + e) * 2 + (e == 0)) * AD_SHARED_WORDS;
                    a[k] = ad_look2(part + h * D + c);
                    b[k] = ad_look2(part + h * D + c + 2);
                    ml[k] = ad_look2(part + AD_SHARED_ML + 2 * h);
                }
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const int e = e0 + k * lanes;
                    if (e >= n || gone) continue;
                    const uint2 *part =
                        p.shared_parts + (size_t)((c0 + e) * 2 + (e == 0)) * AD_SHARED_WORDS;
                    if (!ad_get(part + h * D + c, part + AD_SHARED_ML + 2 * h, round, a[k], b[k],
                                ml[k])) {
                        set_status(p.wait_status, ST_SCHED_TIMEOUT);
                        gone = true;
                        continue;
                    }
                    ad_merge(top, sum, acc, __uint_as_float(ml[k].x), __uint_as_float(ml[k].z),
                             make_float4(__uint_as_float(a[k].x), __uint_as_float(a[k].z),
                                         __uint_as_float(b[k].x), __uint_as_float(b[k].z)));
                }
            }
            for (int o = 1; o < lanes; o <<= 1) {
                float4 v;
                const float pm = __shfl_xor_sync(0xffffffffu, top, o),
                            ps = __shfl_xor_sync(0xffffffffu, sum, o);
                v.x = __shfl_xor_sync(0xffffffffu, acc.x, o);
                v.y = __shfl_xor_sync(0xffffffffu, acc.y, o);
                v.z = __shfl_xor_sync(0xffffffffu, acc.z, o);
                v.w = __shfl_xor_sync(0xffffffffu, acc.w, o);
                ad_merge(top, sum, acc, pm, ps, v);
            }
            if (real && sub == 0) ad_finish4(p.a, row, head, D, c, acc, top, sum, gate);
        }
    }
    if (tid == 0 && seen == gridDim.x - 1) atomicExch(p.sync + AD_SYNC_ROUND, round);
}

}  // namespace apus
