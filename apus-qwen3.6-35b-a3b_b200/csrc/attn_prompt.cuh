/*
 * attn_prompt.cuh — attention of packed prompts on the 5th-generation tensor cores.
 *
 *   S = Q K^T,  p = exp2(scale log2(e) (S - m)) over the keys that a row sees,
 *   O = P V / sum(p) * sigmoid(gate),  lse = log sum exp(scale S)
 *
 * One pass over the keys with a running maximum and sum.  The heads of a key head are rows: a
 * tile of 128 rows is 128 / group tokens times the group's heads, so that short prompts fill it,
 * every key is fetched once for all its heads, and the causal edge costs few masked scores.
 *
 * One persistent CTA per SM takes such tiles from a counter, the last sequence first and of each
 * the last tiles first, which see most of its keys.  Its warps:
 *   warp 0     finds the tile's sequence, loads Q (64 KB at head_dim 256) and a ring of 32 KB
 *              pieces of K and V
 *   warp 1     issues tcgen05.mma: S(j+1) before O += P(j) V(j), so that the tensor cores work
 *              while the softmax of a step of 128 keys runs
 *   warps 4-11 softmax, two warps to each quarter of the rows with half of the 128 scores each;
 *              outputs at the end
 * S is double-buffered in tensor memory (2 x 128 columns), O takes head_dim columns.  P stays
 * there as well: narrowed to BF16 it overwrites its own scores and is the MMA's A operand, so that
 * shared memory carries Q, K and V only.  (K and Q are K-major; V's rows are its K dimension: the
 * MN-major form of the same 128B-swizzled tile.)  MMAs of one issuer run in the order of their
 * issue: S(j+2) may overwrite the P(j) that the product before it reads.  BF16 because that is what
 * the MMA takes beside V (its form of 19 bits runs at half the rate, with V widened).  The sum that
 * divides keeps the weights' 32 bits.  Against 64 bits results are off by 1.9e-3 to 2.3e-3 of their
 * norm; with 32-bit weights it is 1.7e-3, which is the result's own narrowing.
 *
 * The maximum that a row's weights are taken against moves only when a score is 2^8 above it: any
 * reference within the range of fp32 and BF16 gives the same quotient, and O in tensor memory
 * is then hardly ever scaled again (that takes its columns through registers).
 *
 * Few rows and many keys (the next part of a prompt behind a long one) would leave most SMs
 * idle: then several CTAs share a tile's keys, leave their sums in fp32 and a second kernel
 * adds them up in order.
 *
 * Bound at head_dim 256 and long prompts: shared memory (Q and K for S, V, and what TMA writes:
 * 2560 cycles for 128 keys) beside 2048 of MMAs and 1024 of exponentials (16 a cycle and SM); at
 * 128 the same at half the size, 1280 beside 1024 and 1024; at 64 the exponentials.
 */
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "attn_decode.cuh"
#include "attn_view.cuh"
#include "common.cuh"
#include "prefill_gemm.cuh"

namespace apus {

constexpr int AP_ROWS = 128;                 /* rows of a tile, keys of a step */
constexpr int AP_SOFT_WARPS = 8;
constexpr int AP_THREADS = 128 + AP_SOFT_WARPS * 32;
/* The registers of a block of twelve warps are 168 a thread.  The two warps that issue loads and
 * MMAs (and two that only fill up their group) need few; the softmax warps take over the rest:
 * 128 x 40 + 256 x 232 = 384 x 168 (checked before the first launch: a sum above what the block
 * has would wait for ever). */
constexpr int AP_REGS_ISSUE = 40, AP_REGS_SOFT = 232;
constexpr int AP_TMEM_COLS = 512;
constexpr int AP_TMEM_O = 256;               /* scores in columns 0..255 */
constexpr int AP_ITEMS = 2;
constexpr int AP_MAX_SPLITS = 16;
/* outputs of 128 rows as they are in tensor memory, then each row's maximum and sum */
constexpr int AP_PART_FLOATS = AP_ROWS * (256 + 2);

template <int D>
struct ApShape {
    static constexpr int BLOCKS = D / 64;                 /* of 64 values: a swizzle row */
    static constexpr int Q_BYTES = AP_ROWS * D * 2;
    static constexpr int UNITS = D == 256 ? 2 : 1;        /* pieces of a tile of K or of V */
    static constexpr int UNIT_BYTES = AP_ROWS * D * 2 / UNITS;
    static constexpr int V_ROWS = AP_ROWS / UNITS;        /* keys of a piece of V (all values) */
    static constexpr int K_BLOCKS = BLOCKS / UNITS;       /* blocks of a piece of K (all keys) */
    static constexpr int STAGES = D == 256 ? 5 : D == 128 ? 6 : 8;
};

struct PromptParams {
    AttnView a;
    const int32_t *cu_q, *cu_k;
    int k_rows, seqs, causal, kv_heads;
    int tile_tokens;                         /* 128 / group */
    int slots, items;                        /* tiles there may be, times key heads and splits */
    int splits;                              /* CTAs that share a tile's keys */
    float *parts;                            /* with splits: [items][AP_PART_FLOATS] */
    unsigned *sched;                         /* next item; [32]: CTAs that are through */
    int absent;                              /* a CTA that loads three pieces (a test's), or -1 */
    int *status;
};

struct ApItem {
    int token, tokens;                       /* first row of q; tokens of the tile, -1: the end */
    int head, tiles;                         /* key head, steps of 128 keys */
    int key, keys;                           /* first row of k; keys that the last token sees */
    int sees;                                /* keys that the first token sees */
    int part;                                /* with splits: whose result it is */
};
struct ApShared {
    uint64_t kv_full[8], kv_empty[8], q_full, q_empty, s_full[2], p_full[2], pv_done[2], o_free,
        through;
    uint64_t item_full[AP_ITEMS], item_empty[AP_ITEMS], pair[4];
    ApItem item[AP_ITEMS];
    uint32_t tmem;
    int abort_flag;
    float shown[2][2][AP_ROWS];              /* what a pair of warps tells one another, in turns */
};
template <int D>
constexpr int ap_smem_bytes() {
    return ApShape<D>::Q_BYTES + ApShape<D>::STAGES * ApShape<D>::UNIT_BYTES +
           (int)sizeof(ApShared);
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int x, int y,
                                            int z, int w, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::"
        "complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}
/* D[tmem] (+)= A[smem] * B[smem] and A[tmem] * B[smem].  Of a descriptor only the low word, with
 * the address, changes from one MMA to the next. */
__device__ __forceinline__ void ap_mma_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi,
                                          uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        ".reg .b64 a, b;\n\t"
        "mov.b64 a, {%1, %2};\n\t"
        "mov.b64 b, {%3, %4};\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n\t"
        "}\n" ::"r"(d_tmem),
        "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void ap_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo,
                                          uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        ".reg .b64 b;\n\t"
        "mov.b64 b, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t"
        "}\n" ::"r"(d_tmem),
        "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, "
        "%31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
        "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
        "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
        "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
        "r"(r[15])
        : "memory");
}
/* 16 rows x 8 columns at a time: lane 4 g + t has columns 2 t, 2 t + 1 of rows g and g + 8 */
__device__ __forceinline__ void tmem_ld_16x256(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
        "%30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
          "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
          "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld_16x256(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
/* two fp32 operations in one instruction */
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
/* Four lanes with four pairs each: pair w of lane t to lane w, as its pair t. */
__device__ __forceinline__ void ap_turn(uint32_t (&e)[4][2], int t) {
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const bool odd = t & 1, high = t & 2;
        const uint32_t x = __shfl_xor_sync(0xffffffffu, odd ? e[0][k] : e[1][k], 1),
                       y = __shfl_xor_sync(0xffffffffu, odd ? e[2][k] : e[3][k], 1);
        const uint32_t a0 = odd ? x : e[0][k], a1 = odd ? e[1][k] : x, a2 = odd ? y : e[2][k],
                       a3 = odd ? e[3][k] : y;
        const uint32_t u = __shfl_xor_sync(0xffffffffu, high ? a0 : a2, 2),
                       v = __shfl_xor_sync(0xffffffffu, high ? a1 : a3, 2);
        e[0][k] = high ? u : a0;
        e[1][k] = high ? v : a1;
        e[2][k] = high ? a2 : u;
        e[3][k] = high ? a3 : v;
    }
}
/* B whose N dimension is contiguous (V: keys are K): 64 values x 8 keys to a swizzle atom of
 * 1024 bytes, the next 8 keys SBO behind it, the next 64 values LBO */
__device__ __forceinline__ uint64_t ap_desc_mn(uint32_t saddr, uint32_t block_bytes) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3ffffu) >> 4);
    d |= (uint64_t)(block_bytes >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
constexpr uint32_t AP_B_MN = 1u << 16;       /* instruction descriptor: B is MN-major */

/* The tile of an index (without splits), by a whole warp.  Sequence i's tiles have the slots from
 * cu_q[i] / tile_tokens + i on: one more than it needs, at most, and no sums over sequences. */
__device__ __forceinline__ ApItem ap_find(const PromptParams &p, int index) {
    const int lane = threadIdx.x & 31, T = p.tile_tokens;
    const int slot = p.slots - 1 - index / p.kv_heads;
    auto base = [&](int i) { return __ldg(p.cu_q + i) / T + i; };
    int lo = 0, hi = p.seqs;
    while (hi - lo > 1) {                    /* the last sequence that starts at or before it */
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const unsigned m = __ballot_sync(0xffffffffu, at < hi && base(at) <= slot);
        const int n = m ? 32 - __clz(m) : 1;
        lo += (n - 1) * step;
        hi = min(hi, lo + step);
    }
    ApItem t;
    const int q0 = min(max(__ldg(p.cu_q + lo), 0), p.a.rows),
              q1 = min(max(__ldg(p.cu_q + lo + 1), q0), p.a.rows);
    const int k0 = min(max(__ldg(p.cu_k + lo), 0), p.k_rows),
              k1 = min(max(__ldg(p.cu_k + lo + 1), k0), p.k_rows);
    const long first = (long)(slot - base(lo)) * T;       /* of the sequence's rows */
    t.token = q0 + (int)first;
    t.tokens = first < 0 || first >= q1 - q0 ? 0 : min(T, q1 - q0 - (int)first);
    t.head = index % p.kv_heads;
    t.key = k0;
    t.keys = t.sees = k1 - k0;
    if (p.causal) {
        t.sees = k1 - k0 - (q1 - q0) + (int)first + 1;
        t.keys = max(0, t.sees + t.tokens - 1);
    }
    t.tiles = (t.keys + AP_ROWS - 1) / AP_ROWS;
    t.part = 0;
    return t;
}
/* The same where CTAs share a tile: the keys of one of them, as if they were all there are. */
__device__ __forceinline__ ApItem ap_find_part(const PromptParams &p, int index) {
    ApItem t = ap_find(p, index / p.splits);
    const int per = (t.tiles + p.splits - 1) / p.splits * AP_ROWS;
    const int from = (index % p.splits) * per;
    t.key += from;
    t.sees -= from;
    t.keys = min(max(t.keys - from, 0), per);
    t.tiles = (t.keys + AP_ROWS - 1) / AP_ROWS;
    t.part = index;
    return t;
}

/* SPLIT: CTAs share the keys of a tile, and what a tile ends with is left as it is. */
template <int D, bool SPLIT>
__global__ void __launch_bounds__(AP_THREADS, 1)
attn_prompt_kernel(const __grid_constant__ CUtensorMap map_q,
                   const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v,
                   const __grid_constant__ PromptParams p) {
    using S = ApShape<D>;
    constexpr int STAGES = S::STAGES;
    extern __shared__ __align__(1024) unsigned char ap_smem[];
    unsigned char *q_smem = ap_smem, *ring = ap_smem + S::Q_BYTES;
    ApShared &s = *reinterpret_cast<ApShared *>(ring + STAGES * S::UNIT_BYTES);
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);   /* known to be the warp's */
    if (smem_u32(ap_smem) & 1023) {          /* swizzled tiles: the same answer in all threads */
        if (tid == 0) set_status(p.status, ST_BAD_INDEX);
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < STAGES; i++) {
            mbar_init(&s.kv_full[i], 1);
            mbar_init(&s.kv_empty[i], 1);
        }
        mbar_init(&s.q_full, 1);
        mbar_init(&s.q_empty, 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&s.s_full[i], 1);
            mbar_init(&s.p_full[i], AP_SOFT_WARPS);
            mbar_init(&s.pv_done[i], 1);
        }
        mbar_init(&s.o_free, AP_SOFT_WARPS);
        mbar_init(&s.through, 1);
        for (int i = 0; i < AP_ITEMS; i++) {
            mbar_init(&s.item_full[i], 1);
            mbar_init(&s.item_empty[i], 1 + AP_SOFT_WARPS);
        }
        for (int i = 0; i < 4; i++) mbar_init(&s.pair[i], 2);
        s.abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc(&s.tmem, AP_TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s.tmem;
    volatile int *abort_flag = &s.abort_flag;
    pdl_enter();

    /* the next tile, for all roles but the one that finds it */
    auto next_item = [&](int n, ApItem &t) -> bool {
        const int i = n % AP_ITEMS;
        if (!pg_wait_warp(&s.item_full[i], (uint32_t)(n / AP_ITEMS) & 1u, abort_flag, p.status,
                          ST_SCHED_TIMEOUT))
            return false;
        /* by shuffles, so that what follows from it (loops, descriptors) is known to be the
         * same in all lanes and is kept in uniform registers, where MMAs want it */
        const int *from = reinterpret_cast<const int *>(&s.item[i]);
        int *to = reinterpret_cast<int *>(&t);
#pragma unroll
        for (int w = 0; w < (int)(sizeof(ApItem) / 4); w++)
            to[w] = __shfl_sync(0xffffffffu, from[w], 0);
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.item_empty[i]);
        return t.tokens >= 0;
    };

    if (warp < 4) {
        /* (one instruction for the four warps of the group) */
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(AP_REGS_ISSUE));
    if (warp == 0) {
        /* ---------------- tiles and loads ---------------- */
        uint32_t unit = 0;
        int full = 0, asked = 0;             /* tiles that see keys; those whose Q was asked for */
        int index = blockIdx.x;
        bool alive = true;
        auto load = [&](bool keys, const ApItem &t, int j) {
            for (int u = 0; u < S::UNITS && alive; u++, unit++) {
                const int st = (int)(unit % STAGES);
                if ((unit == 3 && (int)blockIdx.x == p.absent) ||
                    !pg_wait(&s.kv_empty[st], ((unit / STAGES) & 1u) ^ 1u, abort_flag, p.status,
                             ST_MBAR_TIMEOUT)) {
                    alive = false;
                    return;
                }
                const uint32_t dst = smem_u32(ring + st * S::UNIT_BYTES);
                mbar_expect_tx(&s.kv_full[st], S::UNIT_BYTES);
                if (keys) {
#pragma unroll
                    for (int b = 0; b < S::K_BLOCKS; b++)
                        tma_load_4d(dst + b * AP_ROWS * 128, &map_k, 0, t.key + j * AP_ROWS,
                                    t.head, u * S::K_BLOCKS + b, &s.kv_full[st]);
                } else {
#pragma unroll
                    for (int b = 0; b < S::BLOCKS; b++)
                        tma_load_4d(dst + b * S::V_ROWS * 128, &map_v, 0,
                                    t.key + j * AP_ROWS + u * S::V_ROWS, t.head, b,
                                    &s.kv_full[st]);
                }
            }
        };
        for (int n = 0; alive; n++) {
            ApItem t;
            t.tokens = -1;
            while (index < p.items) {
                t = SPLIT ? ap_find_part(p, index) : ap_find(p, index);
                if (t.tokens > 0) break;
                t.tokens = -1;
                index = p.items > (int)gridDim.x
                            ? __shfl_sync(0xffffffffu,
                                          lane == 0 ? (int)(gridDim.x + atomicAdd(p.sched, 1u)) : 0,
                                          0)
                            : p.items;
            }
            const int i = n % AP_ITEMS;
            if (!pg_wait_warp(&s.item_empty[i], ((uint32_t)(n / AP_ITEMS) & 1u) ^ 1u, abort_flag,
                              p.status, ST_SCHED_TIMEOUT))
                break;
            if (lane == 0) {
                s.item[i] = t;
                mbar_arrive(&s.item_full[i]);
            }
            __syncwarp();
            if (t.tokens < 0) break;
            if (lane == 0 && t.tiles > 0) {
                if (!pg_wait(&s.q_empty, ((uint32_t)full & 1u) ^ 1u, abort_flag, p.status,
                             ST_MBAR_TIMEOUT)) {
                    alive = false;
                } else {
                    const int rows = p.a.group * p.tile_tokens;
                    asked++;
                    mbar_expect_tx(&s.q_full, (uint32_t)(S::BLOCKS * rows * 128));
#pragma unroll
                    for (int b = 0; b < S::BLOCKS; b++)
                        tma_load_4d(smem_u32(q_smem + b * AP_ROWS * 128), &map_q, 0,
                                    t.head * p.a.group, t.token, b, &s.q_full);
                    load(true, t, 0);
                    for (int j = 0; j < t.tiles && alive; j++) {
                        if (j + 1 < t.tiles) load(true, t, j + 1);
                        load(false, t, j);
                    }
                }
            }
            if (t.tiles > 0) full++;
            index = p.items;
            if (p.items > (int)gridDim.x) {
                if (lane == 0) index = (int)(gridDim.x + atomicAdd(p.sched, 1u));
                index = __shfl_sync(0xffffffffu, index, 0);
            }
            alive = __all_sync(0xffffffffu, alive);
        }
        /* given up: copies that are under way land before the CTA leaves */
        if (lane == 0 && *abort_flag) {
            for (uint32_t u = unit > STAGES ? unit - STAGES : 0; u < unit; u++)
                mbar_wait(&s.kv_full[u % STAGES], (u / STAGES) & 1u);
            if (asked) mbar_wait(&s.q_full, (uint32_t)(asked - 1) & 1u);
        }
        /* the last CTA that asks no more sets the counters back */
        if (lane == 0 && p.items > (int)gridDim.x) {
            __threadfence();
            if (atomicInc(p.sched + 32, gridDim.x - 1) == gridDim.x - 1) atomicExch(p.sched, 0u);
        }
    } else if (warp == 1) {
        /* ---------------- MMA issuer ---------------- */
        uint32_t unit = 0, scores = 0, sums = 0;
        int full = 0;
        bool alive = true;
        const uint64_t q_desc = umma_smem_desc(smem_u32(q_smem));
        const uint32_t q_lo = (uint32_t)q_desc, q_hi = (uint32_t)(q_desc >> 32);
        const uint32_t ring_addr = smem_u32(ring);
        ApItem t = {};
        auto wait = [&](uint64_t *bar, uint32_t parity) {
            alive = alive && pg_wait_warp(bar, parity & 1u, abort_flag, p.status, ST_TMEM_TIMEOUT);
            tc_fence_after();
            return alive;
        };
        /* A wait costs this warp about 170 cycles even where there is nothing to wait for, and the
         * tensor cores have one or two MMAs queued meanwhile: a barrier is looked at before the
         * MMAs that come before it are issued, and waited for only where that said no. */
        bool unit_ready = false, weights_ready = false;
        auto wait_seen = [&](bool seen, uint64_t *bar, uint32_t parity) {
            if (!__all_sync(0xffffffffu, seen)) return wait(bar, parity);
            tc_fence_after();
            return alive;
        };
        auto look_ahead = [&]() {            /* at the piece after this one */
            const uint32_t next = unit + 1;
            unit_ready = mbar_test(&s.kv_full[next % STAGES], (next / STAGES) & 1u);
        };
        auto score = [&](int j) {
            const uint32_t d = tmem + (scores & 1u) * AP_ROWS;
            /* no more columns than there are keys (what lies behind them is masked) */
            const int cols = min(AP_ROWS, ((t.keys - j * AP_ROWS) + 15) & ~15);
            const uint32_t idesc = umma_idesc(cols);
            for (int u = 0; u < S::UNITS; u++, unit++) {
                const int st = (int)(unit % STAGES);
                if (!wait_seen(unit_ready, &s.kv_full[st], unit / STAGES)) return;
                look_ahead();
                if (u + 1 == S::UNITS)
                    weights_ready = mbar_test(&s.p_full[sums & 1u], (sums >> 1) & 1u);
                const uint32_t k_lo = (uint32_t)umma_smem_desc(ring_addr + st * S::UNIT_BYTES);
                const uint32_t q_at = q_lo + u * S::K_BLOCKS * (AP_ROWS * 128 / 16);
                if (pg_elect()) {
#pragma unroll
                    for (int b = 0; b < S::K_BLOCKS; b++)
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const uint32_t off = b * (AP_ROWS * 128 / 16) + 2 * k;
                            ap_mma_ss(d, q_at + off, q_hi, k_lo + off, q_hi, idesc,
                                      (u | b | k) ? 1u : 0u);
                        }
                    umma_commit(&s.kv_empty[st]);
                }
            }
            if (pg_elect()) {
                umma_commit(&s.s_full[scores & 1u]);
                if (j + 1 == t.tiles) umma_commit(&s.q_empty);
            }
            scores++;
        };
        for (int n = 0; alive && next_item(n, t); n++) {
            if (!t.tiles) continue;
            if (!wait(&s.q_full, (uint32_t)full)) break;
            score(0);
            for (int j = 0; j < t.tiles && alive; j++) {
                weights_ready = false;
                if (j + 1 < t.tiles) score(j + 1);
                if (!alive || !wait_seen(weights_ready, &s.p_full[sums & 1u], sums >> 1)) break;
                /* the tile before is out of tensor memory */
                if (j == 0 && full > 0 && !wait(&s.o_free, (uint32_t)(full - 1))) break;
                const uint32_t pa = tmem + (sums & 1u) * AP_ROWS;
                const int keys = min(AP_ROWS, t.keys - j * AP_ROWS);
                for (int u = 0; u < S::UNITS; u++, unit++) {
                    const int st = (int)(unit % STAGES);
                    if (!wait_seen(unit_ready, &s.kv_full[st], unit / STAGES)) break;
                    look_ahead();
                    const int here = min(max(keys - u * S::V_ROWS, 0), S::V_ROWS);
                    /* Keys behind the last one that any row sees have weight zero, but their
                     * values may be anything, and 0 * NaN is not 0: whole steps of 16 of them
                     * are left out, the rest of the last step is cleared. */
                    const int steps = (here + 15) / 16;
                    if (here & 15) {
                        unsigned char *v = ring + st * S::UNIT_BYTES;
                        const int rows = steps * 16 - here;
                        for (int i = lane; i < S::BLOCKS * rows * 8; i += 32) {
                            const int b = i / (rows * 8), r = i - b * rows * 8;
                            *reinterpret_cast<uint4 *>(v + b * S::V_ROWS * 128 + here * 128 +
                                                       r * 16) = make_uint4(0, 0, 0, 0);
                        }
                        fence_proxy_async();
                        __syncwarp();
                    }
                    const uint64_t v_desc =
                        ap_desc_mn(ring_addr + st * S::UNIT_BYTES, S::V_ROWS * 128);
                    const uint32_t v_lo = (uint32_t)v_desc, v_hi = (uint32_t)(v_desc >> 32);
                    if (pg_elect()) {
#pragma unroll
                        for (int k = 0; k < S::V_ROWS / 16; k++)
                            if (k < steps)
                                ap_mma_ts(tmem + AP_TMEM_O, pa + (u * S::V_ROWS / 16 + k) * 8,
                                          v_lo + k * (16 * 128 / 16), v_hi,
                                          umma_idesc(D) | AP_B_MN,
                                          (j | u | k) ? 1u : 0u);
                        umma_commit(&s.kv_empty[st]);
                    }
                }
                if (!alive) break;
                if (pg_elect()) umma_commit(&s.pv_done[sums & 1u]);
                sums++;
            }
            full++;
        }
        if (*abort_flag) {                   /* given up: no MMA outlives the CTA's tensor memory */
            if (pg_elect()) umma_commit(&s.through);
            __syncwarp();
            mbar_wait(&s.through, 0);
            __syncwarp();
        }
    }
    } else {
        /* ---------------- softmax and outputs ---------------- */
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(AP_REGS_SOFT));
        constexpr int COLS = AP_ROWS / 2;    /* scores of a row that a thread has */
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        const int row = quarter * 32 + lane;
        /* row / group as a product (rows below 128, groups up to 16) */
        const int by_group = 65536 / p.a.group + 1;
        const int my_token = (row * by_group) >> 16, my_head = row - my_token * p.a.group;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const float sc = p.a.scale * LOG2E;
        uint32_t first = 0, rounds = 0;      /* steps before this tile; exchanges of a pair of warps */
        bool alive = true;
        ApItem t = {};
        auto wait = [&](uint64_t *bar, uint32_t parity) {
            alive = alive && pg_wait_warp(bar, parity & 1u, abort_flag, p.status, ST_TMEM_TIMEOUT);
            tc_fence_after();
            return alive;
        };
        /* a row's other half; two buffers in turns: who writes one has seen the other warp through
         * with it, at the exchange between */
        auto exchange = [&](float &x) {
            float (&shown)[2][AP_ROWS] = s.shown[rounds & 1u];
            shown[half][row] = x;
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.pair[quarter]);
            if (!wait(&s.pair[quarter], rounds++)) return false;
            x = shown[half ^ 1][row];
            return true;
        };
        /* O holds step i.  A parity tells a phase only from the one before it, and that this warp
         * (or its pair) has seen i's scores says no more than that step i - 2 is through: two
         * barriers in turn. */
        auto wait_outputs = [&](uint32_t i) { return wait(&s.pv_done[i & 1u], i >> 1); };
        for (int n = 0; alive && next_item(n, t); n++) {
            const int sees = p.causal ? min(max(t.sees + my_token, 0), t.keys) : t.keys;
            const bool real = my_token < t.tokens;
            const long r = t.token + my_token;
            const int h = t.head * p.a.group + my_head;
            if (!SPLIT && p.a.gate && real)               /* to L2, for the end of the tile */
#pragma unroll
                for (int c = 0; c < D / 2; c += 64)
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(
                        p.a.gate + r * p.a.gate_stride + (size_t)h * D + half * (D / 2) + c));
            float top = -INFINITY, sum = 0.0f;            /* top: of scores times sc */
            for (int j = 0; j < t.tiles; j++) {
                const uint32_t step = first + j, buf = step & 1u;
                if (!wait(&s.s_full[buf], step >> 1)) break;
                const uint32_t ts = tmem + lanes + buf * AP_ROWS;
                uint32_t x[COLS / 32][32];
#pragma unroll
                for (int c = 0; c < COLS / 32; c++)
                    tmem_ld32(ts + half * COLS + c * 32, x[c]);
                tmem_ld_wait();
                const int lim = sees - j * AP_ROWS - half * COLS;
                if (!__all_sync(0xffffffffu, lim >= COLS)) {
#pragma unroll
                    for (int c = 0; c < COLS; c++)
                        if (c >= lim) x[c >> 5][c & 31] = 0xff800000u;
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < COLS; c++)
                    mx[c & 3] = fmaxf(mx[c & 3], __uint_as_float(x[c >> 5][c & 31]));
                const float m_here = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc;
                float m = m_here;
                if (!exchange(m)) break;
                m = fmaxf(m, m_here);
                const bool move = m > top + 8.0f || (top == -INFINITY && m > -INFINITY);
                if (__any_sync(0xffffffffu, move)) {
                    const float f = move ? exp2_fast(top - m) : 1.0f;
                    if (move) top = m;
                    sum *= f;
                    if (j > 0) {
                        if (!wait_outputs(step - 1)) break;
                        const uint32_t to = tmem + lanes + AP_TMEM_O + half * (D / 2);
#pragma unroll 1
                        for (int c = 0; c < D / 2; c += 32) {
                            uint32_t o[32];
                            tmem_ld32(to + c, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; i++)
                                o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tmem_st32(to + c, o);
                        }
                        tmem_st_wait();
                    }
                }
                const float base = top == -INFINITY ? 0.0f : top;
                const float2 sc2 = make_float2(sc, sc), base2 = make_float2(-base, -base);
                float2 part[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (int c = 0; c < COLS / 32; c++) {
                    uint32_t pk[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float2 z = fma2(make_float2(__uint_as_float(x[c][2 * i]),
                                                          __uint_as_float(x[c][2 * i + 1])),
                                              sc2, base2);
                        const float2 w = make_float2(exp2_fast(z.x), exp2_fast(z.y));
                        part[i & 1] = add2(part[i & 1], w);
                        pk[i] = pack_bf16_rn(w.x, w.y);   /* the weights' one rounding */
                    }
                    tmem_st16(ts + half * (COLS / 2) + c * 16, pk);
                }
                part[0] = add2(part[0], part[1]);
                sum += part[0].x + part[0].y;
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s.p_full[buf]);
            }
            if (!alive) break;
            /* ---- the tile's outputs ----
             * Read from tensor memory as 16 rows x 8 values a step, four lanes to a row with two
             * values each: after a 4 x 4 exchange a lane has 8 values side by side, and a
             * warp's load or store is 64 bytes of each of 8 rows (a row to a lane would be 32 lines
             * an instruction).  The loop stays one: unrolled, its instructions took longer to
             * come than to run (12000 cycles a tile). */
            constexpr int CHUNK = D / 2 < 64 ? D / 2 : 64, PIECES = CHUNK / 32;
            constexpr int CHUNKS = D / 2 / CHUNK;         /* steps for each 16 rows */
            const int t4 = lane & 3, g = lane >> 2;
            auto place = [&](int i, int k, long &token, int &in) {
                const int o_row = quarter * 32 + (i / CHUNKS) * 16 + k * 8 + g;
                const int in_tile = (o_row * by_group) >> 16;
                token = t.token + in_tile;
                in = (t.head * p.a.group + o_row - in_tile * p.a.group) * D + half * (D / 2) +
                     (i % CHUNKS) * CHUNK + t4 * 8;
                return in_tile < t.tokens;
            };
            uint4 gate[2][PIECES];                        /* of the next step, under way */
            auto load_gate = [&](int i) {
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    long token;
                    int in;
                    if (place(i, k, token, in))
#pragma unroll
                        for (int w = 0; w < PIECES; w++)
                            gate[k][w] = ldg16(p.a.gate + token * p.a.gate_stride + in + w * 32);
                }
                __syncwarp();
            };
            if (p.a.gate && !SPLIT) load_gate(0);
            if (t.tiles) {
                float other = sum;
                if (!exchange(other)) break;
                sum += other;
                if (!wait_outputs(first + t.tiles - 1)) break;
            }
            const float inv = __fdividef(1.0f, sum);
#pragma unroll 1
            for (int i = 0; i < (SPLIT && !t.tiles ? 0 : 2 * CHUNKS); i++) {
                uint4 now[2][PIECES];
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int w = 0; w < PIECES; w++) now[k][w] = gate[k][w];
                if (p.a.gate && !SPLIT && i + 1 < 2 * CHUNKS) load_gate(i + 1);
                uint32_t o[CHUNK / 2];
                if (t.tiles) {
                    tmem_ld_16x256(tmem + lanes + ((uint32_t)(i / CHUNKS * 16) << 16) + AP_TMEM_O +
                                       half * (D / 2) + (i % CHUNKS) * CHUNK,
                                   o);
                    tmem_ld_wait();
                }
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    long token;
                    int in;
                    const bool there = place(i, k, token, in);
                    const int from = (i / CHUNKS) * 16 + k * 8 + g;
                    const float f = __shfl_sync(0xffffffffu, inv, from);
                    const float2 f2 = make_float2(f, f);
                    const bool none = __shfl_sync(0xffffffffu, sum, from) == 0.0f;
#pragma unroll
                    for (int w = 0; w < PIECES; w++) {
                        uint32_t e[4][2];
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            e[x][0] = o[(w * 4 + x) * 4 + k * 2];
                            e[x][1] = o[(w * 4 + x) * 4 + k * 2 + 1];
                        }
                        ap_turn(e, t4);
                        if (SPLIT) {                      /* as it is, for attn_prompt_join_kernel */
                            float *to = p.parts + (size_t)t.part * AP_PART_FLOATS +
                                        (quarter * 32 + from) * D + half * (D / 2) +
                                        (i % CHUNKS) * CHUNK + t4 * 8 + w * 32;
                            uint4 *to4 = reinterpret_cast<uint4 *>(to);
                            to4[0] = make_uint4(e[0][0], e[0][1], e[1][0], e[1][1]);
                            to4[1] = make_uint4(e[2][0], e[2][1], e[3][0], e[3][1]);
                            continue;
                        }
                        uint32_t v[4];
                        const uint32_t z[4] = {now[k][w].x, now[k][w].y, now[k][w].z, now[k][w].w};
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            float2 y = mul2(make_float2(__uint_as_float(e[x][0]),
                                                        __uint_as_float(e[x][1])), f2);
                            if (p.a.gate)
                                y = mul2(y, make_float2(ad_gate(bf16lo(z[x])), ad_gate(bf16hi(z[x]))));
                            /* no key: zero, whatever O holds */
                            v[x] = none ? 0u : pack_bf16_rn(y.x, y.y);
                        }
                        if (there)
                            *reinterpret_cast<uint4 *>(p.a.out + token * p.a.out_stride + in +
                                                       w * 32) =
                                make_uint4(v[0], v[1], v[2], v[3]);
                    }
                }
                __syncwarp();
            }
            if (SPLIT && half == 0)
                *reinterpret_cast<float2 *>(p.parts + (size_t)t.part * AP_PART_FLOATS +
                                            AP_ROWS * 256 + row * 2) = make_float2(top, sum);
            if (!SPLIT && p.a.lse && real && half == 0)
                p.a.lse[r * p.a.heads + h] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * LN2;
            if (t.tiles) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s.o_free);
            }
            first += t.tiles;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, AP_TMEM_COLS);
    }
}

/* Tiles whose keys several CTAs have shared: a warp to a row, the parts in order. */
template <int D>
__global__ void __launch_bounds__(256) attn_prompt_join_kernel(const __grid_constant__ PromptParams p) {
    pdl_enter();
    constexpr int N = D / 32;                /* values of a lane */
    const ApItem t = ap_find(p, blockIdx.x);
    const int lane = threadIdx.x & 31;
    for (int row = blockIdx.y * 8 + (threadIdx.x >> 5); row < t.tokens * p.a.group;
         row += 8 * gridDim.y) {
        float2 ml[AP_MAX_SPLITS];
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int k = 0; k < AP_MAX_SPLITS; k++)
            if (k < p.splits) {
                ml[k] = *reinterpret_cast<const float2 *>(
                    p.parts + (size_t)(blockIdx.x * p.splits + k) * AP_PART_FLOATS +
                    AP_ROWS * 256 + row * 2);
                top = fmaxf(top, ml[k].x);
            }
        float acc[N] = {};
#pragma unroll
        for (int k = 0; k < AP_MAX_SPLITS; k++)
            if (k < p.splits && ml[k].y != 0.0f) {        /* (a part without keys has no outputs) */
                const float f = exp2_fast(ml[k].x - top);
                const float *o = p.parts + (size_t)(blockIdx.x * p.splits + k) * AP_PART_FLOATS +
                                 row * D + lane * N;
                sum = fmaf(f, ml[k].y, sum);
#pragma unroll
                for (int i = 0; i < N; i += 2) {
                    const float2 v = *reinterpret_cast<const float2 *>(o + i);
                    acc[i] = fmaf(f, v.x, acc[i]);
                    acc[i + 1] = fmaf(f, v.y, acc[i + 1]);
                }
            }
        const int in_tile = row / p.a.group;
        const long token = t.token + in_tile;
        const int head = t.head * p.a.group + row - in_tile * p.a.group;
        const float inv = sum == 0.0f ? 0.0f : __fdividef(1.0f, sum);
        const int at = head * D + lane * N;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            float a = acc[i] * inv, b = acc[i + 1] * inv;
            if (p.a.gate) {
                const uint32_t z = *reinterpret_cast<const uint32_t *>(
                    p.a.gate + token * p.a.gate_stride + at + i);
                a *= ad_gate(bf16lo(z));
                b *= ad_gate(bf16hi(z));
            }
            if (sum == 0.0f) a = b = 0.0f;   /* no key, whatever the gate is */
            *reinterpret_cast<uint32_t *>(p.a.out + token * p.a.out_stride + at + i) =
                pack_bf16_rn(a, b);
        }
        if (p.a.lse && lane == 0)
            p.a.lse[token * p.a.heads + head] =
                sum == 0.0f ? -INFINITY : (top + log2f(sum)) * LN2;
    }
}

}  // namespace apus
