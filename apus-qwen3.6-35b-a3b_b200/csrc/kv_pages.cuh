/*
 * kv_pages.cuh — the page book-keeping of a key-value cache, on the device: sequences take
 * pages, share them, give them back, and the pages in use are moved together.  (Net-new: the
 * engine keeps one plain cache per process, c/attn.h.)
 *
 * The state is three integer arrays of the caller's: refs [pages] (sequences that hold a page,
 * 0: free), table [seqs][max_pages] (a sequence's pages in order) and len [seqs].  Which pages a
 * call takes follows from them alone (the lowest free ones, in the order of its list), so a
 * result does not depend on the order in which threads run.
 *
 * A call that has to decide for the whole cache first (extend, fork, compact) does so in one CTA
 * (the "plan"): it checks the list, counts, and finds free pages by one look at refs, 4 bytes a
 * page by 32 warps with eight loads under way each.  What bounds it is the round trips to L2 that
 * depend on one another (about 0.7 us each), so refs is asked for before the list, and marks of
 * sequences are bits in shared memory.  A plan that cannot be carried out leaves a status and
 * changes nothing.  What moves bytes (kv_apply_kernel) runs on all SMs and reads the plan: its
 * bound is HBM, each page read once and written once (241 MB moved together: 75 us, 6.4 TB/s of
 * reads and writes).
 *
 * One SM's loads bound a plan over a large pool: 0.08 to 0.09 us a thousand pages for each look at refs
 * (two to find free pages, three to close up).  Closing up with nothing to move takes 5 us over
 * 2000 pages, 34 over 100 000, 146 over 500 000; 8192 tokens of 256 sequences with their places 20
 * us over 8192 pages, 37 and 102; tokens that need no page 7, and 8 with places, over any pool.
 */
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/backend_cuda.h"
#include "common.cuh"

namespace apus {

constexpr int KV_PLAN_THREADS = 1024;
constexpr int KV_APPLY_THREADS = 256;

/* what went wrong first, in work[0] until the caller clears it */
enum : int { KV_OK = 0, KV_NO_PAGES = 1, KV_BAD_LIST = 2, KV_BAD_PAGE = 3 };

constexpr int KV_MAX_SEQS = 65536;
constexpr int KV_CHECK_PAGES = 1 << 18, KV_CHECK_LIST = 4096;

/* the caller's scratch: work[0] status, [1] copies, [2] pages in use, [3] plan accepted;
 * from 64 on: copy sources, copy targets, page map, marks of pages; then per entry of a list
 * first fresh page, and where a sequence's new tokens start */
struct KvView {
    uint16_t *k, *v;
    int32_t *refs, *table, *len, *work;
    int layers, pages, page_tokens, seqs, max_pages;
    int page_elems;                /* kv_heads * page_tokens * head_dim */
    __device__ int32_t *status() const { return work; }
    __device__ int32_t *copy_src() const { return work + 64; }
    __device__ int32_t *copy_dst() const { return work + 64 + pages; }
    __device__ int32_t *map() const { return work + 64 + 2 * (size_t)pages; }
    __device__ int32_t *mark() const { return work + 64 + 3 * (size_t)pages; }
    __device__ int32_t *first() const { return work + 64 + 4 * (size_t)pages; }
    __device__ int32_t *starts() const { return first() + seqs; }
    /* pages that `tokens` tokens take */
    __device__ int held(int tokens) const {
        return tokens <= 0 ? 0 : min((int)(((unsigned)tokens + page_tokens - 1) / page_tokens),
                                     max_pages);
    }
};

/* exclusive prefix over the CTA and the total */
__device__ __forceinline__ int kv_block_scan(int v, int *total, int *smem /* [33] */) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) smem[warp] = x;
    __syncthreads();
    if (warp == 0) {
        const int w = lane < (int)(blockDim.x >> 5) ? smem[lane] : 0;
        int s = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        smem[lane] = s - w;
        if (lane == 31) smem[32] = s;
    }
    __syncthreads();
    *total = smem[32];
    return smem[warp] + x - v;
}

/* The pages by the whole CTA, 32 warps with a piece each, in ascending order within it.  The
 * first 256 of a piece (all of it up to 8192 pages) are asked for when the object is made. */
struct KvPages {
    const KvView &kv;
    int lo, hi, ahead[8];
    __device__ __forceinline__ explicit KvPages(const KvView &kv_) : kv(kv_) {
        const int warp = threadIdx.x >> 5;
        const int piece = ((kv.pages + 31) / 32 + 255) / 256 * 256;
        lo = min(warp * piece, kv.pages);
        hi = min(lo + piece, kv.pages);
        load(lo, ahead);
    }
    __device__ __forceinline__ void load(int p0, int (&r)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int p = p0 + i * 32 + (threadIdx.x & 31);
            r[i] = p < hi ? kv.refs[p] : 0;
        }
    }
    /* f(page, whether it is one, whether it is in use), by full warps */
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        for (int p0 = lo; p0 < hi; p0 += 256) {
            int r[8];
            if (p0 == lo) {
#pragma unroll
                for (int i = 0; i < 8; i++) r[i] = ahead[i];
            } else {
                load(p0, r);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int p = p0 + i * 32 + (threadIdx.x & 31);
                f(p, p < hi, r[i] != 0);
            }
        }
    }
    /* The first `want` free pages in ascending order into list; how many are free. */
    __device__ __forceinline__ int find_free(int want, int32_t *list, int *smem) const {
        const int lane = threadIdx.x & 31;
        int mine = 0;
        each([&](int, bool there, bool used) {
            mine += __popc(__ballot_sync(0xffffffffu, there && !used));
        });
        int total;
        int at = kv_block_scan(lane == 0 ? mine : 0, &total, smem);
        at = __shfl_sync(0xffffffffu, at, 0);
        if (total >= want)
            each([&](int p, bool there, bool used) {
                const unsigned freed = __ballot_sync(0xffffffffu, there && !used);
                const int r = at + __popc(freed & ((1u << lane) - 1));
                if (there && !used && r < want) list[r] = p;
                at += __popc(freed);
            });
        __syncthreads();
        return total;
    }
};

/* Sequences of a list: in range, none twice; their bits are set then.  (All threads; true where
 * the list is sound.) */
__device__ __forceinline__ bool kv_check_list(const KvView &kv, const int32_t *seq, int n,
                                              unsigned *bits /* [KV_MAX_SEQS / 32] */) {
    for (int i = threadIdx.x; i < (kv.seqs + 31) / 32; i += blockDim.x) bits[i] = 0;
    __syncthreads();
    int bad = 0;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int s = seq ? seq[i] : i;
        if ((unsigned)s >= (unsigned)kv.seqs) bad = 1;
        else if (atomicOr(&bits[s >> 5], 1u << (s & 31)) >> (s & 31) & 1) bad = 1;
    }
    return !__syncthreads_or(bad);
}

/* Room for cu[i+1] - cu[i] more tokens in sequence seq[i]; slot [rows] (or null): where the
 * packed rows' tokens go, -1 for all of them where the call is refused, and for rows outside of cu. */
__global__ void __launch_bounds__(KV_PLAN_THREADS)
kv_extend_kernel(KvView kv, const int32_t *__restrict__ seq, const int32_t *__restrict__ cu, int n,
                 int32_t *__restrict__ slot, int rows) {
    pdl_enter();
    __shared__ int smem[33];
    __shared__ unsigned bits[KV_MAX_SEQS / 32];
    const int tid = threadIdx.x;
    const KvPages pages(kv);
    int code = kv_check_list(kv, seq, n, bits) ? KV_OK : KV_BAD_LIST;
    int taken = 0;
    if (code == KV_OK) {
        int bad = 0;
        for (int i0 = 0; i0 < n; i0 += KV_PLAN_THREADS) {
            const int i = i0 + tid;
            int need = 0;
            if (i < n) {
                const int add = cu[i + 1] - cu[i], old = kv.len[seq ? seq[i] : i];
                const long long now = (long long)old + add;
                if (add < 0 || old < 0 || now > (long long)kv.max_pages * kv.page_tokens) bad = 1;
                else need = kv.held((int)now) - kv.held(old);
            }
            int total;
            const int at = kv_block_scan(need, &total, smem);
            if (i < n) kv.first()[i] = taken + at;
            taken = (int)min((long long)taken + total, 0x7fffffffLL);
        }
        if (__syncthreads_or(bad)) code = KV_BAD_LIST;
    }
    if (code == KV_OK && taken > 0) {
        if (taken > kv.pages || pages.find_free(taken, kv.copy_src(), smem) < taken)
            code = KV_NO_PAGES;
    }
    if (code != KV_OK) {
        if (tid == 0) atomicCAS(kv.status(), 0, code);
        if (slot)
            for (int t = tid; t < rows; t += KV_PLAN_THREADS) slot[t] = -1;
        return;
    }
    /* a warp to a sequence: its new pages */
    for (int i = tid >> 5; i < n; i += KV_PLAN_THREADS / 32) {
        const int s = seq ? seq[i] : i, old = kv.len[s], now = old + cu[i + 1] - cu[i];
        const int from = kv.held(old), to = kv.held(now), first = kv.first()[i];
        for (int j = from + (tid & 31); j < to; j += 32) {
            const int p = kv.copy_src()[first + j - from];
            kv.table[(size_t)s * kv.max_pages + j] = p;
            kv.refs[p] = 1;
        }
        if ((tid & 31) == 0) kv.starts()[s] = old;
        __syncwarp();
        if ((tid & 31) == 0) kv.len[s] = now;
    }
    if (!slot) return;
    __syncthreads();
    for (int t = tid; t < rows; t += KV_PLAN_THREADS) {
        int lo = 0, hi = n;                    /* the last i with cu[i] <= t */
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (cu[mid + 1] <= t) lo = mid + 1;
            else hi = mid;
        }
        int where = -1;
        if (lo < n && t >= cu[lo]) {
            const int s = seq ? seq[lo] : lo, at = kv.starts()[s] + t - cu[lo];
            const int p = kv.table[(size_t)s * kv.max_pages + at / kv.page_tokens];
            if ((unsigned)p < (unsigned)kv.pages) where = p * kv.page_tokens + at % kv.page_tokens;
            else atomicCAS(kv.status(), 0, KV_BAD_PAGE);
        }
        slot[t] = where;
    }
}

/* The pages of a list of sequences, one CTA each.  A sequence that the list names twice has
 * nothing left the second time. */
__global__ void __launch_bounds__(128)
kv_free_kernel(KvView kv, const int32_t *__restrict__ seq, int n) {
    pdl_enter();
    __shared__ int held;
    for (int i = blockIdx.x; i < n; i += gridDim.x) {
        const int s = seq ? seq[i] : i;
        if (s < 0 || s >= kv.seqs) {
            if (threadIdx.x == 0) atomicCAS(kv.status(), 0, KV_BAD_LIST);
            continue;
        }
        if (threadIdx.x == 0) held = kv.held(atomicExch(&kv.len[s], 0));
        __syncthreads();
        for (int j = threadIdx.x; j < held; j += blockDim.x) {
            int32_t *e = &kv.table[(size_t)s * kv.max_pages + j];
            const int p = *e;
            *e = -1;
            if ((unsigned)p >= (unsigned)kv.pages) {
                atomicCAS(kv.status(), 0, KV_BAD_PAGE);
            } else if (atomicSub(&kv.refs[p], 1) <= 0) {
                atomicAdd(&kv.refs[p], 1);
                atomicCAS(kv.status(), 0, KV_BAD_PAGE);
            }
        }
        __syncthreads();
    }
}

/* dst[i] becomes a second owner of src[i]'s full pages; a page that is not full is copied into a
 * fresh one, so that only full pages are ever shared and none is written twice. */
__global__ void __launch_bounds__(KV_PLAN_THREADS)
kv_fork_plan_kernel(KvView kv, const int32_t *__restrict__ src, const int32_t *__restrict__ dst,
                    int n) {
    pdl_enter();
    __shared__ int smem[33];
    __shared__ unsigned bits[KV_MAX_SEQS / 32];
    const int tid = threadIdx.x;
    const KvPages pages(kv);
    int code = kv_check_list(kv, dst, n, bits) ? KV_OK : KV_BAD_LIST, taken = 0;
    int bad = 0;
    if (code == KV_OK) {
        for (int i0 = 0; i0 < n; i0 += KV_PLAN_THREADS) {
            const int i = i0 + tid;
            int need = 0;
            if (i < n) {
                const int s = src[i];
                /* (none is written that another one is read from) */
                if ((unsigned)s >= (unsigned)kv.seqs || (bits[s >> 5] >> (s & 31) & 1)) {
                    bad = 1;
                } else {
                    const int tokens = kv.len[s];
                    if (tokens < 0 || tokens > kv.max_pages * kv.page_tokens ||
                        kv.len[dst[i]] != 0)
                        bad = 1;
                    else need = tokens % kv.page_tokens ? 1 : 0;
                }
            }
            int total;
            const int at = kv_block_scan(need, &total, smem);
            if (i < n) kv.first()[i] = taken + at;
            taken += total;
        }
        if (__syncthreads_or(bad)) code = KV_BAD_LIST;
    }
    if (code == KV_OK && taken &&
        (taken > kv.pages || pages.find_free(taken, kv.copy_dst(), smem) < taken))
        code = KV_NO_PAGES;
    if (code == KV_OK) {
        for (int i = tid; i < n; i += KV_PLAN_THREADS) {
            const int tokens = kv.len[src[i]];
            if (tokens % kv.page_tokens) {
                const int p =
                    kv.table[(size_t)src[i] * kv.max_pages + tokens / kv.page_tokens];
                if ((unsigned)p >= (unsigned)kv.pages) bad = 1;
                kv.copy_src()[kv.first()[i]] = p;
            }
        }
        if (__syncthreads_or(bad)) code = KV_BAD_PAGE;
    }
    if (tid == 0) {
        if (code != KV_OK) atomicCAS(kv.status(), 0, code);
        kv.work[1] = code == KV_OK ? taken : 0;
        kv.work[3] = code == KV_OK;
    }
}

/* Pages in use at or behind the number of pages in use go, in order, into the free ones before
 * it: sources and targets are apart, so that they may be copied in any order. */
__global__ void __launch_bounds__(KV_PLAN_THREADS)
kv_compact_plan_kernel(KvView kv) {
    pdl_enter();
    __shared__ int smem[33];
    const int lane = threadIdx.x & 31;
    const KvPages pages(kv);
    int mine = 0, live;
    pages.each([&](int, bool there, bool used) {
        mine += __popc(__ballot_sync(0xffffffffu, there && used));
    });
    kv_block_scan(lane == 0 ? mine : 0, &live, smem);
    int leave = 0, fill = 0;
    pages.each([&](int p, bool there, bool used) {
        leave += __popc(__ballot_sync(0xffffffffu, there && used && p >= live));
        fill += __popc(__ballot_sync(0xffffffffu, there && !used && p < live));
    });
    int moves, same;
    int at_leave = kv_block_scan(lane == 0 ? leave : 0, &moves, smem);
    int at_fill = kv_block_scan(lane == 0 ? fill : 0, &same, smem);
    at_leave = __shfl_sync(0xffffffffu, at_leave, 0);
    at_fill = __shfl_sync(0xffffffffu, at_fill, 0);
    pages.each([&](int p, bool there, bool used) {
        const unsigned below = (1u << lane) - 1;
        const bool l = there && used && p >= live, f = there && !used && p < live;
        const unsigned bl = __ballot_sync(0xffffffffu, l), bf = __ballot_sync(0xffffffffu, f);
        if (l) kv.copy_src()[at_leave + __popc(bl & below)] = p;
        if (f) kv.copy_dst()[at_fill + __popc(bf & below)] = p;
        at_leave += __popc(bl);
        at_fill += __popc(bf);
    });
    __syncthreads();
    for (int i = threadIdx.x; i < moves; i += KV_PLAN_THREADS) {
        const int from = kv.copy_src()[i], to = kv.copy_dst()[i];
        kv.map()[from] = to;
        kv.refs[to] = kv.refs[from];
        kv.refs[from] = 0;
    }
    if (threadIdx.x == 0) {
        kv.work[1] = moves;
        kv.work[2] = live;
        kv.work[3] = 1;
    }
}

/* A list of pages as it came: in range, no target twice or a source as well.  (Long lists and large
 * pools; else every CTA that copies looks for itself.) */
__global__ void __launch_bounds__(KV_PLAN_THREADS)
kv_copy_plan_kernel(KvView kv, const int32_t *__restrict__ src, const int32_t *__restrict__ dst,
                    int n) {
    pdl_enter();
    int bad = 0;
    for (int i = threadIdx.x; i < n; i += KV_PLAN_THREADS) {
        const int s = src[i], d = dst[i];
        if ((unsigned)s >= (unsigned)kv.pages || (unsigned)d >= (unsigned)kv.pages) {
            bad = 1;
        } else {
            kv.mark()[s] = 0;
            kv.mark()[d] = 0;
            kv.copy_src()[i] = s;
            kv.copy_dst()[i] = d;
        }
    }
    int code = __syncthreads_or(bad) ? KV_BAD_PAGE : KV_OK;
    if (code == KV_OK) {
        for (int i = threadIdx.x; i < n; i += KV_PLAN_THREADS)
            if (atomicAdd(&kv.mark()[dst[i]], 1)) bad = 1;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += KV_PLAN_THREADS)
            if (kv.mark()[src[i]]) bad = 1;
        if (__syncthreads_or(bad)) code = KV_BAD_LIST;
    }
    if (threadIdx.x == 0) {
        if (code != KV_OK) atomicCAS(kv.status(), 0, code);
        kv.work[1] = code == KV_OK ? n : 0;
        kv.work[3] = code == KV_OK;
    }
}

/* The plan carried out: tables (fork: a CTA to an entry of the list; compact: a warp to a
 * sequence), then the copies, 16 KB of a page at a time. */
enum : int { KV_APPLY_COPY = 0, KV_APPLY_FORK = 1, KV_APPLY_COMPACT = 2, KV_APPLY_LIST = 3 };
template <int WHAT>
__global__ void __launch_bounds__(KV_APPLY_THREADS)
kv_apply_kernel(KvView kv, const int32_t *__restrict__ src, const int32_t *__restrict__ dst,
                int n) {
    pdl_enter();
    const int tid = threadIdx.x;
    extern __shared__ unsigned kv_bits[];
    if (WHAT == KV_APPLY_LIST) {
        /* the list as it came, checked by every CTA with a bit for each page: one launch less */
        for (int i = tid; i < (kv.pages + 31) / 32; i += KV_APPLY_THREADS) kv_bits[i] = 0;
        __syncthreads();
        int code = KV_OK;
        for (int i = tid; i < n; i += KV_APPLY_THREADS) {
            const unsigned s = src[i], d = dst[i];
            if (s >= (unsigned)kv.pages || d >= (unsigned)kv.pages) code = KV_BAD_PAGE;
            else if (atomicOr(&kv_bits[d >> 5], 1u << (d & 31)) >> (d & 31) & 1)
                code = KV_BAD_LIST;
        }
        __syncthreads();
        for (int i = tid; i < n; i += KV_APPLY_THREADS) {
            const unsigned s = src[i];
            if (s < (unsigned)kv.pages && (kv_bits[s >> 5] >> (s & 31) & 1) && code == KV_OK)
                code = KV_BAD_LIST;
        }
        const bool page = __syncthreads_or(code == KV_BAD_PAGE),
                   list = __syncthreads_or(code == KV_BAD_LIST);
        if (page || list) {
            if (blockIdx.x == 0 && tid == 0)
                atomicCAS(kv.status(), 0, page ? KV_BAD_PAGE : KV_BAD_LIST);
            return;
        }
    } else if (!kv.work[3]) {
        return;
    }
    if (WHAT == KV_APPLY_FORK) {
        for (int i = blockIdx.x; i < n; i += gridDim.x) {
            const int s = src[i], d = dst[i], tokens = kv.len[s];
            const int held = kv.held(tokens), full = tokens / kv.page_tokens;
            for (int j = tid; j < held; j += KV_APPLY_THREADS) {
                int p = kv.table[(size_t)s * kv.max_pages + j];
                if (j >= full) {
                    p = kv.copy_dst()[kv.first()[i]];
                    kv.refs[p] = 1;
                } else if ((unsigned)p < (unsigned)kv.pages) {
                    atomicAdd(&kv.refs[p], 1);
                } else {
                    atomicCAS(kv.status(), 0, KV_BAD_PAGE);
                }
                kv.table[(size_t)d * kv.max_pages + j] = p;
            }
            if (tid == 0) kv.len[d] = tokens;
        }
    }
    if (WHAT == KV_APPLY_COMPACT) {
        const int warps = KV_APPLY_THREADS / 32, live = kv.work[2];
        for (int s = blockIdx.x * warps + (tid >> 5); s < kv.seqs; s += gridDim.x * warps) {
            const int held = kv.held(kv.len[s]);
            for (int j = tid & 31; j < held; j += 32) {
                int32_t *e = &kv.table[(size_t)s * kv.max_pages + j];
                const int p = *e;
                if ((unsigned)p >= (unsigned)kv.pages) atomicCAS(kv.status(), 0, KV_BAD_PAGE);
                else if (p >= live) *e = kv.map()[p];
            }
        }
    }
    const int copies = WHAT == KV_APPLY_LIST ? n : kv.work[1];
    const int32_t *from_page = WHAT == KV_APPLY_LIST ? src : kv.copy_src(),
                  *to_page = WHAT == KV_APPLY_LIST ? dst : kv.copy_dst();
    const int page16 = kv.page_elems / 8;                 /* 16-byte pieces of a page */
    constexpr int UNIT = 4 * KV_APPLY_THREADS;            /* of which a CTA takes these at a time */
    const int units = (page16 + UNIT - 1) / UNIT;
    const long total = (long)copies * kv.layers * 2 * units;
    for (long u = blockIdx.x; u < total; u += gridDim.x) {
        const int part = (int)(u % units);
        long r = u / units;
        uint16_t *pool = r & 1 ? kv.v : kv.k;
        r >>= 1;
        const int layer = (int)(r % kv.layers), i = (int)(r / kv.layers);
        const size_t base = (size_t)layer * kv.pages;
        const uint4 *from =
            reinterpret_cast<const uint4 *>(pool + (base + from_page[i]) * kv.page_elems);
        uint4 *to = reinterpret_cast<uint4 *>(pool + (base + to_page[i]) * kv.page_elems);
        uint4 x[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int at = part * UNIT + j * KV_APPLY_THREADS + tid;
            if (at < page16) x[j] = from[at];
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int at = part * UNIT + j * KV_APPLY_THREADS + tid;
            if (at < page16) to[at] = x[j];
        }
    }
}

}  // namespace apus
