/*
 * attention_abi.h — C-ABI of the attention half's operators (include/backend_cuda.h): checks
 * of arguments, views for the kernels, launches.  Part of backend_cuda.cu, which holds the
 * context, the order of calls on different streams and the error text.
 */
#pragma once

/* calls run on the backend's device whatever the thread's current one is */
struct DeviceGuard {
    int old = -1;
    bool changed = false;
    explicit DeviceGuard(int device) {
        if (cudaGetDevice(&old) == cudaSuccess && old != device)
            changed = cudaSetDevice(device) == cudaSuccess;
    }
    ~DeviceGuard() {
        if (changed) cudaSetDevice(old);
    }
};

static bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

static int kv_view(const ApusCudaKvCache *kv, const char *what, KvView *out) {
    if (!kv || !kv->k || !kv->v || !kv->refs || !kv->table || !kv->len || !kv->work)
        return fail("%s: the cache has a null pointer", what);
    if (!kv->layers || !kv->pages || !kv->kv_heads || !kv->seqs || !kv->max_pages)
        return fail("%s: the cache has a zero size", what);
    if (!kv->page_tokens || kv->page_tokens % 16 || kv->page_tokens > 256)
        return fail("%s: page_tokens must be a multiple of 16, at most 256", what);
    if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256)
        return fail("%s: head_dim must be 64, 128 or 256", what);
    if (!aligned16(kv->k) || !aligned16(kv->v))
        return fail("%s: the pools must be 16-byte aligned", what);
    const size_t most = 0x7fffffff;
    if (kv->kv_heads > 1024 || kv->pages > most / (kv->page_tokens * kv->kv_heads) ||
        kv->max_pages > most / kv->page_tokens || kv->layers > 65536 ||
        kv->seqs > (size_t)KV_MAX_SEQS || kv->max_pages > most / kv->seqs ||
        kv->kv_heads * kv->page_tokens > most / kv->head_dim)
        return fail("%s: the cache is too large", what);
    KvView v;
    v.k = kv->k;
    v.v = kv->v;
    v.refs = kv->refs;
    v.table = kv->table;
    v.len = kv->len;
    v.work = kv->work;
    v.layers = (int)kv->layers;
    v.pages = (int)kv->pages;
    v.page_tokens = (int)kv->page_tokens;
    v.seqs = (int)kv->seqs;
    v.max_pages = (int)kv->max_pages;
    v.page_elems = (int)(kv->kv_heads * kv->page_tokens * kv->head_dim);
    *out = v;
    return 0;
}

#define LAUNCH_OK(call)                                                          \
    do {                                                                         \
        cudaError_t e_ = (call);                                                 \
        if (e_ != cudaSuccess) {                                                 \
            cudaGetLastError();                                                  \
            return fail("kernel launch: %s (%s:%d)", cudaGetErrorString(e_),     \
                        __FILE__, __LINE__);                                     \
        }                                                                        \
        g_ctx->launches++;                                                       \
    } while (0)

/* all CTAs at the same time */
template <typename... KArgs, typename... Args>
static cudaError_t launch_coop_k(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem,
                                 cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g_apus_use_pdl ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

static unsigned kv_apply_grid(const Ctx *c) {
    return (unsigned)c->sm_count * (2048 / KV_APPLY_THREADS);
}

extern "C" int apus_cuda_kv_extend_dev(const ApusCudaKvCache *kv, const int32_t *d_seq,
                                       const int32_t *d_cu, size_t n, int32_t *d_slot,
                                       size_t rows, void *stream) {
    KvView v;
    if (kv_view(kv, "kv_extend_dev", &v)) return 1;
    if (!n && (!d_slot || !rows)) return 0;       /* (without a list no row has a place) */
    if ((n && !d_cu) || n > kv->seqs || (d_slot && rows > (1u << 30)))
        return fail("kv_extend_dev: bad args");
    std::lock_guard<std::recursive_mutex> lk(g_mu);
    if (ctx_init()) return 1;
    DeviceGuard dev(g_ctx->device);
    LAUNCH_OK(launch_k(kv_extend_kernel, dim3(1), dim3(KV_PLAN_THREADS), 0, (cudaStream_t)stream,
                       v, d_seq, d_cu, (int)n, d_slot, (int)rows));
    return 0;
}

extern "C" int apus_cuda_kv_free_dev(const ApusCudaKvCache *kv, const int32_t *d_seq, size_t n,
                                     void *stream) {
    KvView v;
    if (kv_view(kv, "kv_free_dev", &v)) return 1;
    if (!n) return 0;
    if (n > (1u << 30) || (!d_seq && n > kv->seqs)) return fail("kv_free_dev: bad args");
    std::lock_guard<std::recursive_mutex> lk(g_mu);
    if (ctx_init()) return 1;
    DeviceGuard dev(g_ctx->device);
    const size_t most = (size_t)g_ctx->sm_count * 16;
    LAUNCH_OK(launch_k(kv_free_kernel, dim3((unsigned)(n < most ? n : most)), dim3(128), 0,
                       (cudaStream_t)stream, v, d_seq, (int)n));
    return 0;
}

extern "C" int apus_cuda_kv_fork_dev(const ApusCudaKvCache *kv, const int32_t *d_src,
                                     const int32_t *d_dst, size_t n, void *stream) {
    KvView v;
    if (kv_view(kv, "kv_fork_dev", &v)) return 1;
    if (!n) return 0;
    if (!d_src || !d_dst || n > kv->seqs) return fail("kv_fork_dev: bad args");
    std::lock_guard<std::recursive_mutex> lk(g_mu);
    if (ctx_init()) return 1;
    DeviceGuard dev(g_ctx->device);
    cudaStream_t st = (cudaStream_t)stream;
    LAUNCH_OK(launch_k(kv_fork_plan_kernel, dim3(1), dim3(KV_PLAN_THREADS), 0, st, v, d_src,
                       d_dst, (int)n));
    LAUNCH_OK(launch_k(kv_apply_kernel<KV_APPLY_FORK>, dim3(kv_apply_grid(g_ctx)),
                       dim3(KV_APPLY_THREADS), 0, st, v, d_src, d_dst, (int)n));
    return 0;
}

extern "C" int apus_cuda_kv_compact_dev(const ApusCudaKvCache *kv, void *stream) {
    KvView v;
    if (kv_view(kv, "kv_compact_dev", &v)) return 1;
    std::lock_guard<std::recursive_mutex> lk(g_mu);
    if (ctx_init()) return 1;
    DeviceGuard dev(g_ctx->device);
    cudaStream_t st = (cudaStream_t)stream;
    const int32_t *none = nullptr;
    LAUNCH_OK(launch_k(kv_compact_plan_kernel, dim3(1), dim3(KV_PLAN_THREADS), 0, st, v));
    LAUNCH_OK(launch_k(kv_apply_kernel<KV_APPLY_COMPACT>, dim3(kv_apply_grid(g_ctx)),
                       dim3(KV_APPLY_THREADS), 0, st, v, none, none, 0));
    return 0;
}

extern "C" int apus_cuda_kv_copy_dev(const ApusCudaKvCache *kv, const int32_t *d_src,
                                     const int32_t *d_dst, size_t n, void *stream) {
    KvView v;
    if (kv_view(kv, "kv_copy_dev", &v)) return 1;
    if (!n) return 0;
    if (!d_src || !d_dst || n > kv->pages) return fail("kv_copy_dev: bad args");
    std::lock_guard<std::recursive_mutex> lk(g_mu);
    if (ctx_init()) return 1;
    DeviceGuard dev(g_ctx->device);
    cudaStream_t st = (cudaStream_t)stream;
    if (n <= KV_CHECK_LIST && v.pages <= KV_CHECK_PAGES) {
        LAUNCH_OK(launch_k(kv_apply_kernel<KV_APPLY_LIST>, dim3(kv_apply_grid(g_ctx)),
                           dim3(KV_APPLY_THREADS), ((size_t)v.pages + 31) / 32 * 4, st, v, d_src,
                           d_dst, (int)n));
        return 0;
    }
    LAUNCH_OK(launch_k(kv_copy_plan_kernel, dim3(1), dim3(KV_PLAN_THREADS), 0, st, v, d_src,
                       d_dst, (int)n));
    LAUNCH_OK(launch_k(kv_apply_kernel<KV_APPLY_COPY>, dim3(kv_apply_grid(g_ctx)),
                       dim3(KV_APPLY_THREADS), 0, st, v, d_src, d_dst, (int)n));
    return 0;
}

/* a tensor of rows: its stride, or 0 where it is none that the kernels can read */
static long row_stride(const void *p, size_t stride, size_t heads, size_t head_dim) {
    const size_t s = stride ? stride : heads * head_dim;
    if (!p || !aligned16(p) || s % 8 || s < heads * head_dim || s > ((size_t)1 << 32)) return 0;
    return (long)s;
}

static int heads_check(const char *what, size_t heads, size_t kv_heads, size_t head_dim) {
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return fail("%s: head_dim must be 64, 128 or 256", what);
    if (!heads || !kv_heads || heads % kv_heads || heads / kv_heads > 16 || kv_heads > 1024)
        return fail("%s: heads must be a multiple of kv_heads, at most 16 times as many", what);
    return 0;
}

extern "C" int apus_cuda_rope_dev(const ApusCudaRope *r, const ApusCudaKvCache *kv, size_t layer,
                                  const int32_t *d_slot, void *stream) {
    if (!r) return fail("rope_dev: bad args");
    if (heads_check("rope_dev", r->heads, r->kv_heads, r->head_dim)) return 1;
    if (!r->rot_dim || r->rot_dim % 16 || r->rot_dim > r->head_dim)
        return fail("rope_dev: rot_dim must be a multiple of 16, at most head_dim");
    if (!r->axes || r->axes > 4 || !(r->theta >= 1.0) || r->theta > 1e30)
        return fail("rope_dev: 1 to 4 axes and a theta of 1 to 1e30");
    RopeParams p = {};
    const size_t pairs = r->rot_dim / 2;
    size_t count[4] = {}, sum = 0;
    for (size_t a = 0; a < r->axes; a++) {
        if (r->sections[a] > pairs) return fail("rope_dev: sections must add up to rot_dim / 2");
        sum += r->sections[a];
    }
    if (sum != pairs) return fail("rope_dev: sections must add up to rot_dim / 2");
    /* theta^(-2 i / rot_dim) / 2 pi, as products of 64 bits: a last bit of a double at most */
    const long double ratio = powl((long double)r->theta, -2.0L / (long double)r->rot_dim);
    long double turns = 1.0L / 6.283185307179586476925286766559L;
    for (size_t i = 0, a = 0, in = 0; i < pairs; i++) {
        if (r->interleaved) {
            a = i % r->axes;
            if (count[a] >= r->sections[a]) a = 0;
        } else {
            while (in >= r->sections[a]) {
                a++;
                in = 0;
            }
            in++;
        }
        count[a]++;
        p.axis[i] = (unsigned char)a;
        p.turns[i] = (double)turns;
        turns *= ratio;
    }
    for (size_t a = 0; a < r->axes; a++)
        if (count[a] != r->sections[a])
            return fail("rope_dev: the sections cannot be interleaved over these axes");
    KvView v = {};
    if (kv) {
        if (kv_view(kv, "rope_dev", &v)) return 1;
        if (kv->kv_heads != r->kv_heads || kv->head_dim != r->head_dim || layer >= kv->layers)
            return fail("rope_dev: the cache has other heads or fewer layers");
    }
    if (!r->rows) return 0;
    if (r->rows > (1u << 30) || !r->pos || (kv && !d_slot)) return fail("rope_dev: bad args");
    p.q_stride = row_stride(r->q, r->q_stride, r->heads, r->head_dim);
    p.k_stride = row_stride(r->k, r->k_stride, r->kv_heads, r->head_dim);
    p.q_out_stride = row_stride(r->q_out, r->q_out_stride, r->heads, r->head_dim);
    p.k_out_stride = r->k_out ? row_stride(r->k_out, r->k_out_stride, r->kv_heads, r->head_dim) : 1;
    p.v_stride = kv ? row_stride(r->v, r->v_stride, r->kv_heads, r->head_dim) : 1;
    if (!p.q_stride || !p.k_stride || !p.q_out_stride || !p.k_out_stride || !p.v_stride ||
        (!kv && !r->k_out))
        return fail("rope_dev: a tensor is missing, or its address or stride is not a multiple "
                    "of 16 bytes or less than a row");
    if ((r->q == r->q_out && p.q_stride != p.q_out_stride) ||
        (r->k == r->k_out && p.k_stride != p.k_out_stride))
        return fail("rope_dev: in place needs equal strides");
    p.q = r->q;
    p.k = r->k;
    p.v = r->v;
    p.q_out = r->q_out;
    p.k_out = r->k_out;
    p.rows = (int)r->rows;
    p.heads = (int)r->heads;
    p.kv_heads = (int)r->kv_heads;
    p.head_dim = (int)r->head_dim;
    p.rot = (int)r->rot_dim;
    p.pos = r->pos;
    if (kv) {
        p.slot = d_slot;
        const size_t at = layer * kv->pages * (size_t)v.page_elems;
        p.cache_k = kv->k + at;
        p.cache_v = kv->v + at;
        p.page_tokens = v.page_tokens;
        p.pages = v.pages;
        p.status = kv->work;
    }
    std::lock_guard<std::recursive_mutex> lk(g_mu);
    if (ctx_init()) return 1;
    DeviceGuard dev(g_ctx->device);
    /* warps to a token: as many as its vectors are worth, while there are SMs without any */
    const size_t vectors = r->heads + r->kv_heads * (kv ? 2 : 1), at_once = 256 / r->head_dim;
    size_t split = 1;
    while (2 * split * at_once <= vectors && r->rows * split < 8 * (size_t)g_ctx->sm_count) split *= 2;
    p.split = (int)split;
    constexpr size_t warps = ROPE_THREADS / 32;
    const dim3 grid((unsigned)((r->rows * split + warps - 1) / warps));
    cudaStream_t st = (cudaStream_t)stream;
    if (r->head_dim == 64) LAUNCH_OK(launch_k(rope_kernel<64>, grid, dim3(ROPE_THREADS), 0, st, p));
    else if (r->head_dim == 128)
        LAUNCH_OK(launch_k(rope_kernel<128>, grid, dim3(ROPE_THREADS), 0, st, p));
    else LAUNCH_OK(launch_k(rope_kernel<256>, grid, dim3(ROPE_THREADS), 0, st, p));
    return 0;
}

static int attn_view(const ApusCudaAttn *a, const char *what, AttnView *out) {
    if (heads_check(what, a->heads, a->kv_heads, a->head_dim)) return 1;
    if (!(a->scale > 0.0f) || a->scale > 1e30f) return fail("%s: scale must be positive", what);
    if (a->rows > (1u << 30)) return fail("%s: too many rows", what);
    AttnView v = {};
    v.rows = (int)a->rows;
    v.heads = (int)a->heads;
    v.group = (int)(a->heads / a->kv_heads);
    v.scale = a->scale;
    *out = v;
    if (!a->rows) return 0;
    v.q = a->q;
    v.gate = a->gate;
    v.out = a->out;
    v.lse = a->lse;
    v.q_stride = row_stride(a->q, a->q_stride, a->heads, a->head_dim);
    v.out_stride = row_stride(a->out, a->out_stride, a->heads, a->head_dim);
    v.gate_stride = a->gate ? row_stride(a->gate, a->gate_stride, a->heads, a->head_dim) : 1;
    if (!v.q_stride || !v.out_stride || !v.gate_stride)
        return fail("%s: q, gate or out is missing, or its address or stride is not a multiple "
                    "of 16 bytes or less than a row", what);
    *out = v;
    return 0;
}

/* rows x heads x head_dim values as {64, heads, rows, head_dim / 64} or {64, rows, heads, ...}:
 * boxes of one 128-byte swizzle row by `heads` and `rows` */
static int attn_map(CUtensorMap *m, const uint16_t *base, size_t rows, size_t stride, size_t heads,
                    size_t D, bool heads_first, int box_heads, int box_rows) {
    PFN_encodeTiled_local enc = tensor_map_encoder();
    if (!enc) return fail("%s", prefill_last_error());
    const int h = heads_first ? 1 : 2, r = heads_first ? 2 : 1;
    cuuint64_t dims[4] = {64, 0, 0, (cuuint64_t)(D / 64)}, strides[3] = {0, 0, 128};
    cuuint32_t box[4] = {64, 0, 0, 1}, estr[4] = {1, 1, 1, 1};
    dims[h] = heads;
    dims[r] = rows;
    strides[h - 1] = D * 2;
    strides[r - 1] = stride * 2;
    box[h] = (cuuint32_t)box_heads;
    box[r] = (cuuint32_t)box_rows;
    CUresult e = enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<uint16_t *>(base), dims,
                     strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return e == CUDA_SUCCESS ? 0
                             : fail("attn_prompt_dev: cuTensorMapEncodeTiled failed (%d)", (int)e);
}

template <int D>
static int launch_prompt(Ctx *c, const PromptParams &p, const ApusCudaAttnKeys *keys,
                         long k_stride, long v_stride, cudaStream_t st) {
    CUtensorMap mq, mk, mv;
    /* no key at all: nothing is loaded, any address does */
    const uint16_t *k = keys->rows ? keys->k : p.a.q, *v = keys->rows ? keys->v : p.a.q;
    const size_t rows = keys->rows ? keys->rows : 1;
    if (!keys->rows) k_stride = v_stride = (long)p.kv_heads * D;
    if (attn_map(&mq, p.a.q, p.a.rows, p.a.q_stride, p.a.heads, D, true, p.a.group,
                 p.tile_tokens) ||
        attn_map(&mk, k, rows, k_stride, p.kv_heads, D, false, 1, AP_ROWS) ||
        attn_map(&mv, v, rows, v_stride, p.kv_heads, D, false, 1, ApShape<D>::V_ROWS))
        return 1;
    constexpr int smem = ap_smem_bytes<D>();
    static bool set = false;
    if (!set) {
        const cudaFuncAttribute attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
        CU_OK(cudaFuncSetAttribute(attn_prompt_kernel<D, false>, attr, smem));
        CU_OK(cudaFuncSetAttribute(attn_prompt_kernel<D, true>, attr, smem));
        cudaFuncAttributes one, two;
        CU_OK(cudaFuncGetAttributes(&one, attn_prompt_kernel<D, false>));
        CU_OK(cudaFuncGetAttributes(&two, attn_prompt_kernel<D, true>));
        const int regs = one.numRegs < two.numRegs ? one.numRegs : two.numRegs;
        if (128 * AP_REGS_ISSUE + (AP_THREADS - 128) * AP_REGS_SOFT > AP_THREADS * regs)
            return fail("attn_prompt_dev: built with %d registers a thread, fewer than its warps "
                        "hand over", regs);
        set = true;
    }
    const dim3 grid(p.items < c->sm_count ? p.items : c->sm_count), block(AP_THREADS);
    if (p.splits == 1) {
        LAUNCH_OK(launch_k(attn_prompt_kernel<D, false>, grid, block, smem, st, mq, mk, mv, p));
        return 0;
    }
    LAUNCH_OK(launch_k(attn_prompt_kernel<D, true>, grid, block, smem, st, mq, mk, mv, p));
    LAUNCH_OK(launch_k(attn_prompt_join_kernel<D>, dim3(p.items / p.splits, 4), dim3(256), 0, st,
                       p));
    return 0;
}

extern "C" int apus_cuda_attn_prompt_dev(const ApusCudaAttn *a, const ApusCudaAttnKeys *keys,
                                         void *stream) {
    if (!a || !keys) return fail("attn_prompt_dev: bad args");
    PromptParams p = {};
    if (attn_view(a, "attn_prompt_dev", &p.a)) return 1;
    if (keys->rows > (1u << 30) || keys->seqs > (1u << 24))
        return fail("attn_prompt_dev: too many keys or sequences");
    if (!a->rows || !keys->seqs) return 0;
    if (!keys->cu_q || !keys->cu_k) return fail("attn_prompt_dev: bad args");
    long k_stride = 0, v_stride = 0;
    if (keys->rows) {
        k_stride = row_stride(keys->k, keys->k_stride, a->kv_heads, a->head_dim);
        v_stride = row_stride(keys->v, keys->v_stride, a->kv_heads, a->head_dim);
        if (!k_stride || !v_stride)
            return fail("attn_prompt_dev: k or v is missing, or its address or stride is not a "
                        "multiple of 16 bytes or less than a row");
    }
    p.cu_q = keys->cu_q;
    p.cu_k = keys->cu_k;
    p.k_rows = (int)keys->rows;
    p.seqs = (int)keys->seqs;
    p.causal = keys->causal != 0;
    p.kv_heads = (int)a->kv_heads;
    p.tile_tokens = AP_ROWS / p.a.group;
    const size_t slots = a->rows / p.tile_tokens + keys->seqs;
    if (slots * a->kv_heads > (1u << 30)) return fail("attn_prompt_dev: too many rows");
    p.slots = (int)slots;
    p.items = (int)(slots * a->kv_heads);
    std::lock_guard<std::recursive_mutex> lk(g_mu);
    if (ctx_init()) return 1;
    Ctx *c = g_ctx;
    DeviceGuard dev(c->device);
    cudaStream_t st = (cudaStream_t)stream;
    Ordered ord(c, st);
    if (ord.rc) return 1;
    /* Tiles that leave SMs idle share their keys, by four steps of 128 at least: the second kernel
     * takes as long as two or three.  head_dim 256, 2 key heads: 16 rows over 4096 keys 48 -> 28
     * us, 128 rows over 30128 320 -> 68, one row over 1000 17 -> 16 (head_dim 64: 35 -> 15, 231 ->
     * 39, 12 -> 11).  Where the parts would fill the SMs, their way through memory takes longer than a
     * few steps: 400 rows over 1000 keys 21 -> 26, so only from sixteen steps on.  (Found at 256: at
     * 64 such rows are 26 tiles, which do not fill them, and are shared, 12.5 -> 16.2.)
     *
     * How many steps a tile has is on the device; the caller may say how many keys the longest
     * sequence has.  Else all of them count, which one sequence may hold nearly alone: a row over
     * 4000 beside seven over 50 would take 48 us by the mean, and takes 18.  Where they are even,
     * parts are short or empty without that number: eight rows over 200 keys each 13.1 us, 9.5 with
     * it. */
    const size_t most = keys->longest && keys->longest < keys->rows ? keys->longest : keys->rows;
    const size_t steps = (most + AP_ROWS - 1) / AP_ROWS;
    size_t splits = (size_t)c->sm_count / p.items;
    if (splits > steps / 4) splits = steps / 4;
    if (splits > AP_MAX_SPLITS) splits = AP_MAX_SPLITS;
    if (steps < 16 && 2 * splits * p.items > (size_t)c->sm_count) splits = 1;
    p.splits = splits > 1 ? (int)splits : 1;
    p.items *= p.splits;
    p.parts = c->d_attn_split;
    p.sched = c->d_attn_sync + AD_SYNC_WORDS;
    p.status = c->d_status;
    p.absent = c->attn_absent;
    c->attn_absent = -1;
    if (a->head_dim == 64) return launch_prompt<64>(c, p, keys, k_stride, v_stride, st);
    if (a->head_dim == 128) return launch_prompt<128>(c, p, keys, k_stride, v_stride, st);
    return launch_prompt<256>(c, p, keys, k_stride, v_stride, st);
}

/* rows of head_dim values, 16 tokens of 64 values at a time, 128B swizzle */
static int decode_map(CUtensorMap *m, const uint16_t *base, size_t rows, size_t D) {
    PFN_encodeTiled_local enc = tensor_map_encoder();
    if (!enc) return fail("%s", prefill_last_error());
    cuuint64_t dims[3] = {64, (cuuint64_t)rows, (cuuint64_t)(D / 64)};
    cuuint64_t strides[2] = {(cuuint64_t)D * 2, 128};
    cuuint32_t box[3] = {64, AD_TILE, (cuuint32_t)(D / 64)}, estr[3] = {1, 1, 1};
    CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<uint16_t *>(base), dims,
                     strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : fail("attn_decode_dev: cuTensorMapEncodeTiled failed (%d)", (int)r);
}

template <int D, int NH>
static int launch_decode(Ctx *c, const CUtensorMap &mk, const CUtensorMap &mv, DecodeParams p,
                         cudaStream_t st) {
    const int smem = ad_smem_bytes();
    static bool set = false;
    if (!set) {
        CU_OK(cudaFuncSetAttribute(attn_decode_kernel<D, NH>,
                                   cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        set = true;
    }
    for (int row = 0; row < p.a.rows; row += AD_MAX_ROWS) {
        p.row0 = row;
        p.rows = p.a.rows - row < AD_MAX_ROWS ? p.a.rows - row : AD_MAX_ROWS;
        /* no more CTAs than have a tile for each warp, were all sequences as long as they may be */
        const size_t tiles = (size_t)p.rows * p.kv_heads * p.max_pages * p.page_tiles;
        size_t grid = (tiles + AD_WARPS - 1) / AD_WARPS;
        if (grid > (size_t)c->sm_count) grid = c->sm_count;
        LAUNCH_OK(launch_coop_k(attn_decode_kernel<D, NH>, dim3((unsigned)grid), dim3(AD_THREADS), smem,
                                st, mk, mv, p));
    }
    return 0;
}

extern "C" int apus_cuda_attn_decode_dev(const ApusCudaAttn *a, const ApusCudaKvCache *kv,
                                         size_t layer, const int32_t *d_seq, void *stream) {
    if (!a) return fail("attn_decode_dev: bad args");
    DecodeParams p = {};
    KvView c;
    if (attn_view(a, "attn_decode_dev", &p.a)) return 1;
    if (kv_view(kv, "attn_decode_dev", &c)) return 1;
    if (kv->kv_heads != a->kv_heads || kv->head_dim != a->head_dim || layer >= kv->layers)
        return fail("attn_decode_dev: the cache has other heads or fewer layers");
    if (!d_seq && a->rows > kv->seqs) return fail("attn_decode_dev: more rows than sequences");
    if (!a->rows) return 0;
    p.table = kv->table;
    p.len = kv->len;
    p.seq = d_seq;
    p.status = kv->work;
    p.pages = c.pages;
    p.page_tokens = c.page_tokens;
    p.page_tiles = c.page_tokens / AD_TILE;
    p.seqs = c.seqs;
    p.max_pages = c.max_pages;
    p.kv_heads = (int)kv->kv_heads;
    std::lock_guard<std::recursive_mutex> lk(g_mu);
    if (ctx_init()) return 1;
    Ctx *x = g_ctx;
    DeviceGuard dev(x->device);
    CUtensorMap mk, mv;
    const size_t D = kv->head_dim, at = layer * kv->pages * (size_t)c.page_elems;
    const size_t rows = kv->pages * kv->kv_heads * kv->page_tokens;
    if (decode_map(&mk, kv->k + at, rows, D) || decode_map(&mv, kv->v + at, rows, D)) return 1;
    cudaStream_t st = (cudaStream_t)stream;
    Ordered ord(x, st);
    if (ord.rc) return 1;
    p.wait_status = x->d_status;
    p.shared_parts = x->d_attn_parts;
    p.parts = reinterpret_cast<float *>(x->d_attn_parts +
                                        (size_t)x->sm_count * 2 * AD_SHARED_WORDS);
    p.blocks = x->sm_count;
    p.absent = x->attn_absent;
    x->attn_absent = -1;
    p.sync = x->d_attn_sync;
    const bool wide = p.a.group > 8;
    if (D == 64) return wide ? launch_decode<64, 16>(x, mk, mv, p, st)
                             : launch_decode<64, 8>(x, mk, mv, p, st);
    if (D == 128) return wide ? launch_decode<128, 16>(x, mk, mv, p, st)
                              : launch_decode<128, 8>(x, mk, mv, p, st);
    return wide ? launch_decode<256, 16>(x, mk, mv, p, st)
                : launch_decode<256, 8>(x, mk, mv, p, st);
}

extern "C" int apus_cuda_debug_attn_rounds(uint32_t rounds) {
    std::lock_guard<std::recursive_mutex> lk(g_mu);
    if (ctx_init()) return 1;
    DeviceGuard dev(g_ctx->device);
    CU_OK(cudaDeviceSynchronize());
    CU_OK(cudaMemcpy(g_ctx->d_attn_sync + AD_SYNC_ROUND, &rounds, sizeof rounds,
                     cudaMemcpyHostToDevice));
    return 0;
}
extern "C" int apus_cuda_debug_attn_absent(int cta) {
    std::lock_guard<std::recursive_mutex> lk(g_mu);
    if (ctx_init()) return 1;
    g_ctx->attn_absent = cta;
    return 0;
}
