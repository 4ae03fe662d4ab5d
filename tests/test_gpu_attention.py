"""Attention of packed prompts and of single tokens over the paged cache, against 64-bit
softmax sums of the same inputs; rows that see nothing, padded batches, strides, values that
are not finite where nothing may see them, streams and graphs."""
import math

import pytest

pytestmark = pytest.mark.gpu

HEADS = [(16, 2, 256), (32, 8, 128), (20, 4, 128), (12, 12, 64), (16, 1, 128), (6, 2, 64),
         (3, 3, 256), (16, 1, 256)]


def _prompt(gpu, torch, nq, nk, heads, kv_heads, dim, causal=True, gate=True, pad=0, seed=0,
            scale=None, spoil=False):
    import attn_util as u
    import apus_b200.backend as B
    rows, keys = sum(nq) + pad, sum(nk)
    q, g = u.normal(rows, 2, heads, dim, seed=seed, scale=1.5).unbind(1)
    k, v = u.normal(keys + 9, 2, kv_heads, dim, seed=seed + 1).unbind(1)
    if spoil:                       # behind the last key
        k[keys:] = math.nan
        v[keys:] = math.inf
    out = torch.full((rows, heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((rows, heads), 7.0, device="cuda")
    a = u.attn(q, out, lse, g if gate else None, kv_heads=kv_heads, scale=scale)
    cq, ck = u.bounds(nq), u.bounds(nk)
    dq, dk = u.ints(cq), u.ints(ck)
    kk = B.AttnKeys(k=k.data_ptr(), v=v.data_ptr(), k_stride=k.stride(0), v_stride=v.stride(0),
                    rows=keys + 9, cu_q=dq.data_ptr(), cu_k=dk.data_ptr(), seqs=len(nq),
                    causal=int(causal))
    gpu.attn_prompt_dev(a, kk, stream=u.stream())
    torch.cuda.synchronize()
    assert gpu.last_block_status() == 0
    for i in range(len(nq)):
        n, m = nq[i], nk[i]
        limit = torch.full((n,), m, device="cuda")
        if causal:
            limit = (m - n + 1 + torch.arange(n, device="cuda")).clamp(min=0)
        qs, ks = slice(cq[i], cq[i + 1]), slice(ck[i], ck[i + 1])
        ref = u.exact(q[qs], k[ks], v[ks], limit, a.scale, g[qs] if gate else None)
        u.check(out[qs], lse[qs], ref, (i, n, m))
    assert (out[sum(nq):] == 7).all() and (lse[sum(nq):] == 7).all()
    return out, lse


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_packed(gpu, heads, kv_heads, dim, causal):
    import torch
    n = [1, 16, 130, 0, 77, 257]
    _prompt(gpu, torch, n, n, heads, kv_heads, dim, causal, pad=3)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 700])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompt_one(gpu, n, dim):
    import torch
    _prompt(gpu, torch, [n], [n], 8, 1, dim, gate=False, seed=n)


@pytest.mark.parametrize("nq,nk", [([1], [1000]), ([5, 40], [133, 900]), ([100], [0]),
                                   ([200, 3], [150, 3]), ([0, 0], [5, 0]), ([300], [1])])
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 256), (8, 2, 128), (4, 4, 64)])
def test_prompt_keys_before_and_missing(gpu, nq, nk, heads, kv_heads, dim):
    import torch
    _prompt(gpu, torch, nq, nk, heads, kv_heads, dim, seed=3)
    _prompt(gpu, torch, nq, nk, heads, kv_heads, dim, causal=False, seed=4)


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 256), (8, 1, 128), (4, 2, 64),
                                                (5, 1, 128)])
@pytest.mark.parametrize("nq,nk", [([1], [5000]), ([20], [4111]), ([3, 9], [2000, 1]),
                                   ([7, 2], [0, 3001]), ([33], [1024])])
def test_prompt_few_rows_many_keys(gpu, heads, kv_heads, dim, nq, nk):
    """Keys shared by several CTAs: parts that see all, some and no keys of theirs."""
    import torch
    _prompt(gpu, torch, nq, nk, heads, kv_heads, dim, seed=5)
    _prompt(gpu, torch, nq, nk, heads, kv_heads, dim, causal=False, gate=False, seed=6, spoil=True)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompt_many_items(gpu, dim):
    """More tiles than SMs, lengths from one token to many."""
    import torch
    n = [1 + (i * 37) % 400 for i in range(60)] + [1500, 1, 2]
    _prompt(gpu, torch, n, n, 8, 4, dim, pad=100)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompt_large_scores(gpu, dim):
    """Scores in the hundreds, rising along the row: the running maximum moves far."""
    import torch
    _prompt(gpu, torch, [600], [600], 4, 1, dim, scale=2.0)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompt_rising_keys(gpu, dim):
    """Every later block of keys scores higher than all before: what has been summed has to be
    scaled down again and again."""
    import torch
    import attn_util as u
    import apus_b200.backend as B
    n, H = 1024, 4
    q = torch.zeros(n, H, dim, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 8.0
    k = u.normal(n, 1, dim, seed=2)
    k[:, 0, 0] = (torch.arange(n, device="cuda") // 16).bfloat16()
    v = u.normal(n, 1, dim, seed=3)
    out = torch.empty_like(q)
    lse = torch.empty(n, H, device="cuda")
    a = u.attn(q, out, lse, kv_heads=1, scale=0.25)
    cu = u.ints([0, n])
    kk = B.AttnKeys(k=k.data_ptr(), v=v.data_ptr(), rows=n, cu_q=cu.data_ptr(),
                    cu_k=cu.data_ptr(), seqs=1, causal=1)
    gpu.attn_prompt_dev(a, kk, stream=u.stream())
    torch.cuda.synchronize()
    ref = u.exact(q, k, v, torch.arange(1, n + 1, device="cuda"), 0.25)
    u.check(out, lse, ref)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,keys", [(300, 300), (5, 3000), (1, 700)])
@pytest.mark.parametrize("unit", [32.0, 2.0 ** 16])
def test_scores_far_from_zero(gpu, dim, rows, keys, unit):
    """Scores up to 8128 units (2^29), 64 of them apart at least, both signs: a softmax takes the largest
    one, wherever it is, and splits evenly among equal ones.  The products are exact in fp32, so
    that what is left are a weight's rounding and the result's, 2^-8 each, and for lse those of
    (score log2(e) + log2(sum)) ln(2), a step of fp32 each."""
    import torch
    import attn_util as u
    import apus_b200.backend as B
    H, g = 4, torch.Generator().manual_seed(rows)
    q = torch.zeros(rows, H, dim, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 64.0
    k = torch.zeros(keys, 1, dim, dtype=torch.bfloat16, device="cuda")
    k[:, 0, 0] = (torch.randint(-127, 128, (keys,), generator=g) * unit).bfloat16().cuda()
    v = u.normal(keys, 1, dim, seed=1)
    out, lse = torch.empty_like(q), torch.empty(rows, H, device="cuda")
    cq, ck = u.ints([0, rows]), u.ints([0, keys])
    gpu.attn_prompt_dev(u.attn(q, out, lse, kv_heads=1, scale=1.0),
                        B.AttnKeys(k=k.data_ptr(), v=v.data_ptr(), rows=keys, cu_q=cq.data_ptr(),
                                   cu_k=ck.data_ptr(), seqs=1, causal=1), stream=u.stream())
    cache = u.Cache(1, 200, 1, 16, dim, 1, 200).hold([keys])
    pages = cache.table[0, :-(-keys // 16)].long()
    fill = torch.zeros(2, len(pages) * 16, dim, dtype=torch.bfloat16, device="cuda")
    fill[0, :keys], fill[1, :keys] = k[:, 0], v[:, 0]
    cache.k[0, pages, 0], cache.v[0, pages, 0] = fill.view(2, -1, 16, dim).unbind(0)
    one, one_lse = torch.empty_like(q[:1]), torch.empty(1, H, device="cuda")
    gpu.attn_decode_dev(u.attn(q[-1:], one, one_lse, kv_heads=1, scale=1.0), cache.c, 0,
                        stream=u.stream())
    torch.cuda.synchronize()
    assert gpu.last_block_status() == 0 and cache.status() == 0
    score = 64.0 * k[:, 0, 0].double()
    for i in range(rows):
        seen = score[:keys - rows + 1 + i]
        at = (seen == seen.max()).nonzero()[:, 0]
        want, size = v[at, 0].double().mean(0), v[at, 0].double().abs().mean(0)
        want_lse = float(seen.max()) + math.log(len(at))
        for o, l in [(out[i], lse[i])] + ([(one[0], one_lse[0])] if i == rows - 1 else []):
            assert ((o.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -7 * size).all()
            assert ((l.double() - want_lse).abs() <= 2.0 ** -21 * abs(want_lse) + 2.0 ** -20).all()


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 256), (8, 8, 128), (8, 1, 64)])
def test_prompt_not_finite_where_nothing_sees(gpu, heads, kv_heads, dim):
    """NaN and infinity behind the last key, and in the sequences beside a sound one."""
    import torch
    import attn_util as u
    import apus_b200.backend as B
    _prompt(gpu, torch, [50, 100], [50, 100], heads, kv_heads, dim, spoil=True)
    n = [33, 90, 41]
    cu = u.bounds(n)
    q, k, v = (u.normal(sum(n), h, dim, seed=i) for i, h in enumerate((heads, kv_heads, kv_heads)))
    for t in (k, v):
        t[:cu[1]] = math.nan
        t[cu[2]:] = math.inf
    q[cu[2]:] = math.nan
    out = torch.empty_like(q)
    a = u.attn(q, out, kv_heads=kv_heads)
    d = u.ints(cu)
    kk = B.AttnKeys(k=k.data_ptr(), v=v.data_ptr(), rows=sum(n), cu_q=d.data_ptr(),
                    cu_k=d.data_ptr(), seqs=3, causal=1)
    gpu.attn_prompt_dev(a, kk, stream=u.stream())
    torch.cuda.synchronize()
    s = slice(cu[1], cu[2])
    ref = u.exact(q[s], k[s], v[s], torch.arange(1, n[1] + 1, device="cuda"), a.scale)
    u.check(out[s], None, ref)


def _decode(gpu, torch, lengths, heads, kv_heads, dim, page, gate=True, seq=None, layers=1,
            seed=0, scale=None, width=None):
    import attn_util as u
    held = [-(-n // page) for n in lengths]
    cache = u.Cache(layers, sum(held) + 3, kv_heads, page, dim, len(lengths),
                    width or max(held) + 2, seed).hold(lengths, seed)
    # nothing behind a sequence's last token may matter
    inside = torch.zeros(cache.pages, page, dtype=torch.bool, device="cuda")
    for s, n in enumerate(lengths):
        t = torch.arange(n, device="cuda")
        inside[cache.table[s, (t // page)].long(), t % page] = True
    cache.k.transpose(2, 3)[:, ~inside] = math.nan
    cache.v.transpose(2, 3)[:, ~inside] = math.inf
    order = list(range(len(lengths))) if seq is None else seq
    q, g = u.normal(len(order), 2, heads, dim, seed=seed + 5, scale=1.5).unbind(1)
    out = torch.full((len(order), heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((len(order), heads), 7.0, device="cuda")
    a = u.attn(q, out, lse, g if gate else None, kv_heads=kv_heads, scale=scale)
    d = u.ints(order) if seq is not None else None
    gpu.attn_decode_dev(a, cache.c, layers - 1, d.data_ptr() if seq is not None else None,
                        stream=u.stream())
    torch.cuda.synchronize()
    assert cache.status() == 0
    for b, s in enumerate(order):
        if s < 0:
            assert (out[b] == 7).all() and (lse[b] == 7).all()
            continue
        k, v = cache.tokens(layers - 1, s)
        ref = u.exact(q[b:b + 1], k, v, u.ints([lengths[s]]), a.scale,
                      g[b:b + 1] if gate else None)
        u.check(out[b:b + 1], lse[b:b + 1], ref, (b, s, lengths[s]))
    return a, cache, q, g, out, lse, d


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("page", [16, 32, 48, 256])
def test_decode_lengths(gpu, heads, kv_heads, dim, page):
    import torch
    _decode(gpu, torch, [1, 15, 16, 17, 0, 31, 64, 65, 127, 300, 1023], heads, kv_heads, dim, page)


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
def test_decode_long(gpu, heads, kv_heads, dim):
    """One sequence over all SMs; two of very different lengths."""
    import torch
    _decode(gpu, torch, [20011], heads, kv_heads, dim, 64, gate=False, seed=1)
    _decode(gpu, torch, [9000, 3], heads, kv_heads, dim, 16, seed=2)


def test_decode_many_sequences(gpu):
    import torch
    n = [(i * 131) % 900 for i in range(333)]
    _decode(gpu, torch, n, 8, 2, 128, 32)


def test_decode_more_rows_than_a_launch_takes(gpu):
    import torch
    n = [(i * 7) % 40 for i in range(2600)]
    _decode(gpu, torch, n, 4, 2, 64, 16, gate=False)


def test_decode_order_padding_and_repeats(gpu):
    """Rows in another order than the table, rows of no sequence, one sequence twice."""
    import torch
    _decode(gpu, torch, [40, 500, 0, 7], 16, 2, 256, 32, seq=[3, -1, 0, 1, 1, 2, -1, 0], layers=3)


def test_decode_large_scores(gpu):
    import torch
    _decode(gpu, torch, [700, 33], 16, 2, 256, 32, scale=2.0)


def test_decode_bad_pages_and_sequences(gpu):
    """A page number outside of the pool: its tokens are left out, the status says so.  A
    sequence that there is not: its row stays as it is."""
    import torch
    import attn_util as u
    a, cache, q, g, out, lse, d = _decode(gpu, torch, [100, 200], 8, 2, 128, 32)
    k, v = cache.tokens(0, 1)
    cache.table[1, 2] = cache.pages
    out.fill_(7.0)
    gpu.attn_decode_dev(a, cache.c, 0, None, stream=u.stream())
    torch.cuda.synchronize()
    assert cache.status() == 3
    kept = torch.cat([torch.arange(64), torch.arange(96, 200)]).cuda()
    ref = u.exact(q[1:], k[kept], v[kept], u.ints([168]), a.scale, g[1:])
    u.check(out[1:], lse[1:], ref)
    cache.work[0] = 0
    out.fill_(7.0)
    seq = u.ints([5, 0])
    gpu.attn_decode_dev(a, cache.c, 0, seq.data_ptr(), stream=u.stream())
    torch.cuda.synchronize()
    assert cache.status() == 2 and (out[0] == 7).all() and not (out[1] == 7).any()


def test_decode_far_into_a_large_pool(gpu):
    """Elements behind 2^31 of the pool."""
    import torch
    import attn_util as u
    pages, page, K, D = 17000, 256, 2, 256
    if torch.cuda.mem_get_info()[0] < 12e9:
        pytest.skip("not enough memory")
    k = torch.zeros(1, pages, K, page, D, dtype=torch.bfloat16, device="cuda")
    cache = u.Cache(1, 1, K, page, D, 1, 4)
    cache.refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    cache.work = torch.zeros(4 * pages + 100, dtype=torch.int32, device="cuda")
    use = [16999, 0, 16998]
    for i, p in enumerate(use):
        k[0, p] = u.normal(K, page, D, seed=i)
    cache.k = cache.v = k
    cache.table[0, :3] = u.ints(use)
    cache.len[0] = 700
    c = cache.c
    c.k = c.v = k.data_ptr()
    c.refs, c.work, c.pages = cache.refs.data_ptr(), cache.work.data_ptr(), pages
    q = u.normal(1, 16, D, seed=9)
    out = torch.empty_like(q)
    a = u.attn(q, out, kv_heads=K)
    gpu.attn_decode_dev(a, c, 0, None, stream=u.stream())
    torch.cuda.synchronize()
    kk, vv = cache.tokens(0, 0)
    u.check(out, None, u.exact(q, kk, vv, u.ints([700]), a.scale))


def test_same_result_twice_on_streams_and_in_a_graph(gpu):
    """Bit for bit the same: called again, called on two streams at once, replayed from a graph
    after the inputs have changed."""
    import torch
    import attn_util as u
    import apus_b200.backend as B
    a, cache, q, g, out, lse, d = _decode(gpu, torch, [3000, 40, 777], 16, 2, 256, 64, seed=4)
    n = [300, 45]
    pq, pk, pv = (u.normal(sum(n), h, 256, seed=i) for i, h in enumerate((16, 2, 2)))
    pout = torch.empty_like(pq)
    cu = u.ints(u.bounds(n))
    pa = u.attn(pq, pout, kv_heads=2)
    kk = B.AttnKeys(k=pk.data_ptr(), v=pv.data_ptr(), rows=sum(n), cu_q=cu.data_ptr(),
                    cu_k=cu.data_ptr(), seqs=2, causal=1)

    def both(s):
        gpu.attn_prompt_dev(pa, kk, stream=s)
        gpu.attn_decode_dev(a, cache.c, 0, None, stream=s)

    both(u.stream())
    torch.cuda.synchronize()
    first = out.clone(), lse.clone(), pout.clone()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        out.zero_()
        pout.zero_()
        torch.cuda.synchronize()
        gpu.attn_decode_dev(a, cache.c, 0, None, stream=s1.cuda_stream)
        gpu.attn_prompt_dev(pa, kk, stream=s2.cuda_stream)
        gpu.attn_decode_dev(a, cache.c, 0, None, stream=s2.cuda_stream)
        gpu.attn_prompt_dev(pa, kk, stream=s1.cuda_stream)
        torch.cuda.synchronize()
        for x, y in zip(first, (out, lse, pout)):
            assert torch.equal(x, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both(u.stream())
    old = q.clone(), pq.clone()
    q.copy_(-q)
    pq.copy_(-pq)
    graph.replay()
    torch.cuda.synchronize()
    assert not torch.equal(first[0], out) and not torch.equal(first[2], pout)
    q.copy_(old[0])
    pq.copy_(old[1])
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(first, (out, lse, pout)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dim", [64, 256])
def test_not_finite_where_a_row_looks(gpu, dim):
    """NaN and infinity that a row does see come out as they would of the formula."""
    import torch
    import attn_util as u
    import apus_b200.backend as B
    n, H, K = 300, 8, 2
    q, k, v = (u.normal(n, h, dim, seed=i) for i, h in enumerate((H, K, K)))
    q[7, 3, 5] = math.nan                    # one row
    v[20, 1, 9] = math.inf                   # a key of head 1: rows from 20 on
    k[200, 0, 0] = math.nan                  # a key of head 0: rows from 200 on
    out, lse = torch.empty_like(q), torch.empty(n, H, device="cuda")
    a = u.attn(q, out, lse, kv_heads=K)
    cu = u.ints([0, n])
    kk = B.AttnKeys(k=k.data_ptr(), v=v.data_ptr(), rows=n, cu_q=cu.data_ptr(),
                    cu_k=cu.data_ptr(), seqs=1, causal=1)
    gpu.attn_prompt_dev(a, kk, stream=u.stream())
    torch.cuda.synchronize()
    assert out[7, 3].isnan().all() and lse[7, 3].isnan()
    assert out[200:, :4].isnan().all() and lse[200:, :4].isnan().all()
    assert (out[32:, 4:, 9] == math.inf).all()
    fine = torch.ones(n, H, dim, dtype=torch.bool, device="cuda")
    fine[7, 3] = False
    fine[200:, :4] = False
    fine[:, 4:, 9] = False                   # (its tile, 128 / 4 = 32 tokens, has 0 * inf before)
    assert out[fine].isfinite().all() and lse[:200, 4:].isfinite().all()
    cache = u.Cache(1, 14, K, 32, dim, 2, 10).hold([n, 40])
    for s, m in ((0, n), (1, 40)):
        t = torch.arange(m, device="cuda")
        at = cache.table[s, t // 32].long(), t % 32
        cache.k[0].transpose(1, 2)[at] = k[:m]
        cache.v[0].transpose(1, 2)[at] = v[:m]
    q2 = u.normal(2, H, dim, seed=7)
    out2 = torch.empty_like(q2)
    a2 = u.attn(q2, out2, kv_heads=K)
    gpu.attn_decode_dev(a2, cache.c, 0, None, stream=u.stream())
    torch.cuda.synchronize()
    assert out2[0, :4].isnan().all() and not out2[1, :4].isnan().any()
    assert (out2[:, 4:, 9] == math.inf).all()


def test_a_step_in_a_graph(gpu):
    """Places, positions and cache, attention and the end of sequences captured once and replayed:
    the same bits as the calls."""
    import torch
    import attn_util as u
    import apus_b200.backend as B
    H, K, D, page, n = 8, 2, 128, 16, 5
    lengths = [30, 1, 15, 16, 100]

    def make():
        c = u.Cache(1, 40, K, page, D, n, 10, seed=3).hold(lengths, seed=3)
        x = u.normal(n, H + 2 * K, D, seed=4)
        q = torch.empty(n, H, D, dtype=torch.bfloat16, device="cuda")
        t = dict(c=c, x=x, q=q, out=torch.empty_like(q), slot=u.ints([-1] * n),
                 cu=u.ints(range(n + 1)), pos=u.ints([lengths]), gone=u.ints([1, 3]))
        r = B.Rope(q=x.data_ptr(), k=x[:, H:].data_ptr(), v=x[:, H + K:].data_ptr(),
                   q_out=q.data_ptr(), k_out=None, q_stride=x.stride(0), k_stride=x.stride(0),
                   v_stride=x.stride(0), rows=n, heads=H, kv_heads=K, head_dim=D, rot_dim=64,
                   pos=t["pos"].data_ptr(), axes=1, sections=(32,), theta=1e4)
        a = u.attn(q, t["out"], kv_heads=K)

        def step():
            st = u.stream()
            gpu.kv_extend_dev(c.c, None, t["cu"].data_ptr(), n, t["slot"].data_ptr(), n, stream=st)
            gpu.rope_dev(r, c.c, 0, t["slot"].data_ptr(), stream=st)
            gpu.attn_decode_dev(a, c.c, 0, None, stream=st)
            gpu.kv_free_dev(c.c, t["gone"].data_ptr(), 2, stream=st)
            gpu.kv_compact_dev(c.c, stream=st)
        return t, step

    one, step = make()
    for _ in range(4):
        step()
    torch.cuda.synchronize()
    two, step2 = make()
    graph = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=s):
        step2()
    for _ in range(4):
        graph.replay()
    torch.cuda.synchronize()
    assert one["c"].status() == 0 and two["c"].status() == 0
    for x, y in zip(one["c"].state() + [one["out"], one["c"].k, one["c"].v],
                    two["c"].state() + [two["out"], two["c"].k, two["c"].v]):
        assert torch.equal(x, y)


def _no_key(out, lse):
    return bool((out == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 256), (8, 2, 128), (16, 1, 64)])
@pytest.mark.parametrize("nq,nk,launches", [([7, 2], [0, 3001], 2), ([40, 1], [30, 4000], 2),
                                            ([200, 3], [150, 3], 1), ([90], [0], 1)])
def test_prompt_rows_without_keys_beside_a_gate_that_is_not_finite(gpu, heads, kv_heads, dim, nq,
                                                                   nk, launches):
    """Zeros and -inf whatever the gate is, with shared keys and without."""
    import torch
    import attn_util as u
    import apus_b200.backend as B
    rows, keys = sum(nq), sum(nk)
    q, g = u.normal(rows, 2, heads, dim, seed=1).unbind(1)
    k, v = u.normal(keys + 1, 2, kv_heads, dim, seed=2).unbind(1)
    blind = max(0, nq[0] - nk[0])            # the first sequence's first rows
    for i, x in enumerate((math.nan, math.inf, -math.inf)):
        g[i:blind:3] = x
    out, lse = torch.full_like(q, 7.0).contiguous(), torch.full((rows, heads), 7.0, device="cuda")
    cq, ck = u.ints(u.bounds(nq)), u.ints(u.bounds(nk))
    a = u.attn(q, out, lse, g, kv_heads=kv_heads)
    before = gpu.launches()
    gpu.attn_prompt_dev(a, B.AttnKeys(k=k.data_ptr(), v=v.data_ptr(), k_stride=k.stride(0),
                                      v_stride=v.stride(0), rows=keys, cu_q=cq.data_ptr(),
                                      cu_k=ck.data_ptr(), seqs=len(nq), causal=1),
                        stream=u.stream())
    torch.cuda.synchronize()
    assert gpu.launches() - before == launches
    assert _no_key(out[:blind], lse[:blind])
    at = 0
    for i, (n, m) in enumerate(zip(nq, nk)):
        s = slice(at + max(0, n - m), at + n)
        limit = m - (s.stop - s.start) + 1 + torch.arange(s.stop - s.start, device="cuda")
        ks = slice(sum(nk[:i]), sum(nk[:i + 1]))
        if s.stop > s.start:
            u.check(out[s], lse[s], u.exact(q[s], k[ks], v[ks], limit, a.scale, g[s]))
        at += n


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 256), (8, 2, 128), (16, 1, 64)])
@pytest.mark.parametrize("lengths", [[10, 40], [20, 33], [3000, 50], [700] + [9] * 150,
                                     [9] + [1500] * 64, [9000] + [16] * 20])
def test_decode_rows_without_a_page_beside_a_gate_that_is_not_finite(gpu, heads, kv_heads, dim,
                                                                     lengths):
    """All page numbers of a sequence outside of the pool: zeros and -inf whatever the gate is, where one
    warp, one SM and several of them sum such a row up; the others are what they would be."""
    import torch
    import attn_util as u
    page, n = 16, len(lengths)
    held = [-(-m // page) for m in lengths]
    cache = u.Cache(1, sum(held) + 1, kv_heads, page, dim, n, max(held) + 1).hold(lengths)
    bad = [0] + list(range(3, n, 5))
    for s in bad:
        cache.table[s] = cache.pages + s
    q, g = u.normal(n, 2, heads, dim, seed=3).unbind(1)
    for i, s in enumerate(bad):
        g[s] = (math.nan, math.inf, -math.inf)[i % 3]
    out, lse = torch.full_like(q, 7.0).contiguous(), torch.full((n, heads), 7.0, device="cuda")
    a = u.attn(q, out, lse, g, kv_heads=kv_heads)
    gpu.attn_decode_dev(a, cache.c, 0, None, stream=u.stream())
    torch.cuda.synchronize()
    assert cache.status() == 3
    assert _no_key(out[bad], lse[bad])
    for s in (1, 2, n - 1):
        if s < n and s not in bad:
            k, v = cache.tokens(0, s)
            u.check(out[s:s + 1], lse[s:s + 1], u.exact(q[s:s + 1], k, v, u.ints([lengths[s]]),
                                                        a.scale, g[s:s + 1]))


@pytest.mark.parametrize("heads,kv_heads,dim,lengths", [(16, 2, 256, [977]), (8, 1, 128, [20011]),
                                                        (6, 2, 64, [3000, 700, 41])])
def test_parts_of_other_sms_are_of_this_call(gpu, heads, kv_heads, dim, lengths):
    """Two queries in turns, many times with nothing between: every result has the bits that it has
    alone, so no value of the call before passes as this one's."""
    import torch
    import attn_util as u
    n = len(lengths)
    held = [-(-m // 32) for m in lengths]
    cache = u.Cache(1, sum(held) + 1, kv_heads, 32, dim, n, max(held) + 1).hold(lengths)
    qs = [u.normal(n, heads, dim, seed=s) for s in (1, 2)]
    outs = [torch.empty_like(q) for q in qs]
    lses = [torch.empty(n, heads, device="cuda") for _ in qs]
    calls = [u.attn(*t, kv_heads=kv_heads) for t in zip(qs, outs, lses)]
    want = []
    for c, o, l in zip(calls, outs, lses):
        gpu.attn_decode_dev(c, cache.c, 0, None, stream=u.stream())
        torch.cuda.synchronize()
        want.append((o.clone(), l.clone()))
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(20):
            for c in calls:
                gpu.attn_decode_dev(c, cache.c, 0, None, stream=u.stream())
        for (o, l), (p, m) in zip(zip(outs, lses), want):
            wrong += (o != p).sum() + (l != m).sum()
    for _ in range(100):
        graph.replay()
    for _ in range(200):
        for c, o, l, (p, m) in zip(calls, outs, lses, want):
            gpu.attn_decode_dev(c, cache.c, 0, None, stream=u.stream())
            wrong += (o != p).sum() + (l != m).sum()
    torch.cuda.synchronize()
    assert int(wrong) == 0 and gpu.last_block_status() == 0


def test_decode_at_the_end_of_the_round_counter(gpu):
    """Words of parts that go from SM to SM carry their round, and the counter wraps: neither words
    that nobody has written nor those of a turn ago pass as this call's."""
    import torch
    import attn_util as u
    END = (1 << 32) - 1
    runs = []
    for lengths, kv_heads, seed in (([9000, 700], 2, 1), ([977], 2, 2), ([20], 1, 3)):
        held = [-(-m // 32) for m in lengths]
        cache = u.Cache(1, sum(held), kv_heads, 32, 128, len(lengths), max(held)).hold(lengths)
        q = u.normal(len(lengths), 8 * kv_heads, 128, seed=seed)
        out = torch.empty_like(q)
        runs.append((u.attn(q, out, kv_heads=kv_heads), cache, q, out))

    def run(i):
        a, cache, _, out = runs[i]
        out.fill_(7.0)
        gpu.attn_decode_dev(a, cache.c, 0, None, stream=u.stream())
        torch.cuda.synchronize()
        assert gpu.last_block_status() == 0
        return out.clone()

    gpu.debug_attn_rounds(END - 2)                # nothing has been written yet
    early = [run(0) for _ in range(6)]
    gpu.disable()
    gpu.enable()
    want = [run(i) for i in range(3)]
    k, v = runs[0][1].tokens(0, 0)
    u.check(want[0][:1], None, u.exact(runs[0][2][:1], k, v, u.ints([9000]), 128 ** -0.5))
    assert all(torch.equal(x, want[0]) for x in early)
    for clearing in (0x40000000, 0xbfffffff):
        gpu.debug_attn_rounds(1000)
        old = runs[0][2].clone()
        runs[0][2].copy_(-old)
        assert not torch.equal(run(0), want[0])   # words of rounds 1001 to 1004
        run(0), run(0), run(0)
        runs[0][2].copy_(old)
        gpu.debug_attn_rounds(clearing - 2)       # one CTA, which clears the words of all
        for _ in range(4):
            assert torch.equal(run(2), want[2])
        gpu.debug_attn_rounds(1000)
        for i in (0, 1, 0, 0):
            assert torch.equal(run(i), want[i])
        gpu.debug_attn_rounds(clearing - 3)       # and launches that clear and sum up
        for i in (0, 1, 0, 0, 1, 0):
            assert torch.equal(run(i), want[i])
    gpu.debug_attn_rounds(END - 3)
    for i in (0, 1, 0, 0, 1, 2, 0):
        assert torch.equal(run(i), want[i])


def _with_a_cta_that_gives_up(gpu, torch, call, results, cta, codes):
    import time
    call()
    torch.cuda.synchronize()
    want = [r.clone() for r in results]
    assert gpu.last_block_status() == 0
    gpu.debug_attn_absent(cta)
    t = time.monotonic()
    call()
    torch.cuda.synchronize()
    took = time.monotonic() - t
    assert gpu.last_block_status() in codes
    assert took < 10, took                   # a few limits of about a second, not one for each copy
    for _ in range(3):
        for r in results:
            r.fill_(7.0)
        call()
        torch.cuda.synchronize()
        assert gpu.last_block_status() == 0
        assert all(torch.equal(r, w) for r, w in zip(results, want))


@pytest.mark.parametrize("heads,kv_heads,dim,lengths,cta", [
    (16, 2, 256, [20011], 5), (8, 1, 128, [20011], 0), (12, 12, 64, [1500] * 64, 147),
    (16, 1, 256, [700, 9000], 30), (6, 2, 64, [20], 0)])
def test_decode_with_keys_that_never_come(gpu, heads, kv_heads, dim, lengths, cta):
    """A CTA that asks for no keys: its waits for them and the others' for its parts run out, the
    status says so, and the next calls are right."""
    import torch
    import attn_util as u
    n = len(lengths)
    held = [-(-m // 32) for m in lengths]
    cache = u.Cache(1, sum(held), kv_heads, 32, dim, n, max(held)).hold(lengths)
    q = u.normal(n, heads, dim, seed=1)
    out, lse = torch.empty_like(q), torch.empty(n, heads, device="cuda")
    a = u.attn(q, out, lse, kv_heads=kv_heads)
    _with_a_cta_that_gives_up(gpu, torch, lambda: gpu.attn_decode_dev(
        a, cache.c, 0, None, stream=u.stream()), [out, lse], cta, (1, 4))


@pytest.mark.parametrize("heads,kv_heads,dim,nq,nk,cta", [
    (16, 2, 256, [900, 70], [900, 70], 3), (32, 8, 128, [3000], [3000], 100),
    (8, 2, 64, [700], [700], 0), (16, 2, 256, [20], [9000], 7), (16, 2, 256, [77], [77], 1),
    (12, 12, 64, [33], [5000], 0)])
def test_prompt_with_keys_that_never_come(gpu, heads, kv_heads, dim, nq, nk, cta):
    """A CTA whose loads end in the middle of a tile: no MMA, load or wait outlives it, the status
    says so, and the next calls are right."""
    import torch
    import attn_util as u
    import apus_b200.backend as B
    q, g = u.normal(sum(nq), 2, heads, dim, seed=1).unbind(1)
    k, v = u.normal(sum(nk), 2, kv_heads, dim, seed=2).unbind(1)
    out = torch.empty(sum(nq), heads, dim, dtype=torch.bfloat16, device="cuda")
    lse = torch.empty(sum(nq), heads, device="cuda")
    cq, ck = u.ints(u.bounds(nq)), u.ints(u.bounds(nk))
    a = u.attn(q, out, lse, g, kv_heads=kv_heads)
    kk = B.AttnKeys(k=k.data_ptr(), v=v.data_ptr(), k_stride=k.stride(0), v_stride=v.stride(0),
                    rows=sum(nk), cu_q=cq.data_ptr(), cu_k=ck.data_ptr(), seqs=len(nq), causal=1)
    _with_a_cta_that_gives_up(gpu, torch, lambda: gpu.attn_prompt_dev(a, kk, stream=u.stream()),
                              [out, lse], cta, (2,))


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 256), (32, 8, 128), (8, 2, 64)])
def test_prompt_short_sequences_do_not_share_keys(gpu, heads, kv_heads, dim):
    """Where the caller says how long the longest sequence is, keys are shared only if a tile has
    enough of them for two CTAs, however many they are together.  A number that is too small or too
    large changes nothing of the result but the order of its sums."""
    import torch
    import attn_util as u
    import apus_b200.backend as B
    for nq, nk, longest, launches in (([1] * 8, [200] * 8, 200, 1), ([5, 40], [133, 870], 870, 1),
                                      ([5, 40], [133, 900], 900, 2),        # (eight steps)
                                      ([1], [1600], 1600, 2), ([1], [1600], 0, 2),
                                      ([1, 1], [2000, 3], 2000, 2), ([1, 1], [2000, 3], 17, 1),
                                      ([1, 1], [2000, 3], 0xffffffff, 2)):
        q, k, v = (u.normal(sum(n), h, dim, seed=i) for i, (n, h) in
                   enumerate(((nq, heads), (nk, kv_heads), (nk, kv_heads))))
        out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
        cq, ck = u.bounds(nq), u.bounds(nk)
        dq, dk = u.ints(cq), u.ints(ck)
        a = u.attn(q, out, lse, kv_heads=kv_heads)
        before = gpu.launches()
        gpu.attn_prompt_dev(a, B.AttnKeys(k=k.data_ptr(), v=v.data_ptr(), rows=sum(nk),
                                          cu_q=dq.data_ptr(), cu_k=dk.data_ptr(), seqs=len(nq),
                                          causal=1, longest=longest), stream=u.stream())
        torch.cuda.synchronize()
        assert gpu.launches() - before == launches, (nk, longest)
        for i in range(len(nq)):
            qs, ks = slice(cq[i], cq[i + 1]), slice(ck[i], ck[i + 1])
            limit = nk[i] - nq[i] + 1 + torch.arange(nq[i], device="cuda")
            u.check(out[qs], lse[qs], u.exact(q[qs], k[ks], v[ks], limit, a.scale))


def _counted(n, dim, turn):
    """Which value of a head counts a token: those of 16 tokens the same one, and another pairing
    of such tiles with each turn."""
    import torch
    tile = torch.arange(n, device="cuda") // 16
    return (tile + turn * 37 * (tile // dim)) % dim


def _check_counts(out, lse, limit, code, dim):
    """Equal scores: a value is the share of its tokens, lse the logarithm of their number.  Counts
    are exact in fp32 (weights of one, below 2^24); what is left are the division and the product, 2 and
    1/2 steps of 2^-23, and the narrowing, 2^-8; and for log2 and the product with ln(2) a step of fp32
    each, of values below 2^4: 2 * 2^-20 at most.  A tile of 16 tokens more or less is 16 of
    the 16 * (tiles / dim + 1) that its value counts."""
    import torch
    hot = torch.nn.functional.one_hot(code, dim).double().cumsum(0)
    for i, n in enumerate(limit):
        want = hot[n - 1] / n
        assert ((out[i].double() - want).abs() <= (2.0 ** -8 + 2.0 ** -21) * want).all(), (i, n)
        assert ((lse[i].double() - math.log(n)).abs() <= 2.0 ** -19).all(), (i, n)


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("lengths", [[20011], [9000, 3], [1500] * 9 + [40, 16, 700], [130] * 90,
                                     [5003, 17, 30000]])
def test_decode_counts_every_tile_once(gpu, heads, kv_heads, dim, lengths):
    import torch
    import attn_util as u
    page, n = 32, len(lengths)
    held = [-(-m // page) for m in lengths]
    cache = u.Cache(1, sum(held) + 1, kv_heads, page, dim, n, max(held) + 1).hold(lengths)
    q = torch.zeros(n, heads, dim, dtype=torch.bfloat16, device="cuda")
    for turn in (0, 1):
        codes = [_counted(m, dim, turn) for m in lengths]
        cache.v.fill_(math.nan)
        for s, c in enumerate(codes):
            t = torch.arange(lengths[s], device="cuda")
            hot = torch.nn.functional.one_hot(c, dim).bfloat16()
            cache.v[0].transpose(1, 2)[cache.table[s][t // page].long(), t % page] = \
                hot[:, None].expand(-1, kv_heads, -1)
        out, lse = torch.full_like(q, 7.0), torch.full((n, heads), 7.0, device="cuda")
        gpu.attn_decode_dev(u.attn(q, out, lse, kv_heads=kv_heads), cache.c, 0, None,
                            stream=u.stream())
        torch.cuda.synchronize()
        assert cache.status() == 0 and gpu.last_block_status() == 0
        for s, c in enumerate(codes):
            _check_counts(out[s:s + 1], lse[s:s + 1], [lengths[s]], c, dim)


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("nq,nk,launches", [([1], [20011], 2), ([33], [5000], 2),
                                            ([3, 9], [2000, 1800], 2), ([300], [3000], None),
                                            ([700, 90], [700, 2500], None)])
def test_prompt_counts_every_tile_once(gpu, heads, kv_heads, dim, nq, nk, launches):
    import torch
    import attn_util as u
    import apus_b200.backend as B
    q = torch.zeros(sum(nq), heads, dim, dtype=torch.bfloat16, device="cuda")
    k = u.normal(sum(nk), kv_heads, dim)
    cq, ck = u.bounds(nq), u.bounds(nk)
    dq, dk = u.ints(cq), u.ints(ck)
    for turn in (0, 1):
        codes = [_counted(m, dim, turn) for m in nk]
        v = torch.nn.functional.one_hot(torch.cat(codes), dim).bfloat16()[:, None].expand(
            -1, kv_heads, -1).contiguous()
        out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
        before = gpu.launches()
        gpu.attn_prompt_dev(u.attn(q, out, lse, kv_heads=kv_heads),
                            B.AttnKeys(k=k.data_ptr(), v=v.data_ptr(), rows=sum(nk),
                                       cu_q=dq.data_ptr(), cu_k=dk.data_ptr(), seqs=len(nq),
                                       causal=1), stream=u.stream())
        torch.cuda.synchronize()
        assert gpu.last_block_status() == 0
        assert launches is None or gpu.launches() - before == launches
        for i, c in enumerate(codes):
            s = slice(cq[i], cq[i + 1])
            _check_counts(out[s], lse[s], [nk[i] - nq[i] + 1 + j for j in range(nq[i])], c, dim)


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("lengths", [[5000], [700, 2000, 31], [300] * 150])
def test_decode_rising_keys(gpu, heads, kv_heads, dim, lengths):
    """Every later tile of keys scores higher than all before, some by less than what a reference
    has to move for and some by more: within a warp, between warps and between SMs."""
    import torch
    import attn_util as u
    page = 16
    held = [-(-m // page) for m in lengths]
    cache = u.Cache(1, sum(held) + 1, kv_heads, page, dim, len(lengths),
                    max(held) + 1).hold(lengths)
    for s, m in enumerate(lengths):
        t = torch.arange(m, device="cuda")
        # (steps of 1, 2 and 4 times 2 = 8 * 0.25, and those are powers of e)
        cache.k[0].transpose(1, 2)[cache.table[s][t // page].long(), t % page, :, 0] = \
            (t // 16).bfloat16()[:, None]
    q = torch.zeros(len(lengths), heads, dim, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = torch.tensor([8.0, 1.0, -8.0], device="cuda").bfloat16().repeat(heads)[:heads]
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
    a = u.attn(q, out, lse, kv_heads=kv_heads, scale=0.25)
    gpu.attn_decode_dev(a, cache.c, 0, None, stream=u.stream())
    torch.cuda.synchronize()
    assert cache.status() == 0
    for s in range(min(3, len(lengths))):
        k, v = cache.tokens(0, s)
        u.check(out[s:s + 1], lse[s:s + 1],
                u.exact(q[s:s + 1], k, v, u.ints([lengths[s]]), 0.25))
