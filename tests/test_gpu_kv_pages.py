"""The cache's pages (taken, shared, given back, moved together, copied) against a book kept by
hand, rotary positions against 64-bit angles, and the run of all of them as a server makes it."""
import math
import random

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


class Book:
    """The cache's integers and the origin of every page's contents, one step after the other."""

    def __init__(self, cache):
        self.page = cache.page
        self.refs, self.table, self.len = (t.tolist() for t in (cache.refs, cache.table,
                                                                cache.len))
        self.origin = list(range(len(self.refs)))

    def held(self, s):
        return -(-self.len[s] // self.page)

    def extend(self, seq, add):
        need = sum(-(-(self.len[s] + a) // self.page) - self.held(s) for s, a in zip(seq, add))
        if self.refs.count(0) < need:
            return False
        for s, a in zip(seq, add):
            at = self.held(s)
            self.len[s] += a
            for j in range(at, self.held(s)):
                p = self.refs.index(0)
                self.refs[p], self.table[s][j] = 1, p
        return True

    def fork(self, src, dst):
        if self.refs.count(0) < sum(self.len[s] % self.page > 0 for s in src):
            return False
        for s, d in zip(src, dst):
            self.len[d] = self.len[s]
            for j in range(self.held(s)):
                p = self.table[s][j]
                if (j + 1) * self.page > self.len[s]:
                    o = self.origin[p]
                    p = self.refs.index(0)
                    self.origin[p] = o
                    self.refs[p] = 0
                self.refs[p] += 1
                self.table[d][j] = p
        return True

    def free(self, seq):
        for s in seq:
            for j in range(self.held(s)):
                self.refs[self.table[s][j]] -= 1
                self.table[s][j] = -1
            self.len[s] = 0

    def compact(self):
        live = [p for p, r in enumerate(self.refs) if r]
        holes = [p for p in range(len(live)) if not self.refs[p]]
        to = dict(zip([p for p in live if p >= len(live)], holes))
        for p, o in to.items():
            self.refs[o], self.refs[p], self.origin[o] = self.refs[p], 0, self.origin[p]
        for s in range(len(self.len)):
            for j in range(self.held(s)):
                self.table[s][j] = to.get(self.table[s][j], self.table[s][j])

    def check(self, cache, k0, v0):
        import torch
        assert cache.refs.tolist() == self.refs
        assert cache.table.tolist() == self.table
        assert cache.len.tolist() == self.len
        at = torch.tensor(self.origin, device="cuda")
        assert torch.equal(cache.k.view(torch.int16), k0[:, at].view(torch.int16))
        assert torch.equal(cache.v.view(torch.int16), v0[:, at].view(torch.int16))


@pytest.mark.parametrize("pages,page,kv_heads,dim,layers", [
    (50, 16, 2, 256, 3), (333, 32, 1, 64, 1), (2100, 16, 2, 64, 2), (70, 256, 3, 128, 2)])
def test_random_use(gpu, pages, page, kv_heads, dim, layers):
    """A few hundred calls of every kind, refused ones among them, on one cache."""
    import torch
    import attn_util as u
    rng = random.Random(pages)
    seqs, width = 40, max(4, pages // 5)
    cache = u.Cache(layers, pages, kv_heads, page, dim, seqs, width)
    k0, v0 = cache.k.clone(), cache.v.clone()
    book, st = Book(cache), u.stream()
    refused = 0
    for step in range(120):
        what = rng.choice(["extend", "extend", "fork", "free", "compact"])
        if what == "extend":
            seq = rng.sample(range(seqs), rng.randint(1, seqs))
            add = [min(rng.choice([0, 1, page - 1, page, rng.randint(0, 3 * page)]),
                       width * page - book.len[s]) for s in seq]
            cu = [5]
            for a in add:
                cu.append(cu[-1] + a)
            rows = cu[-1] + 4
            slot = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
            ds, dc = u.ints(seq), u.ints(cu)
            before = list(book.len)
            ok = book.extend(seq, add)
            gpu.kv_extend_dev(cache.c, ds.data_ptr(), dc.data_ptr(), len(seq), slot.data_ptr(),
                              rows, stream=st)
            want = [-1] * rows
            if ok:
                for i, s in enumerate(seq):
                    for j in range(add[i]):
                        t = before[s] + j
                        want[cu[i] + j] = book.table[s][t // page] * page + t % page
            assert slot.tolist() == want
        elif what == "fork":
            empty = [s for s in range(seqs) if book.len[s] == 0]
            rng.shuffle(empty)
            n = rng.randint(0, min(6, len(empty)))
            dst = empty[:n]
            src = [rng.choice([s for s in range(seqs) if s not in dst]) for _ in dst]
            if not n:
                continue
            ok = book.fork(src, dst)
            ds, dd = u.ints(src), u.ints(dst)
            gpu.kv_fork_dev(cache.c, ds.data_ptr(), dd.data_ptr(), n, stream=st)
        elif what == "free":
            seq = [rng.randrange(seqs) for _ in range(rng.randint(1, 12))]
            book.free(seq)
            ds = u.ints(seq)
            gpu.kv_free_dev(cache.c, ds.data_ptr(), len(seq), stream=st)
            ok = True
        else:
            book.compact()
            gpu.kv_compact_dev(cache.c, stream=st)
            ok = True
        assert cache.status() == (0 if ok else 1), (step, what)
        refused += not ok
        cache.work[0] = 0
        book.check(cache, k0, v0)
    assert refused or pages > 300


def test_all_sequences_without_a_list(gpu):
    import torch
    import attn_util as u
    cache = u.Cache(1, 64, 1, 16, 64, 8, 8)
    book, k0, v0 = Book(cache), cache.k.clone(), cache.v.clone()
    add = [3, 0, 16, 17, 1, 100, 128, 5]
    cu = u.ints(u.bounds(add))
    gpu.kv_extend_dev(cache.c, None, cu.data_ptr(), 8, stream=u.stream())
    book.extend(range(8), add)
    book.check(cache, k0, v0)
    gpu.kv_free_dev(cache.c, None, 5, stream=u.stream())
    book.free(range(5))
    book.check(cache, k0, v0)
    assert cache.status() == 0


def test_lists_that_are_refused_change_nothing(gpu):
    import torch
    import attn_util as u
    cache = u.Cache(2, 30, 1, 16, 64, 6, 5).hold([20, 33, 0, 0, 16, 0])
    k0, before = cache.k.clone(), cache.state()
    st, one = u.stream(), u.ints([0, 1, 2])

    def refused(code, call, *lists):
        call(*lists)
        assert cache.status() == code
        cache.work[0] = 0
        for x, y in zip(before, cache.state()):
            assert torch.equal(x, y)
        assert torch.equal(k0, cache.k)

    def extend(seq, cu):
        s, c = u.ints(seq), u.ints(cu)
        slot = torch.zeros(4, dtype=torch.int32, device="cuda")
        gpu.kv_extend_dev(cache.c, s.data_ptr(), c.data_ptr(), len(seq), slot.data_ptr(), 4,
                          stream=st)
        assert slot.tolist() == [-1] * 4

    def fork(src, dst):
        s, d = u.ints(src), u.ints(dst)
        gpu.kv_fork_dev(cache.c, s.data_ptr(), d.data_ptr(), len(src), stream=st)

    def copy(src, dst):
        s, d = u.ints(src), u.ints(dst)
        gpu.kv_copy_dev(cache.c, s.data_ptr(), d.data_ptr(), len(src), stream=st)

    refused(2, extend, [1, 1], [0, 1, 2])            # twice
    refused(2, extend, [1, 6], [0, 1, 2])            # no such sequence
    refused(2, extend, [1, -1], [0, 1, 2])
    refused(2, extend, [1, 0], [0, 1, 0])            # shrinks
    refused(2, extend, [2], [0, 81])                 # longer than its row of the table
    refused(2, fork, [0, 1], [2, 2])
    refused(2, fork, [0], [1])                       # not empty
    refused(2, fork, [0, 2], [2, 3])                 # written and read
    refused(2, fork, [7], [2])
    refused(2, fork, [0], [-1])
    refused(3, copy, [0, 30], [1, 2])
    refused(3, copy, [0, -1], [1, 2])
    refused(2, copy, [0, 1], [2, 2])
    refused(2, copy, [0, 1], [1, 2])
    # the sound entries of a list of endings are done, the others say so
    seq = u.ints([9, 0, -3, 0])
    gpu.kv_free_dev(cache.c, seq.data_ptr(), 4, stream=st)
    assert cache.status() == 2 and cache.len.tolist() == [0, 33, 0, 0, 16, 0]
    assert int(cache.refs.sum()) == 4


def test_a_length_beyond_the_table_is_not_forked(gpu):
    import torch
    import attn_util as u
    cache = u.Cache(1, 8, 1, 16, 64, 3, 2)
    cache.len[1] = 33                                     # two pages hold 32
    before, (src, dst) = cache.state(), (u.ints([1]), u.ints([0]))
    gpu.kv_fork_dev(cache.c, src.data_ptr(), dst.data_ptr(), 1, stream=u.stream())
    assert cache.status() == 2
    assert all(torch.equal(x, y) for x, y in zip(before, cache.state()))


@pytest.mark.parametrize("pages,n,layers,kv_heads,page,dim", [
    (400, 190, 3, 2, 32, 128), (12000, 4500, 1, 1, 16, 64), (300000, 40, 1, 1, 16, 64),
    (20, 1, 2, 1, 256, 256)])
def test_copy(gpu, pages, n, layers, kv_heads, page, dim):
    """Short and long lists, small and large pools; a source may go to several pages."""
    import torch
    import attn_util as u
    cache = u.Cache(layers, pages, kv_heads, page, dim, 2, 4)
    want_k, want_v = cache.k.clone(), cache.v.clone()
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).int().cuda()
    src = torch.cat([order[:n // 2], order[:n - n // 2]]).contiguous()
    dst = order[n:2 * n].contiguous()
    want_k[:, dst.long()] = want_k[:, src.long()]
    want_v[:, dst.long()] = want_v[:, src.long()]
    gpu.kv_copy_dev(cache.c, src.data_ptr(), dst.data_ptr(), n, stream=u.stream())
    torch.cuda.synchronize()
    assert cache.status() == 0
    assert torch.equal(cache.k, want_k) and torch.equal(cache.v, want_v)
    if n > 4:
        for bad, code in ((dst.clone(), 2), (src.clone(), 2), (dst.clone(), 3)):
            bad[n - 1] = dst[0] if code == 2 else pages
            gpu.kv_copy_dev(cache.c, src.data_ptr(), bad.data_ptr(), n, stream=u.stream())
            torch.cuda.synchronize()
            assert cache.status() == code
            cache.work[0] = 0
            assert torch.equal(cache.k, want_k) and torch.equal(cache.v, want_v)


def _rope(gpu, torch, T, heads, kv_heads, dim, rot, axes, interleaved, cache=True, in_place=False,
          far=1 << 20, seed=0, k_out=True):
    import attn_util as u
    import apus_b200.backend as B
    rng = np.random.default_rng(seed)
    x = u.normal(T, heads + 2 * kv_heads, dim, seed=seed)
    x0 = x.clone()
    pairs = rot // 2
    sections = [(pairs + axes - 1 - a) // axes for a in range(axes)]
    axis = [i % axes for i in range(pairs)] if interleaved else \
        [a for a, n in enumerate(sections) for _ in range(n)]
    pos = torch.from_numpy(rng.integers(-5, far, (axes, T)).astype(np.int32)).cuda()
    q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    qo = q if in_place else torch.zeros(T, heads, dim, dtype=torch.bfloat16, device="cuda")
    ko = k if in_place else torch.zeros(T, kv_heads, dim, dtype=torch.bfloat16, device="cuda")
    theta = 1e7
    r = B.Rope(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_out=qo.data_ptr(),
               k_out=ko.data_ptr() if k_out else None, q_stride=x.stride(0),
               k_stride=x.stride(0), v_stride=x.stride(0),
               q_out_stride=qo.stride(0) if in_place else 0,
               k_out_stride=ko.stride(0) if in_place else 0, rows=T, heads=heads,
               kv_heads=kv_heads, head_dim=dim, rot_dim=rot, pos=pos.data_ptr(), axes=axes,
               sections=tuple(sections), interleaved=int(interleaved), theta=theta)
    angle = pos.double()[torch.tensor(axis, device="cuda")].t() * \
        theta ** (-2.0 * torch.arange(pairs, device="cuda", dtype=torch.float64) / rot)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    xd = x0[:, :heads + kv_heads].double()
    a, b = xd[..., :pairs], xd[..., pairs:rot]
    ref = torch.cat([a * c - b * s, b * c + a * s, xd[..., rot:]], -1)
    # a turn is off by 2^-24 of one at most (and 2^-24 of the sine), one narrowing to BF16
    tol = 2.0 ** -8 * ref.abs() + 2.0 ** -20 * torch.cat(
        [a.abs() + b.abs(), a.abs() + b.abs(), xd[..., rot:].abs()], -1)
    kv = None
    if cache:
        page = 32
        kv = u.Cache(2, T // page + 5, kv_heads, page, dim, 1, 1, seed)
        want = kv.k.clone(), kv.v.clone()
        slot = torch.from_numpy(rng.permutation(kv.pages * page)[:T].astype(np.int32)).cuda()
        slot[T // 2] = -1
    gpu.rope_dev(r, kv.c if cache else None, 1, slot.data_ptr() if cache else None,
                 stream=u.stream())
    torch.cuda.synchronize()
    assert ((qo.double() - ref[:, :heads]).abs() <= tol[:, :heads]).all()
    assert torch.equal(qo[..., rot:], x0[:, :heads, rot:])
    if k_out:
        assert ((ko.double() - ref[:, heads:]).abs() <= tol[:, heads:]).all()
    assert torch.equal(x0[:, heads + kv_heads:], v)
    if cache:
        assert kv.status() == 0
        for t in range(T):
            at = int(slot[t])
            if at < 0:
                continue
            got = kv.k[1, at // 32, :, at % 32]
            assert ((got.double() - ref[t, heads:]).abs() <= tol[t, heads:]).all()
            if k_out:
                assert torch.equal(got, ko[t])
            want[0][1, at // 32, :, at % 32] = got
            want[1][1, at // 32, :, at % 32] = v[t]
        assert torch.equal(want[0], kv.k) and torch.equal(want[1], kv.v)


@pytest.mark.parametrize("heads,kv_heads,dim,rot", [
    (16, 2, 256, 64), (16, 2, 256, 256), (32, 8, 128, 128), (3, 1, 128, 48), (12, 12, 64, 16),
    (1, 1, 64, 64), (5, 5, 256, 16)])
@pytest.mark.parametrize("T", [1, 7, 131])
def test_rope(gpu, heads, kv_heads, dim, rot, T):
    import torch
    _rope(gpu, torch, T, heads, kv_heads, dim, rot, 1, False)
    _rope(gpu, torch, T, heads, kv_heads, dim, rot, 3, True, seed=1)


@pytest.mark.parametrize("axes,interleaved", [(2, False), (3, False), (4, False), (2, True),
                                              (4, True)])
def test_rope_axes_in_place_and_without_a_cache(gpu, axes, interleaved):
    import torch
    _rope(gpu, torch, 50, 8, 2, 128, 96, axes, interleaved, in_place=True)
    _rope(gpu, torch, 50, 8, 2, 128, 96, axes, interleaved, cache=False, seed=2)
    _rope(gpu, torch, 50, 8, 2, 128, 96, axes, interleaved, k_out=False, seed=3)


def test_rope_many_tokens_and_far_positions(gpu):
    import torch
    _rope(gpu, torch, 3001, 16, 2, 256, 64, 3, True, cache=False, far=2 ** 31 - 1)


def test_rope_places_outside_of_the_pool(gpu):
    import torch
    import attn_util as u
    import apus_b200.backend as B
    x = u.normal(2, 3, 64)
    kv = u.Cache(1, 4, 1, 16, 64, 1, 1)
    k0 = kv.k.clone()
    out = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    pos, slot = u.ints([[1, 2]]), u.ints([64, 3])
    r = B.Rope(q=x.data_ptr(), k=x[:, 1:].data_ptr(), v=x[:, 2:].data_ptr(),
               q_out=out.data_ptr(), k_out=None, q_stride=192, k_stride=192, v_stride=192,
               q_out_stride=128, rows=2, heads=1, kv_heads=1, head_dim=64, rot_dim=64,
               pos=pos.data_ptr(), axes=1, sections=(32,), theta=1e4)
    gpu.rope_dev(r, kv.c, 0, slot.data_ptr(), stream=u.stream())
    torch.cuda.synchronize()
    assert kv.status() == 3
    k0[0, 0, :, 3] = kv.k[0, 0, :, 3]
    assert torch.equal(k0, kv.k)


def test_serving_run(gpu):
    """Two prompts, one of them in two parts and forked after them, then tokens one by one with a
    fork and a compaction between: every row's attention against all keys that its sequence has
    had by then."""
    import torch
    import attn_util as u
    import apus_b200.backend as B
    H, K, D, page, layers = 16, 2, 256, 32, 2
    cache = u.Cache(layers, 64, K, page, D, 6, 12)
    past = [[(torch.zeros(0, K, D, device="cuda"),) * 2 for _ in range(6)] for _ in range(layers)]
    length, st = [0] * 6, u.stream()

    def step(seq, counts, seed):
        """Projections of the new rows of all layers through positions, cache and attention."""
        T, cu = sum(counts), u.ints(u.bounds(counts))
        ds = u.ints(seq)
        slot = torch.zeros(T, dtype=torch.int32, device="cuda")
        gpu.kv_extend_dev(cache.c, ds.data_ptr(), cu.data_ptr(), len(seq), slot.data_ptr(), T,
                          stream=st)
        pos = u.ints([[length[s] + j for s, n in zip(seq, counts) for j in range(n)]])
        for layer in range(layers):
            x = u.normal(T, H + 2 * K, D, seed=seed * 10 + layer)
            q = torch.empty(T, H, D, dtype=torch.bfloat16, device="cuda")
            k = torch.empty(T, K, D, dtype=torch.bfloat16, device="cuda")
            r = B.Rope(q=x.data_ptr(), k=x[:, H:].data_ptr(), v=x[:, H + K:].data_ptr(),
                       q_out=q.data_ptr(), k_out=k.data_ptr(), q_stride=x.stride(0),
                       k_stride=x.stride(0), v_stride=x.stride(0), rows=T, heads=H, kv_heads=K,
                       head_dim=D, rot_dim=64, pos=pos.data_ptr(), axes=1, sections=(32,),
                       theta=1e7)
            gpu.rope_dev(r, cache.c, layer, slot.data_ptr(), stream=st)
            v, out = x[:, H + K:], torch.zeros_like(q)
            at = 0
            for s, n in zip(seq, counts):
                past[layer][s] = tuple(torch.cat([o, y[at:at + n].float()]) for o, y in
                                       zip(past[layer][s], (k, v)))
                at += n
            a = u.attn(q, out, kv_heads=K)
            if max(counts) == 1:
                gpu.attn_decode_dev(a, cache.c, layer, ds.data_ptr(), stream=st)
            else:
                kk, vv = (torch.cat([past[layer][s][i] for s in seq]).bfloat16() for i in (0, 1))
                ck = u.ints(u.bounds([length[s] + n for s, n in zip(seq, counts)]))
                keys = B.AttnKeys(k=kk.data_ptr(), v=vv.data_ptr(), rows=kk.shape[0],
                                  cu_q=cu.data_ptr(), cu_k=ck.data_ptr(), seqs=len(seq), causal=1)
                gpu.attn_prompt_dev(a, keys, stream=st)
            torch.cuda.synchronize()
            at = 0
            for s, n in zip(seq, counts):
                kk, vv = (t.bfloat16() for t in past[layer][s])
                limit = length[s] + 1 + torch.arange(n, device="cuda")
                u.check(out[at:at + n], None, u.exact(q[at:at + n], kk, vv, limit, a.scale))
                at += n
        for s, n in zip(seq, counts):
            length[s] += n

    def fork(src, dst):
        s, d = u.ints(src), u.ints(dst)
        gpu.kv_fork_dev(cache.c, s.data_ptr(), d.data_ptr(), len(src), stream=st)
        for a, b in zip(src, dst):
            length[b] = length[a]
            for layer in range(layers):
                past[layer][b] = past[layer][a]

    step([0, 2], [100, 77], 1)
    step([2], [50], 2)
    fork([2, 2], [4, 1])
    for i in range(3):
        step([4, 0, 2, 1], [1, 1, 1, 1], 3 + i)
    gpu.kv_free_dev(cache.c, u.ints([0, 4]).data_ptr(), 2, stream=st)
    length[0] = length[4] = 0
    for layer in range(layers):
        past[layer][0] = past[layer][4] = (torch.zeros(0, K, D, device="cuda"),) * 2
    gpu.kv_compact_dev(cache.c, stream=st)
    step([3, 0], [40, 3], 10)
    for i in range(2):
        step([0, 1, 2, 3], [1, 1, 1, 1], 20 + i)
    assert cache.status() == 0
    live = int((cache.refs > 0).sum())
    gpu.kv_compact_dev(cache.c, stream=st)
    assert (cache.refs[:live] > 0).all() and (cache.refs[live:] == 0).all()


def test_places_of_an_empty_list(gpu):
    """A step whose list is empty: no row has a place, whatever the step before has left there, and
    positions and cache that are run on these places all the same write nothing."""
    import torch
    import attn_util as u
    import apus_b200.backend as B
    cache = u.Cache(1, 9, 1, 16, 64, 3, 4).hold([20, 5, 0])
    k0, v0, before = cache.k.clone(), cache.v.clone(), cache.state()
    seq, cu = u.ints([0, 1]), u.ints([0, 2, 3])
    for ds, dc in ((seq.data_ptr(), cu.data_ptr()), (None, cu.data_ptr()), (None, None)):
        slot = u.ints([p * 16 + 2 for p in range(5)] + [-7])
        gpu.kv_extend_dev(cache.c, ds, dc, 0, slot.data_ptr(), 5, stream=u.stream())
        assert slot.tolist() == [-1] * 5 + [-7]
    x = u.normal(5, 3, 64)
    q, pos = torch.zeros(5, 1, 64, dtype=torch.bfloat16, device="cuda"), u.ints([range(5)])
    r = B.Rope(q=x.data_ptr(), k=x[:, 1:].data_ptr(), v=x[:, 2:].data_ptr(), q_out=q.data_ptr(),
               q_stride=192, k_stride=192, v_stride=192, rows=5, heads=1, kv_heads=1, head_dim=64,
               rot_dim=64, pos=pos.data_ptr(), axes=1, sections=(32,), theta=1e4)
    gpu.rope_dev(r, cache.c, 0, slot.data_ptr(), stream=u.stream())
    torch.cuda.synchronize()
    assert cache.status() == 0
    for a, b in zip(before + [k0, v0], cache.state() + [cache.k, cache.v]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("pages", [8193, 20000, 300001])
def test_pools_of_more_pages_than_are_asked_for_ahead(gpu, pages):
    """Pages taken, shared, given back and moved together all over a large pool, most of it held
    by a user that is in no row of the table."""
    import torch
    import attn_util as u
    seqs, page = 6, 16
    cache = u.Cache(1, pages, 1, page, 64, seqs, 1200)
    rng = np.random.default_rng(pages)
    used = rng.random(pages) < 0.9
    used[-40:] = False                                   # (the last warp's last piece, too)
    cache.refs.copy_(torch.from_numpy(used.astype(np.int32)))
    k0, v0, book, st = cache.k.clone(), cache.v.clone(), Book(cache), u.stream()

    def extend(seq, add):
        assert book.extend(seq, add)
        ds, dc = u.ints(seq), u.ints(u.bounds(add))
        slot = torch.zeros(sum(add), dtype=torch.int32, device="cuda")
        start = [book.len[s] - a for s, a in zip(seq, add)]
        gpu.kv_extend_dev(cache.c, ds.data_ptr(), dc.data_ptr(), len(seq), slot.data_ptr(),
                          sum(add), stream=st)
        assert slot.tolist() == [book.table[s][t // page] * page + t % page
                                 for s, n, a in zip(seq, start, add) for t in range(n, n + a)]

    free = pages - int(used.sum())
    extend([4, 0, 2], [page * (free // 4), 5, page * (free // 3) + 1] if free < 3000 else
           [page * 1199, 5, page * 1000 + 1])
    book.check(cache, k0, v0)
    assert book.fork([0, 2], [1, 3])
    s, d = u.ints([0, 2]), u.ints([1, 3])
    gpu.kv_fork_dev(cache.c, s.data_ptr(), d.data_ptr(), 2, stream=st)
    book.check(cache, k0, v0)
    extend([1, 5], [40, 77])
    book.free([4])
    gpu.kv_free_dev(cache.c, u.ints([4]).data_ptr(), 1, stream=st)
    book.check(cache, k0, v0)
    book.compact()
    gpu.kv_compact_dev(cache.c, stream=st)
    book.check(cache, k0, v0)
    # one page more than there are: refused, and all as it was
    want = book.refs.count(0) + 1
    if want <= 1200:
        cu, one = u.ints([0, want * page]), u.ints([4])
        gpu.kv_extend_dev(cache.c, one.data_ptr(), cu.data_ptr(), 1, stream=st)
        assert cache.status() == 1
        cache.work[0] = 0
        extend([4], [(want - 1) * page])
        assert 0 not in book.refs
    book.check(cache, k0, v0)
    assert cache.status() == 0
