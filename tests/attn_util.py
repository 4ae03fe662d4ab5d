"""Tensors, argument structs and plain 64-bit forms for the tests of the attention half."""
import math

import torch

import apus_b200.backend as B


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def bounds(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def normal(*shape, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).bfloat16().cuda()


def stream():
    return torch.cuda.current_stream().cuda_stream


class Cache:
    """A cache of the caller's: torch tensors and the struct that names them."""

    def __init__(self, layers, pages, kv_heads, page, dim, seqs, width, seed=0):
        self.k = normal(layers, pages, kv_heads, page, dim, seed=seed + 1)
        self.v = normal(layers, pages, kv_heads, page, dim, seed=seed + 2)
        self.refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        self.table = torch.full((seqs, width), -1, dtype=torch.int32, device="cuda")
        self.len = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        # (the calls need nothing of what scratch held, but for the status word)
        self.work = torch.full((B.kv_work_ints(pages, seqs),), 0x5a5a5a5a, dtype=torch.int32,
                               device="cuda")
        self.work[0] = 0
        self.page, self.pages = page, pages
        self.c = B.KvCache(k=self.k.data_ptr(), v=self.v.data_ptr(), refs=self.refs.data_ptr(),
                           table=self.table.data_ptr(), len=self.len.data_ptr(),
                           work=self.work.data_ptr(), layers=layers, pages=pages,
                           page_tokens=page, kv_heads=kv_heads, head_dim=dim, seqs=seqs,
                           max_pages=width)

    def hold(self, lengths, seed=0):
        """Sequences of these lengths in pages from anywhere in the pool."""
        order = torch.randperm(self.pages, generator=torch.Generator().manual_seed(seed))
        at, table = 0, self.table.cpu()
        for i, n in enumerate(lengths):
            held = -(-n // self.page)
            table[i, :held] = order[at:at + held].int()
            at += held
        assert at <= self.pages
        self.table.copy_(table)
        self.refs[order[:at].cuda()] = 1
        self.len[:len(lengths)] = ints(lengths)
        return self

    def tokens(self, layer, s):
        """k and v [tokens, kv_heads, dim] of a sequence."""
        n = int(self.len[s])
        pages = self.table[s, :-(-n // self.page)].long()
        return [p[layer][pages].transpose(1, 2).flatten(0, 1)[:n] for p in (self.k, self.v)]

    def state(self):
        return [t.clone() for t in (self.refs, self.table, self.len)]

    def status(self):
        return int(self.work[0])


def attn(q, out, lse=None, gate=None, scale=None, kv_heads=None):
    rows, heads, dim = q.shape
    return B.Attn(q=q.data_ptr(), q_stride=q.stride(0) if rows > 1 else 0, out=out.data_ptr(),
                  out_stride=out.stride(0) if rows > 1 else 0,
                  gate=gate.data_ptr() if gate is not None else None,
                  gate_stride=gate.stride(0) if gate is not None and rows > 1 else 0,
                  lse=lse.data_ptr() if lse is not None else None, rows=rows, heads=heads,
                  kv_heads=kv_heads, head_dim=dim, scale=scale or dim ** -0.5)


def exact(q, k, v, limit, scale, gate=None):
    """(out, lse, bound of out, bound of lse) of one sequence in 64 bits: q [n, H, D],
    k and v [m, K, D], row i sees keys below limit[i].

    The bounds count roundings.  A score is an fp32 sum of D products in any order: off by at
    most D 2^-23 sum |q k| (twice the half step, for matrix units that cut off), and as many
    for the scale and the exponential, 2^-20 of the weight; a weight is narrowed to BF16, 2^-8
    of it; the sum of m of them is fp32, m 2^-23; the result is narrowed once, 2^-8 of it."""
    n, H, D = q.shape
    m, K = k.shape[:2]
    g = H // K
    qd = q.double().view(n, K, g, D)
    s = torch.einsum("nkgd,mkd->kgnm", qd, k.double()) * scale
    size = torch.einsum("nkgd,mkd->kgnm", qd.abs(), k.double().abs()) * scale
    seen = torch.arange(m, device="cuda")[None] < limit[:, None]
    s = s.masked_fill(~seen, -math.inf)
    size = size.masked_fill(~seen, 0.0)
    lse = torch.logsumexp(s, dim=-1) if m else torch.full((K, g, n), -math.inf, device="cuda",
                                                          dtype=torch.float64)
    w = torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[..., None]).masked_fill(~seen, 0)
    vd = v.double().masked_fill(~v.isfinite(), 0.0)
    out = torch.einsum("kgnm,mkd->nkgd", w, vd).reshape(n, H, D)
    mass = torch.einsum("kgnm,mkd->nkgd", w, vd.abs()).reshape(n, H, D)
    ds = D * 2.0 ** -23 * (size.amax(-1) if m else torch.zeros_like(lse))
    ds = ds.permute(2, 0, 1).reshape(n, H)
    lse = lse.permute(2, 0, 1).reshape(n, H)
    if gate is not None:
        sg = torch.sigmoid(gate.double())
        out, mass = out * sg, mass * sg
    rel = 2.0 ** -8 + 2 * ds + 2.0 ** -20 + m * 2.0 ** -23
    return (out, lse, 2.0 ** -8 * out.abs() + rel[..., None] * mass + 1e-30,
            ds + 2.0 ** -20 + m * 2.0 ** -24 + lse.abs().nan_to_num(0, 0, 0) * 2.0 ** -22)


def check(out, lse, ref, what=""):
    o, l, bo, bl = ref
    assert torch.isfinite(out.double()).all(), what
    worst = ((out.double() - o).abs() / bo).max() if o.numel() else 0.0
    assert worst <= 1, (what, float(worst))
    if lse is not None:
        none = l == -math.inf
        assert torch.equal(lse.double()[none], l[none]), what
        off = ((lse.double() - l).abs() / bl)[~none]
        assert not off.numel() or off.max() <= 1, (what, float(off.max()))
