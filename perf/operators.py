"""Timing cases of the attention half's operators: a paged key-value cache and the attention
that reads it.

  prompt  attention of packed prompts, causal, grouped heads (apus_cuda_attn_prompt_dev)
  decode  attention of one new token a sequence over the paged cache
          (apus_cuda_attn_decode_dev)
  rope    rotary positions of queries and keys on several axes, keys and values
          written into the cache's pages (apus_cuda_rope_dev)
  pages   the cache's pages: copied, forked, freed, compacted and taken again
          (apus_cuda_kv_copy_dev, _fork_dev, _free_dev, _compact_dev, _extend_dev)

A case names one of them and its sizes; `listed()` holds the fixed ones, `draw()` more of the
same ranges.  `run` computes a pass in elementary torch operations, or, where `own` is true, by
the library's calls on the same tensors.  Everything is BF16 but the logarithms of the softmax
sums, which are fp32; the plain forms compute in 32 bits (the angles in 64) and round once.
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

THETA = 1.0e7
HEADS = [(16, 2, 256), (32, 8, 128), (20, 4, 128), (12, 12, 64), (16, 1, 128), (6, 2, 64)]


def listed():
    return [
        # a short question, alone: latency is all there is
        {"name": "prompt_one_77", "op": "prompt", "seqs": 1, "longest": 77, "past": 0,
         "heads": 16, "kv_heads": 2, "dim": 256, "causal": True, "gate": True, "pad": 0},
        # prompts of a few users, packed as they came, in a buffer with rows to spare
        {"name": "prompt_ragged", "op": "prompt", "seqs": 9, "longest": 2011, "past": 0,
         "heads": 16, "kv_heads": 2, "dim": 256, "causal": True, "gate": True, "pad": 59},
        # parts of prompts behind what earlier parts left, other heads
        {"name": "prompt_parts_d128", "op": "prompt", "seqs": 5, "longest": 1531, "past": 2500,
         "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "gate": False, "pad": 0},
        # one long document
        {"name": "prompt_8192", "op": "prompt", "seqs": 1, "longest": 8192, "past": 0,
         "heads": 16, "kv_heads": 2, "dim": 256, "causal": True, "gate": True, "pad": 0},
        # one sequence generating, not long yet
        {"name": "decode_one_977", "op": "decode", "seqs": 1, "longest": 977,
         "heads": 16, "kv_heads": 2, "dim": 256, "page": 32, "gate": True},
        # a full batch of a server, every length
        {"name": "decode_batch_64", "op": "decode", "seqs": 64, "longest": 32003,
         "heads": 16, "kv_heads": 2, "dim": 256, "page": 64, "gate": True},
        # one long document being asked about; other heads
        {"name": "decode_long_d128", "op": "decode", "seqs": 1, "longest": 131071,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "gate": False},
        # a decode step of a few sequences: one position for each
        {"name": "rope_step_7", "op": "rope", "seqs": 7, "longest": 1, "past": 4000,
         "heads": 16, "kv_heads": 2, "dim": 256, "rot": 64, "page": 32, "axes": 1,
         "interleaved": False},
        # a long prompt with images: time, height and width
        {"name": "rope_images_8192", "op": "rope", "seqs": 3, "longest": 6007, "past": 900,
         "heads": 16, "kv_heads": 2, "dim": 256, "rot": 64, "page": 64, "axes": 3,
         "interleaved": True},
        # pages handed to another worker's part of the pool
        {"name": "pages_copy_97", "op": "pages", "what": "copy", "seqs": 8, "longest": 2048,
         "count": 97, "layers": 10, "kv_heads": 2, "dim": 256, "page": 16},
        # several answers to each of a few questions: forked, continued, dropped
        {"name": "pages_fork_16", "op": "pages", "what": "fork", "seqs": 16, "longest": 3001,
         "count": 0, "layers": 10, "kv_heads": 2, "dim": 256, "page": 64},
        # half of the sequences end, the cache is compacted, new ones come; twice
        {"name": "pages_churn", "op": "pages", "what": "churn", "seqs": 40, "longest": 2501,
         "count": 0, "layers": 10, "kv_heads": 2, "dim": 256, "page": 32},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "decode", "decode", "rope", "pages"])
    heads, kv_heads, dim = rng.choice(HEADS)
    if op == "prompt":
        case = {"op": op, "seqs": _log_int(rng, 1, 24), "longest": _log_int(rng, 1, 6000),
                "past": rng.choice([0, 0, _log_int(rng, 1, 2000)]), "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "causal": rng.random() < 0.85,
                "gate": rng.random() < 0.5, "pad": rng.choice([0, rng.randint(1, 99)])}
        while True:
            q, k = _prompt_lengths(case)
            if sum(q) * sum(k) * heads <= 8192 * 8192 * 16 and work(case)["flops"] <= 5e11:
                return case
            case["seqs"] = max(1, case["seqs"] - 1)
            case["longest"] = max(1, case["longest"] - case["longest"] // 8)
            case["past"] -= case["past"] // 4
    if op == "decode":
        case = {"op": op, "seqs": _log_int(rng, 1, 200), "longest": _log_int(rng, 1, 100000),
                "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "page": rng.choice([16, 32, 64, 128]), "gate": rng.random() < 0.5}
        # (the plain form widens every sequence to the longest)
        while case["seqs"] * case["longest"] * kv_heads * dim > 64 * 32003 * 2 * 256:
            case["longest"] -= case["longest"] // 8
        return case
    if op == "rope":
        axes = rng.choice([1, 2, 3, 4])
        case = {"op": op, "seqs": _log_int(rng, 1, 60), "longest": _log_int(rng, 1, 5000),
                "past": _log_int(rng, 1, 5000), "heads": heads, "kv_heads": kv_heads,
                "dim": dim, "rot": rng.choice([dim // 4, dim // 2, dim]),
                "page": rng.choice([16, 32, 64, 128]), "axes": axes,
                "interleaved": axes > 1 and rng.random() < 0.5}
        while sum(_lengths(case["seqs"], case["longest"])) * (heads + 2 * kv_heads) * dim > \
                8000 * 20 * 256:
            case["longest"] -= case["longest"] // 8
        return case
    what = rng.choice(["copy", "fork", "churn"])
    case = {"op": op, "what": what, "seqs": rng.randint(2, 40),
            "longest": _log_int(rng, 1, 2500), "count": 0, "layers": rng.randint(1, 10),
            "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 32, 64])}
    while sum(_lengths(case["seqs"], case["longest"])) * case["layers"] * kv_heads * dim > \
            15000 * 10 * 2 * 256:
        case["longest"] -= case["longest"] // 8
    if what == "copy":
        case["count"] = _log_int(rng, 1, 200)
    return case


def _lengths(count, longest):
    """`count` lengths from 1 to `longest`, spread over their logarithm, the longest among them:
    a fixed choice for the two numbers."""
    rng = random.Random(count * 1000003 + longest)
    n = [_log_int(rng, max(1, longest // 64), longest) for _ in range(count)]
    n[rng.randrange(count)] = longest
    return n


def _prompt_lengths(case):
    """Rows of each sequence and the keys that they see (those of earlier parts first)."""
    q = _lengths(case["seqs"], case["longest"])
    rng = random.Random(case["past"] + 17)
    return q, [n + (rng.randint(0, case["past"]) if case["past"] else 0) for n in q]


def _bounds(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _sections(case):
    """Rotated pairs of each axis: as even as can be, the first ones longer."""
    pairs, axes = case["rot"] // 2, case["axes"]
    return [(pairs + axes - 1 - a) // axes for a in range(axes)]


def _axis_of_pair(case):
    sections = _sections(case)
    if case["interleaved"]:
        return [i % case["axes"] for i in range(case["rot"] // 2)]
    return [a for a, n in enumerate(sections) for _ in range(n)]


# ---- inputs -----------------------------------------------------------------------


class _Gen:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape, scale=1.0):
        return torch.randn(*shape, generator=self.g, device="cuda",
                           dtype=torch.bfloat16).mul_(scale)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda", dtype=torch.int32)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cache(g, lengths, spare, layers, kv_heads, dim, page, rows=None, room=0):
    """A cache that holds sequences of these lengths in the pages of a used pool: anywhere.
    room: tokens that a sequence may still take; spare: pages that are free."""
    held = [(n + page - 1) // page for n in lengths]
    pages, rows = sum(held) + spare, rows or len(lengths)
    width = max((n + room + page - 1) // page for n in lengths) + 1
    order = g.order(pages)
    table = torch.full((rows, width), -1, dtype=torch.int32)
    at, order_host = 0, order.cpu()
    for i, n in enumerate(held):
        table[i, :n] = order_host[at:at + n]
        at += n
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[order[:at].long()] = 1
    size = (layers, pages, kv_heads, page, dim)
    return {"k": g.normal(*size), "v": g.normal(*size), "refs": refs, "table": table.cuda(),
            "len": _ints(lengths + [0] * (rows - len(lengths))),
            "work": torch.zeros(4 * pages + 4 * rows + 64, dtype=torch.int32, device="cuda")}


def prepare(case, seed):
    g = _Gen(seed)
    s = {"case": case}
    H, K, D = case.get("heads"), case["kv_heads"], case["dim"]
    if case["op"] == "prompt":
        nq, nk = _prompt_lengths(case)
        rows = sum(nq) + case["pad"]
        # rows of a fused projection: the queries beside the gate, the keys beside the values
        s["q"], s["gate"] = g.normal(rows, 2, H, D, scale=1.3).unbind(1)
        s["k"], s["v"] = g.normal(sum(nk), 2, K, D).unbind(1)
        s["cu_q"], s["cu_k"] = _ints(_bounds(nq)), _ints(_bounds(nk))
        s["out"] = torch.zeros(rows, H, D, dtype=torch.bfloat16, device="cuda")
        s["lse"] = torch.zeros(rows, H, device="cuda")
    elif case["op"] == "decode":
        n = _lengths(case["seqs"], case["longest"])
        s["kv"] = _cache(g, n, 7, 1, K, D, case["page"])
        s["seq"] = g.order(case["seqs"])
        s["q"], s["gate"] = g.normal(case["seqs"], 2, H, D, scale=1.3).unbind(1)
        s["out"] = torch.zeros(case["seqs"], H, D, dtype=torch.bfloat16, device="cuda")
        s["lse"] = torch.zeros(case["seqs"], H, device="cuda")
    elif case["op"] == "rope":
        n = _lengths(case["seqs"], case["longest"])
        rng = random.Random(case["past"])
        past = [rng.randint(0, case["past"]) for _ in n]
        T, page = sum(n), case["page"]
        s["kv"] = _cache(g, [a + b for a, b in zip(n, past)], 3, 1, K, D, page)
        table = s["kv"]["table"].cpu()
        at = [(i, past[i] + j) for i in range(len(n)) for j in range(n[i])]
        s["slot"] = _ints([int(table[i, p // page]) * page + p % page for i, p in at])
        pos = [[p if a == 0 else (p * (37 + 4 * a)) % (50 * a + 14) for _, p in at]
               for a in range(case["axes"])]
        s["pos"] = _ints(pos)
        s["qkv"] = g.normal(T, H + 2 * K, D)
        s["q_out"] = torch.zeros(T, H, D, dtype=torch.bfloat16, device="cuda")
        s["k_out"] = torch.zeros(T, K, D, dtype=torch.bfloat16, device="cuda")
    else:
        n = _lengths(case["seqs"], case["longest"])
        page, what = case["page"], case["what"]
        spare = case["count"] if what == "copy" else 2 * case["seqs"] + 5
        s["kv"] = kv = _cache(g, n, spare, case["layers"], K, D, page, room=1,
                              rows=2 * len(n) if what == "fork" else len(n))
        if what == "copy":
            free = torch.nonzero(kv["refs"] == 0).flatten().int()
            used = torch.nonzero(kv["refs"] != 0).flatten().int()
            s["src"] = used[torch.arange(case["count"], device="cuda") * 5 % len(used)]
            s["dst"] = free[g.order(len(free)).long()][:case["count"]].contiguous()
        elif what == "fork":
            s["src"], s["dst"] = _ints(range(len(n))), _ints(range(len(n), 2 * len(n)))
            s["one"] = _ints(range(len(n) + 1))
        else:
            s["seqs"] = [_ints(range(h, len(n), 2)) for h in (0, 1)]
            s["cu"] = [_ints(_bounds(n[h::2])) for h in (0, 1)]
    torch.cuda.synchronize()
    return s


# ---- plain forms ------------------------------------------------------------------


def _softmax(scores, allowed):
    """Weights and the logarithm of their sum over the last axis, in 32 bits; a row that may see
    nothing has weights of zero."""
    scores = torch.where(allowed, scores, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(dim=-1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total), (top + torch.log(total)).squeeze(-1)


def _gated(out, s):
    if s["case"]["gate"]:
        out = out / (1.0 + torch.exp(-s["gate"].float()))
    return out.bfloat16()


def _plain_prompt(s):
    H, K, D = s["case"]["heads"], s["case"]["kv_heads"], s["case"]["dim"]
    Tq, Tk = s["q"].shape[0], s["k"].shape[0]
    row, key = (torch.arange(n, device="cuda") for n in (Tq, Tk))
    sq = torch.searchsorted(s["cu_q"][1:], row, right=True)
    sk = torch.searchsorted(s["cu_k"][1:], key, right=True)
    last = s["cu_k"][1:] - s["cu_q"][1:]
    inside = row < s["cu_q"][-1]
    allowed = sq[:, None] == sk[None, :]
    if s["case"]["causal"]:
        allowed &= key[None, :] <= row[:, None] + last[sq.clamp(max=len(last) - 1)][:, None]
    q = s["q"].float().view(Tq, K, H // K, D).permute(1, 2, 0, 3).reshape(K, -1, D)
    k, v = (s[n].float().permute(1, 0, 2) for n in ("k", "v"))
    scores = torch.bmm(q, k.transpose(1, 2)).mul_(D ** -0.5).view(K, H // K, Tq, Tk)
    p, lse = _softmax(scores, allowed)
    out = torch.bmm(p.view(K, -1, Tk), v).view(H, Tq, D).transpose(0, 1)
    s["out"].copy_(torch.where(inside[:, None, None], _gated(out, s), s["out"]))
    s["lse"].copy_(torch.where(inside[:, None], lse.view(H, Tq).t(), s["lse"]))


def _plain_decode(s):
    H, K, D = s["case"]["heads"], s["case"]["kv_heads"], s["case"]["dim"]
    kv, seq, page = s["kv"], s["seq"].long(), s["case"]["page"]
    n, B = s["case"]["longest"], len(s["seq"])
    at = torch.arange(n, device="cuda")
    pages = kv["table"][seq][:, :(n + page - 1) // page].clamp(min=0).long()
    k, v = (kv[name][0][pages].transpose(1, 2).reshape(B, K, -1, D)[:, :, :n].float()
            for name in ("k", "v"))
    q = s["q"].float().view(B, K, H // K, D)
    scores = torch.matmul(q, k.transpose(2, 3)) * D ** -0.5
    p, lse = _softmax(scores, (at[None, :] < kv["len"][seq][:, None])[:, None, None])
    s["out"].copy_(_gated(torch.matmul(p, v).view(B, H, D), s))
    s["lse"].copy_(lse.view(B, H))


def _plain_rope(s):
    case = s["case"]
    H, K, r = case["heads"], case["kv_heads"], case["rot"]
    pairs = torch.arange(r // 2, device="cuda", dtype=torch.float64)
    axis = torch.tensor(_axis_of_pair(case), device="cuda")
    angle = s["pos"].double()[axis].t() * THETA ** (-2.0 * pairs / r)
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    x = s["qkv"][:, :H + K].float()
    a, b = x[..., :r // 2], x[..., r // 2:r]
    y = torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., r:]], dim=-1).bfloat16()
    s["q_out"].copy_(y[:, :H])
    s["k_out"].copy_(y[:, H:])
    page, offset = s["slot"].long() // case["page"], s["slot"].long() % case["page"]
    s["kv"]["k"][0][page, :, offset] = y[:, H:]
    s["kv"]["v"][0][page, :, offset] = s["qkv"][:, H + K:]


def _held(kv, seq):
    """Which entries of these rows of the table name a page."""
    page = kv["k"].shape[3]
    count = (kv["len"][seq] + page - 1) // page
    return torch.arange(kv["table"].shape[1], device="cuda")[None] < count[:, None]


def _count(kv, pages, mask, by):
    """refs += by for every page that the mask names."""
    total = len(kv["refs"])
    more = torch.zeros(total + 1, dtype=torch.int32, device="cuda")
    at = torch.where(mask, pages, total).flatten().long()
    more.scatter_add_(0, at, torch.full_like(at, by, dtype=torch.int32))
    kv["refs"] += more[:total]


def _free_pages(kv):
    """All pages, the free ones first, in ascending order."""
    return torch.argsort((kv["refs"] != 0).int(), stable=True).int()


def _move(kv, source):
    """Every page's contents become those of its source (all layers)."""
    kv["k"].copy_(kv["k"][:, source])
    kv["v"].copy_(kv["v"][:, source])


def _plain_free(kv, seq):
    seq = seq.long()
    held, rows = _held(kv, seq), kv["table"][seq]
    _count(kv, rows, held, -1)
    kv["table"][seq] = torch.where(held, -1, rows)
    kv["len"][seq] = 0


def _plain_extend(kv, seq, cu):
    seq, page = seq.long(), kv["k"].shape[3]
    before = (kv["len"][seq] + page - 1) // page
    kv["len"][seq] += cu[1:] - cu[:-1]
    after = (kv["len"][seq] + page - 1) // page
    first = torch.cumsum(after - before, 0) - (after - before)
    at = torch.arange(kv["table"].shape[1], device="cuda")[None]
    fresh = (at >= before[:, None]) & (at < after[:, None])
    take = torch.where(fresh, first[:, None] + at - before[:, None], 0)
    rows = torch.where(fresh, _free_pages(kv)[take], kv["table"][seq])
    kv["table"][seq] = rows
    _count(kv, rows, fresh, 1)


def _plain_fork(kv, src, dst):
    src, dst, page = src.long(), dst.long(), kv["k"].shape[3]
    full, rest = kv["len"][src] // page, kv["len"][src] % page
    fresh = _free_pages(kv)[torch.cumsum((rest > 0).int(), 0) - (rest > 0).int()]
    at = torch.arange(kv["table"].shape[1], device="cuda")[None]
    last = (at == full[:, None]) & (rest > 0)[:, None]
    old = kv["table"][src]
    rows = torch.where(_held(kv, src), torch.where(last, fresh[:, None], old), kv["table"][dst])
    total = len(kv["refs"])
    source = torch.arange(total + 1, device="cuda")
    source[torch.where(rest > 0, fresh, total).long()] = \
        old.gather(1, full[:, None].long()).flatten().long()
    _move(kv, source[:total])
    kv["table"][dst] = rows
    kv["len"][dst] = kv["len"][src]
    _count(kv, rows, _held(kv, src), 1)


def _plain_compact(kv):
    total = len(kv["refs"])
    live, at = kv["refs"] > 0, torch.arange(total, device="cuda")
    count = live.sum()
    leave, fill = live & (at >= count), ~live & (at < count)
    # the n-th of those that leave goes to the n-th of those to be filled
    to = torch.argsort((~fill).int(), stable=True)[(torch.cumsum(leave, 0) - 1).clamp(min=0)]
    new = torch.where(leave, to, at)
    source = torch.arange(total + 1, device="cuda")
    source[torch.where(leave, to, total)] = at
    source = source[:total]
    _move(kv, source)
    held = _held(kv, slice(None))
    kv["table"].copy_(torch.where(held, new[kv["table"].clamp(min=0).long()].int(), kv["table"]))
    kv["refs"].copy_(torch.where(leave, 0, kv["refs"][source]))


def _plain_copy(kv, src, dst):
    source = torch.arange(len(kv["refs"]), device="cuda")
    source[dst.long()] = src.long()
    _move(kv, source)


def _plain_pages(s):
    kv, what = s["kv"], s["case"]["what"]
    if what == "copy":
        _plain_copy(kv, s["src"], s["dst"])
    elif what == "fork":
        _plain_fork(kv, s["src"], s["dst"])
        _plain_extend(kv, s["dst"], s["one"])
        _plain_free(kv, s["dst"])
    else:
        _plain_free(kv, s["seqs"][0])
        _plain_compact(kv)
        _plain_extend(kv, s["seqs"][0], s["cu"][0])
        _plain_free(kv, s["seqs"][1])
        _plain_compact(kv)
        _plain_extend(kv, s["seqs"][1], s["cu"][1])


# ---- the library's calls ------------------------------------------------------------

_lib = {}


def _backend():
    """(backend object, its module), loaded by path: the package directory's name is not an
    identifier."""
    if not _lib:
        root = os.path.join(os.getcwd(), "apus-qwen3.6-35b-a3b_b200")
        spec = importlib.util.spec_from_file_location(
            "apus_b200", os.path.join(root, "__init__.py"), submodule_search_locations=[root])
        pkg = importlib.util.module_from_spec(spec)
        sys.modules["apus_b200"] = pkg
        spec.loader.exec_module(pkg)
        be = pkg.Backend()
        be.enable()
        _lib.update(be=be, module=pkg.backend)
    return _lib["be"], _lib["module"]


def _kv_struct(module, kv):
    layers, pages, kv_heads, page, dim = kv["k"].shape
    seqs, width = kv["table"].shape
    return module.KvCache(
        k=kv["k"].data_ptr(), v=kv["v"].data_ptr(), refs=kv["refs"].data_ptr(),
        table=kv["table"].data_ptr(), len=kv["len"].data_ptr(), work=kv["work"].data_ptr(),
        layers=layers, pages=pages, page_tokens=page, kv_heads=kv_heads, head_dim=dim,
        seqs=seqs, max_pages=width)


def _describe(s):
    """The argument structs of the pass: a program fills them once for its buffers."""
    _, module = _backend()
    case = s["case"]
    D = case["dim"]
    if "kv" in s:
        s["kv_struct"] = _kv_struct(module, s["kv"])
    if case["op"] in ("prompt", "decode"):
        s["call"] = module.Attn(
            q=s["q"].data_ptr(), q_stride=s["q"].stride(0),
            gate=s["gate"].data_ptr() if case["gate"] else None, gate_stride=s["gate"].stride(0),
            out=s["out"].data_ptr(), out_stride=s["out"].stride(0), lse=s["lse"].data_ptr(),
            rows=s["q"].shape[0], heads=case["heads"], kv_heads=case["kv_heads"], head_dim=D,
            scale=D ** -0.5)
    if case["op"] == "prompt":
        s["keys"] = module.AttnKeys(
            k=s["k"].data_ptr(), v=s["v"].data_ptr(), k_stride=s["k"].stride(0),
            v_stride=s["v"].stride(0), rows=s["k"].shape[0], cu_q=s["cu_q"].data_ptr(),
            cu_k=s["cu_k"].data_ptr(), seqs=case["seqs"], causal=int(case["causal"]))
    elif case["op"] == "rope":
        H, K = case["heads"], case["kv_heads"]
        row, x = s["qkv"].stride(0), s["qkv"]
        s["call"] = module.Rope(
            q=x.data_ptr(), q_stride=row, q_out=s["q_out"].data_ptr(), q_out_stride=H * D,
            k=x[:, H:].data_ptr(), k_stride=row, k_out=s["k_out"].data_ptr(), k_out_stride=K * D,
            v=x[:, H + K:].data_ptr(), v_stride=row, rows=x.shape[0], heads=H, kv_heads=K,
            head_dim=D, rot_dim=case["rot"], pos=s["pos"].data_ptr(), axes=case["axes"],
            sections=tuple(_sections(case)), interleaved=int(case["interleaved"]), theta=THETA)


def _own(s):
    be, _ = _backend()
    if "kv_struct" not in s and "call" not in s:
        _describe(s)
    case, stream = s["case"], torch.cuda.current_stream().cuda_stream
    if case["op"] == "prompt":
        be.attn_prompt_dev(s["call"], s["keys"], stream=stream)
    elif case["op"] == "decode":
        be.attn_decode_dev(s["call"], s["kv_struct"], 0, s["seq"].data_ptr(), stream=stream)
    elif case["op"] == "rope":
        be.rope_dev(s["call"], s["kv_struct"], 0, s["slot"].data_ptr(), stream=stream)
    elif case["what"] == "copy":
        be.kv_copy_dev(s["kv_struct"], s["src"].data_ptr(), s["dst"].data_ptr(),
                       case["count"], stream=stream)
    elif case["what"] == "fork":
        kv, n, dst = s["kv_struct"], case["seqs"], s["dst"].data_ptr()
        be.kv_fork_dev(kv, s["src"].data_ptr(), dst, n, stream=stream)
        be.kv_extend_dev(kv, dst, s["one"].data_ptr(), n, stream=stream)
        be.kv_free_dev(kv, dst, n, stream=stream)
    else:
        kv = s["kv_struct"]
        for seq, cu in zip(s["seqs"], s["cu"]):
            be.kv_free_dev(kv, seq.data_ptr(), len(seq), stream=stream)
            be.kv_compact_dev(kv, stream=stream)
            be.kv_extend_dev(kv, seq.data_ptr(), cu.data_ptr(), len(seq), stream=stream)


_PLAIN = {"prompt": _plain_prompt, "decode": _plain_decode, "rope": _plain_rope,
          "pages": _plain_pages}


def run(s):
    (_own if own else _PLAIN[s["case"]["op"]])(s)
    if s["case"]["op"] in ("prompt", "decode"):
        return {"out": s["out"], "lse": s["lse"]}
    kv = s["kv"]
    if s["case"]["op"] == "rope":
        return {"q": s["q_out"], "k": s["k_out"], "cache_k": kv["k"], "cache_v": kv["v"]}
    return {name: kv[name] for name in ("k", "v", "refs", "table", "len")}


def work(case):
    H, K, D = case.get("heads", 0), case["kv_heads"], case["dim"]
    if case["op"] == "prompt":
        nq, nk = _prompt_lengths(case)
        seen = sum(a * (b - a) + a * (a + 1) // 2 if case["causal"] else a * b
                   for a, b in zip(nq, nk))
        return {"bytes": sum(nq) * H * (2 * D * (3 if case["gate"] else 2) + 4) +
                4 * sum(nk) * K * D, "flops": 4 * seen * H * D}
    if case["op"] == "decode":
        n = sum(_lengths(case["seqs"], case["longest"]))
        rows = case["seqs"] * H
        return {"bytes": 4 * n * K * D + rows * (2 * D * (3 if case["gate"] else 2) + 4),
                "flops": 4 * n * H * D}
    if case["op"] == "rope":
        T = sum(_lengths(case["seqs"], case["longest"]))
        # in: q, k, v and positions; out: q, k, and k and v in the cache
        return {"bytes": T * (2 * D * (2 * H + 5 * K) + 4 * case["axes"] + 4),
                "flops": T * (H + K) * case["rot"] * 3}
    n, page = _lengths(case["seqs"], case["longest"]), case["page"]
    held = [(a + page - 1) // page for a in n]
    if case["what"] == "copy":
        moved, ints = case["count"], 2 * case["count"]
    elif case["what"] == "fork":
        moved, ints = sum(a % page > 0 for a in n), 6 * sum(held)
    else:
        # those who stay close up, then those who came before close up behind them
        moved, ints = 2 * min(sum(held[0::2]), sum(held[1::2])), 10 * sum(held)
    return {"bytes": 2 * moved * case["layers"] * 2 * K * page * D * 2 + 4 * ints, "flops": 0}


# ---- from the definitions, in 64 bits -------------------------------------------------


def _attend(q, k, v, gate, limit):
    """One sequence: q [n, H, D], k and v [m, K, D], row i sees keys below limit[i]."""
    n, H, D = q.shape
    m, K = k.shape[:2]
    group = H // K
    out = torch.zeros(n, H, D, dtype=torch.float64, device="cuda")
    lse = torch.full((n, H), -math.inf, dtype=torch.float64, device="cuda")
    hidden = torch.arange(m, device="cuda")[None, :] >= limit[:, None]
    for h in range(H):
        score = (q[:, h].double() @ k[:, h // group].double().t()) / math.sqrt(D)
        score.masked_fill_(hidden, -math.inf)
        lse[:, h] = torch.logsumexp(score, dim=1)
        weight = torch.exp(score - lse[:, h, None]).masked_fill_(hidden, 0.0)
        out[:, h] = weight @ v[:, h // group].double()
    return (out * torch.sigmoid(gate.double()) if gate is not None else out), lse


def _exact_prompt(s):
    case, cq, ck = s["case"], s["cu_q"].tolist(), s["cu_k"].tolist()
    out, lse = s["out"].double(), s["lse"].double()
    for i in range(case["seqs"]):
        q, k = slice(cq[i], cq[i + 1]), slice(ck[i], ck[i + 1])
        n, m = cq[i + 1] - cq[i], ck[i + 1] - ck[i]
        limit = torch.full((n,), m, device="cuda")
        if case["causal"]:
            limit = m - n + 1 + torch.arange(n, device="cuda")
        out[q], lse[q] = _attend(s["q"][q], s["k"][k], s["v"][k],
                                 s["gate"][q] if case["gate"] else None, limit)
    return {"out": out, "lse": lse}


def _exact_decode(s):
    case, kv, lengths = s["case"], s["kv"], s["kv"]["len"].tolist()
    out, lse = s["out"].double(), s["lse"].double()
    for b, i in enumerate(s["seq"].tolist()):
        n = lengths[i]
        pages = kv["table"][i, :(n + case["page"] - 1) // case["page"]].long()
        k, v = (kv[name][0][pages].permute(0, 2, 1, 3).flatten(0, 1)[:n] for name in ("k", "v"))
        out[b:b + 1], lse[b:b + 1] = _attend(
            s["q"][b:b + 1], k, v, s["gate"][b:b + 1] if case["gate"] else None,
            torch.tensor([n], device="cuda"))
    return {"out": out, "lse": lse}


def _exact_rope(s):
    case, x = s["case"], s["qkv"].double()
    H, K, half = case["heads"], case["kv_heads"], case["rot"] // 2
    pos = s["pos"].double()
    y = x[:, :H + K].clone()
    for i, a in enumerate(_axis_of_pair(case)):
        turn = torch.polar(torch.ones_like(pos[a]), pos[a] / THETA ** (i / half))
        z = torch.complex(x[:, :H + K, i], x[:, :H + K, i + half]) * turn[:, None]
        y[:, :, i], y[:, :, i + half] = z.real, z.imag
    k, v = s["kv"]["k"].double(), s["kv"]["v"].double()
    page, offset = s["slot"].long() // case["page"], s["slot"].long() % case["page"]
    k[0, page, :, offset] = y[:, H:]
    v[0, page, :, offset] = x[:, H + K:]
    return {"q": y[:, :H], "k": y[:, H:], "cache_k": k, "cache_v": v}


class _Book:
    """The cache's pages kept by hand, one sequence after the other."""

    def __init__(self, kv):
        self.page, self.kv = kv["k"].shape[3], kv
        self.refs, self.len = kv["refs"].tolist(), kv["len"].tolist()
        self.table = kv["table"].tolist()
        self.source = list(range(len(self.refs)))      # whose contents a page has by now

    def pages(self, i):
        return -(-self.len[i] // self.page)

    def take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def free(self, seqs):
        for i in seqs:
            for j in range(self.pages(i)):
                self.refs[self.table[i][j]] -= 1
                self.table[i][j] = -1
            self.len[i] = 0

    def extend(self, seqs, counts):
        for i, n in zip(seqs, counts):
            old = self.pages(i)
            self.len[i] += n
            for j in range(old, self.pages(i)):
                self.table[i][j] = self.take()

    def fork(self, src, dst):
        for i, o in zip(src, dst):
            self.len[o] = self.len[i]
            for j in range(self.pages(i)):
                p = self.table[i][j]
                if (j + 1) * self.page > self.len[i]:
                    p = self.take()
                    self.source[p] = self.source[self.table[i][j]]
                else:
                    self.refs[p] += 1
                self.table[o][j] = p

    def compact(self):
        live = [p for p, r in enumerate(self.refs) if r]
        holes = [p for p in range(len(live)) if not self.refs[p]]
        to = dict(zip([p for p in live if p >= len(live)], holes))
        for p, o in to.items():
            self.refs[o], self.refs[p] = self.refs[p], 0
            self.source[o] = self.source[p]
        for i in range(len(self.len)):
            for j in range(self.pages(i)):
                self.table[i][j] = to.get(self.table[i][j], self.table[i][j])

    def result(self):
        at = torch.tensor(self.source, device="cuda")
        return {"k": self.kv["k"][:, at], "v": self.kv["v"][:, at], "refs": _ints(self.refs),
                "table": _ints(self.table), "len": _ints(self.len)}


def _exact_pages(s):
    case, book = s["case"], _Book(s["kv"])
    n = _lengths(case["seqs"], case["longest"])
    if case["what"] == "copy":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            book.source[b] = a
    elif case["what"] == "fork":
        src, dst = s["src"].tolist(), s["dst"].tolist()
        book.fork(src, dst)
        book.extend(dst, [1] * len(dst))
        book.free(dst)
    else:
        for half in (0, 1):
            seqs = list(range(half, len(n), 2))
            book.free(seqs)
            book.compact()
            book.extend(seqs, n[half::2])
    return book.result()


def exact(case, seed):
    s = prepare(case, seed)
    return {"prompt": _exact_prompt, "decode": _exact_decode, "rope": _exact_rope,
            "pages": _exact_pages}[case["op"]](s)
