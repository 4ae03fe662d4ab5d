"""What the attention half's entry points refuse, before they look for a GPU; calls with nothing
to do succeed without one."""
import ctypes as C

import pytest


@pytest.fixture
def B(pkg):
    import apus_b200.backend as b
    return b


BIG = 1 << 20          # an address that nothing reads


def cache(B, **kw):
    d = dict(k=BIG, v=BIG, refs=BIG, table=BIG, len=BIG, work=BIG, layers=1, pages=10,
             page_tokens=16, kv_heads=2, head_dim=64, seqs=4, max_pages=4)
    d.update(kw)
    return B.KvCache(**d)


def attn(B, **kw):
    d = dict(q=BIG, out=BIG, rows=3, heads=4, kv_heads=2, head_dim=64, scale=0.125)
    d.update(kw)
    return B.Attn(**d)


def keys(B, **kw):
    d = dict(k=BIG, v=BIG, cu_q=BIG, cu_k=BIG, rows=3, seqs=1, causal=1)
    d.update(kw)
    return B.AttnKeys(**d)


def rope(B, **kw):
    d = dict(q=BIG, k=BIG, v=BIG, q_out=BIG, k_out=BIG, rows=2, heads=4, kv_heads=2, head_dim=64,
             rot_dim=32, pos=BIG, axes=1, sections=(16,), theta=1e4)
    d.update(kw)
    return B.Rope(**d)


BAD_CACHE = [dict(k=None), dict(work=None), dict(pages=0), dict(page_tokens=0),
             dict(page_tokens=24), dict(page_tokens=512), dict(head_dim=96), dict(k=BIG + 8),
             dict(pages=1 << 28), dict(seqs=0), dict(seqs=65537), dict(max_pages=1 << 28)]


@pytest.mark.parametrize("bad", BAD_CACHE)
def test_cache_is_refused(be, B, bad):
    c = cache(B, **bad)
    for call in (lambda: be.kv_extend_dev(c, BIG, BIG, 1), lambda: be.kv_fork_dev(c, BIG, BIG, 1),
                 lambda: be.kv_free_dev(c, BIG, 1), lambda: be.kv_compact_dev(c),
                 lambda: be.kv_copy_dev(c, BIG, BIG, 1),
                 lambda: be.attn_decode_dev(attn(B, head_dim=c.head_dim), c, 0, BIG)):
        with pytest.raises(B.BackendError) as e:
            call()
        assert any(w in str(e.value) for w in ("cache", "page_tokens", "head_dim", "aligned"))


def test_lists_are_refused(be, B):
    c = cache(B)
    for call in (lambda: be.kv_extend_dev(c, BIG, None, 1), lambda: be.kv_extend_dev(c, BIG, BIG, 5),
                 lambda: be.kv_fork_dev(c, None, BIG, 1), lambda: be.kv_fork_dev(c, BIG, BIG, 5),
                 lambda: be.kv_free_dev(c, None, 5), lambda: be.kv_copy_dev(c, BIG, None, 1),
                 lambda: be.kv_copy_dev(c, BIG, BIG, 11)):
        with pytest.raises(B.BackendError, match="bad args"):
            call()


@pytest.mark.parametrize("bad", [
    dict(head_dim=80), dict(heads=5), dict(heads=0), dict(kv_heads=0), dict(heads=34),
    dict(scale=0.0), dict(scale=float("nan")), dict(scale=-1.0), dict(q=None), dict(out=None),
    dict(q=BIG + 2), dict(q_stride=250), dict(q_stride=248), dict(out_stride=260),
    dict(gate=BIG + 4), dict(rows=1 << 31)])
def test_attention_is_refused(be, B, bad):
    with pytest.raises(B.BackendError, match="attn_"):
        be.attn_prompt_dev(attn(B, **bad), keys(B))
    with pytest.raises(B.BackendError, match="attn_"):
        be.attn_decode_dev(attn(B, **bad), cache(B), 0, BIG)


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=BIG + 8), dict(k_stride=120),
                                 dict(v_stride=132), dict(cu_q=None), dict(cu_k=None),
                                 dict(rows=1 << 31)])
def test_keys_are_refused(be, B, bad):
    with pytest.raises(B.BackendError, match="attn_prompt_dev"):
        be.attn_prompt_dev(attn(B), keys(B, **bad))


def test_decode_and_cache_have_to_agree(be, B):
    for c, layer, seq, a in ((cache(B, kv_heads=4), 0, BIG, attn(B)),
                             (cache(B, head_dim=128), 0, BIG, attn(B)),
                             (cache(B), 1, BIG, attn(B)),
                             (cache(B), 0, None, attn(B, rows=5))):
        with pytest.raises(B.BackendError, match="attn_decode_dev"):
            be.attn_decode_dev(a, c, layer, seq)


@pytest.mark.parametrize("bad", [
    dict(rot_dim=0), dict(rot_dim=24), dict(rot_dim=80), dict(axes=0), dict(axes=5),
    dict(theta=0.0), dict(theta=float("nan")), dict(sections=(15,)), dict(sections=(17,)),
    dict(axes=2, sections=(12, 4), interleaved=1), dict(axes=2, sections=(2 ** 64 - 1, 17)),
    dict(q=None), dict(q_out=BIG + 8),
    dict(k=BIG + 2), dict(k_stride=8), dict(pos=None), dict(heads=3), dict(head_dim=512)])
def test_rope_is_refused(be, B, bad):
    with pytest.raises(B.BackendError, match="rope_dev"):
        be.rope_dev(rope(B, **bad))


@pytest.mark.parametrize("bad", [
    dict(theta=0.5), dict(theta=1e31), dict(q=BIG, q_out=BIG, q_out_stride=512),
    dict(k=BIG, k_out=BIG, k_stride=512)])
def test_rope_is_refused_outside_of_its_ranges(be, B, bad):
    with pytest.raises(B.BackendError, match="theta|equal strides"):
        be.rope_dev(rope(B, **bad))


def test_a_table_too_large_to_count_is_refused(be, B):
    with pytest.raises(B.BackendError, match="too large"):
        be.kv_free_dev(cache(B, seqs=1 << 10, max_pages=1 << 21), BIG, 1)


def test_lists_whose_count_a_step_would_take_past_31_bits_are_refused(be, B):
    c = cache(B)
    for call in (lambda: be.kv_extend_dev(c, BIG, BIG, 1, BIG, (1 << 30) + 1),
                 lambda: be.kv_extend_dev(c, None, None, 0, BIG, (1 << 31) - 1),
                 lambda: be.kv_free_dev(c, BIG, (1 << 31) - 1)):
        with pytest.raises(B.BackendError, match="bad args"):
            call()


def test_rope_and_cache_have_to_agree(be, B):
    for r, c, layer, slot in ((rope(B), cache(B, kv_heads=1), 0, BIG),
                              (rope(B), cache(B), 1, BIG), (rope(B), cache(B), 0, None),
                              (rope(B, v=None), cache(B), 0, BIG), (rope(B, k_out=None), None, 0, None)):
        with pytest.raises(B.BackendError, match="rope_dev"):
            be.rope_dev(r, c, layer, slot)


def test_nothing_to_do(be, B):
    c = cache(B)
    be.kv_extend_dev(c, None, None, 0)
    be.kv_fork_dev(c, None, None, 0)
    be.kv_free_dev(c, None, 0)
    be.kv_copy_dev(c, None, None, 0)
    be.rope_dev(rope(B, rows=0, q=None, k=None, q_out=None))
    be.attn_prompt_dev(attn(B, rows=0, q=None, out=None), keys(B))
    be.attn_prompt_dev(attn(B), keys(B, seqs=0))
    be.attn_decode_dev(attn(B, rows=0, q=None, out=None), c, 0)


def test_structs_are_the_header_s(be, B, tmp_path):
    """Sizes and offsets of the argument structs, from the C compiler."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src, exe = tmp_path / "s.c", tmp_path / "s"
    pairs = [("ApusCudaKvCache", B.KvCache), ("ApusCudaRope", B.Rope), ("ApusCudaAttn", B.Attn),
             ("ApusCudaAttnKeys", B.AttnKeys)]
    lines = []
    for c_name, t in pairs:
        lines.append(f'printf("%zu\\n", sizeof({c_name}));')
        lines += [f'printf("%zu\\n", offsetof({c_name}, {f[0]}));' for f in t._fields_]
    src.write_text('#include <stdio.h>\n#include "backend_cuda.h"\nint main(void){'
                   + "".join(lines) + 'printf("%zu\\n", APUS_CUDA_KV_WORK_INTS(7, 3));return 0;}')
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(root, "include"),
                    str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, check=True).stdout.split()]
    want = []
    for _, t in pairs:
        want.append(C.sizeof(t))
        want += [getattr(t, f[0]).offset for f in t._fields_]
    assert got == want + [B.kv_work_ints(7, 3)]
