"""Refusals of the quantised-cache, 4-bit attention and GEMM-epilogue entry points: nothing here reaches a device."""
import pytest
import torch

import oracle.ops as O
from tilelang import _native as N
from tilelang import ops

BF, HF, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
A = 4096                       # an aligned address that is never read: every check below comes before a launch


def write(**kw):
    a = dict(slots=A, k=A, kc=A, ks=A, v=None, vc=None, vs=None, tokens=4, sk=128, sv=0, heads=2, dim=64, group=32, pages=4, page=16,
             fmt=N.TL_U4G, dtype=N.TL_BF16)
    a.update(kw)
    return N.load().tl_b200_kv_cache_write(a["slots"], a["k"], a["kc"], a["ks"], a["v"], a["vc"], a["vs"], a["tokens"], a["sk"], a["sv"], a["heads"],
                                           a["dim"], a["group"], a["pages"], a["page"], a["fmt"], a["dtype"], None)


@pytest.mark.parametrize("kw,text", [
    (dict(slots=None), "null"), (dict(k=None), "null"), (dict(ks=None), "null"), (dict(v=A), "null"), (dict(dim=96), "64, 128 or 256"),
    (dict(group=16), "groups"), (dict(group=128), "groups"), (dict(k=A + 2), "aligned"), (dict(sk=129), "aligned"), (dict(kc=A + 8), "aligned"),
    (dict(ks=A + 2), "aligned"), (dict(fmt=N.TL_E4M3), "single kv head"), (dict(fmt=N.TL_E4M3, heads=1, dim=12), "multiple of 8"),
    (dict(fmt=N.TL_E4M3, heads=1, dim=2048), "at most 1024"), (dict(fmt=N.TL_BF16), "format"), (dict(dtype=N.TL_F32), "bfloat16"),
    (dict(tokens=-1), "size"), (dict(page=0), "size"), (dict(pages=2 ** 30, page=4), "too large"), (dict(tokens=2 ** 31), "too large"),
])
def test_kv_cache_write_refuses(kw, text):
    assert write(**kw) == -1 and text in N.last_error()


def test_kv_cache_read_refuses_overlapping_rows():
    rc = N.load().tl_b200_kv_cache_read(A, A, A, A, None, None, None, 4, 64, 0, 2, 64, 32, 4, 16, N.TL_U4G, N.TL_BF16, None)
    assert rc == -1 and "overlap" in N.last_error()


def test_nothing_to_do_is_fine():
    assert write(tokens=0, slots=None, k=None) == 0
    assert attn(batch=0, q=None) == 0 and attn(s_q=0) == 0
    assert gemm(m=0, a=None) == 0


def attn(**kw):
    a = dict(q=A, kc=A, ks=A, vc=A, vs=A, table=A, lens=A, out=A, batch=2, s_q=1, h_q=4, h_kv=2, dim=64, group=32, sb=256, ss=256, page=16, mp=4,
             pages=8, scale=0.1, dtype=N.TL_BF16, ws=A, wb=1 << 30)
    a.update(kw)
    return N.load().tl_b200_attn_decode_paged_int4(*[a[x] for x in ("q", "kc", "ks", "vc", "vs", "table", "lens", "out", "batch", "s_q", "h_q", "h_kv",
                                                                   "dim", "group", "sb", "ss", "page", "mp", "pages", "scale", "dtype", "ws", "wb")], None)


@pytest.mark.parametrize("kw,text", [
    (dict(q=None), "null"), (dict(table=None), "null"), (dict(vs=None), "null"), (dict(dim=80), "64, 128 or 256"), (dict(group=128), "groups"),
    (dict(group=48), "groups"), (dict(h_q=5), "multiple"), (dict(h_kv=0), "size"), (dict(page=0), "size"), (dict(batch=-1), "size"),
    (dict(dtype=N.TL_F32), "bfloat16"), (dict(q=A + 2), "aligned"), (dict(sb=100), "aligned"), (dict(kc=A + 4), "aligned"),
    (dict(pages=2 ** 28, page=16), "too large"), (dict(batch=2 ** 24), "too large"),
])
def test_attn_decode_paged_int4_refuses(kw, text):
    assert attn(**kw) == -1 and text in N.last_error()


def gemm(**kw):
    a = dict(a=A, b=A, bias=None, res=None, c=A, m=4, n=8, k=8, tb=1, act=0, i=N.TL_BF16, o=N.TL_BF16)
    a.update(kw)
    return N.load().tl_b200_gemm_epilogue(*[a[x] for x in ("a", "b", "bias", "res", "c", "m", "n", "k", "tb", "act", "i", "o")], None)


@pytest.mark.parametrize("kw,text", [(dict(a=None), "null"), (dict(k=0), "positive"), (dict(act=9), "activation"), (dict(act=-1), "activation"),
                                     (dict(i=N.TL_E4M3), "input dtype"), (dict(o=N.TL_F16), "output"), (dict(m=-1), "negative"),
                                     (dict(n=2 ** 31), "2^31"), (dict(res=A, o=N.TL_F32), "residual")])
def test_gemm_epilogue_refuses(kw, text):
    assert gemm(**kw) == -1 and text in N.last_error()


def cache(pages=4, heads=2, page=16, dim=64, groups=2, dtype=BF):
    return torch.zeros(pages, heads, page, dim // 2, dtype=torch.uint8), torch.zeros(pages, heads, page, groups, 2, dtype=dtype)


def test_python_checks_of_the_cache():
    c, s = cache()
    x, slots = torch.zeros(3, 2, 64, dtype=BF), torch.zeros(3, dtype=torch.int64)
    for bad, text in [((slots.int(), x, c, s), "int64"), ((slots[:2], x, c, s), "one slot"), ((slots, x.float(), c, s), "bfloat16"),
                      ((slots, x[:, :1], c, s), "must be"), ((slots, x, c.float(), s), "uint8"), ((slots, x, c, s.half()), "k_scale"),
                      ((slots, x, c[0], s), "4-bit cache"), ((slots, x, c, s[:2]), "k_scale"), ((slots, x.transpose(1, 2).contiguous().transpose(1, 2), c, s), "contiguous"),
                      ((slots, x, c, s, x), "together"), ((slots, x, c, s, x.half(), c, s), "v must"),
                      ((slots, x, torch.zeros(4, 16, 2, 64).to(F8), s), "e4m3 cache"),
                      ((slots, x[:, 0], torch.zeros(4, 16, 64).to(F8), torch.zeros(4, 16, dtype=BF)), "float32"),
                      ((slots, x, c, s), "CUDA")]:
        with pytest.raises(ValueError, match=text):
            ops.kv_cache_write(*bad)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_cache_read(slots, c, s, x)


def test_python_checks_of_the_attention():
    c, s = cache()
    q, table, lens = torch.zeros(2, 1, 4, 64, dtype=BF), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    good = dict(q=q, k_cache=c, k_scale=s, v_cache=c, v_scale=s, block_table=table, cache_seqlens=lens, out=q.clone())
    for change, text in [(dict(out=q.half()), "q and out"), (dict(q=q[:, 0]), "q and out"), (dict(k_cache=c[..., :16]), "caches"),
                         (dict(v_cache=c[:2]), "caches"), (dict(v_scale=s.half()), "scales"), (dict(k_scale=s[:, :, :, :, :1]), "scales"),
                         (dict(q=q[:, :, :3], out=q[:, :, :3]), "multiple"), (dict(block_table=table.long()), "int32"),
                         (dict(cache_seqlens=lens[:1]), "int32"), (dict(q=q.transpose(2, 3).contiguous().transpose(2, 3)), "contiguous"), ({}, "CUDA")]:
        with pytest.raises(ValueError, match=text):
            ops.attn_decode_paged_int4(**{**good, **change})


def test_python_checks_of_the_gemm():
    a, b, c = torch.zeros(4, 8, dtype=BF), torch.zeros(8, 16, dtype=BF), torch.zeros(4, 16, dtype=BF)
    for kw, text in [(dict(b=b[:4]), "K shape"), (dict(c=c[:2]), "c must"), (dict(b=b.half()), "share"), (dict(c=c.half()), "share"),
                     (dict(bias=torch.zeros(4, dtype=BF)), "bias"), (dict(bias=torch.zeros(16)), "bias"), (dict(residual=c[:1]), "residual"),
                     (dict(activation="tanh"), "activation"), (dict(activation=[1]), "activation"), ({}, "CUDA")]:
        with pytest.raises(ValueError, match=text):
            ops.gemm_epilogue(**{**dict(a=a, b=b, c=c), **kw})


def test_the_oracle_quantiser_keeps_half_a_step():
    x = torch.randn(50, 128, generator=torch.Generator().manual_seed(1)).to(HF)
    codes, sc = O.quantise_u4g(x, 32)
    step = sc[..., 0].double().repeat_interleave(32, -1)
    assert ((O.values_u4g(codes, sc) - x.double()).abs() <= step * (0.5 + 15 * 2.0 ** -10)).all()


def test_generic_entry_point_reaches_them():
    f = N.float_bits
    assert N.run("kv_cache_write", [A, 0, A, A, 0, 0, 0], [4, 128, 0, 2, 64, 32, 4, 16, N.TL_U4G, N.TL_BF16], None) == -1 and "null" in N.last_error()
    assert N.run("kv_cache_read", [A, A, A, A, 0, 0, 0], [4, 64, 0, 2, 64, 32, 4, 16, N.TL_U4G, N.TL_BF16], None) == -1
    assert "overlap" in N.last_error()
    meta = [2, 1, 4, 2, 80, 16, 320, 320, 16, 4, 8, f(0.1), N.TL_BF16, 1 << 30]
    assert N.run("attn_decode_paged_int4", [A] * 9, meta, None) == -1 and "64, 128 or 256" in N.last_error()
    assert N.run("gemm_epilogue", [A] * 5, [4, 8, 8, 1, 9, N.TL_BF16, N.TL_BF16], None) == -1 and "activation" in N.last_error()


def test_library_programs_bind():
    from tilelang import programs as P
    from tilelang.engine.matcher import bind
    for prog, entry, names in [
            (P.kv_cache_write(3, 2, 64, 4, 16, 32), "tl_b200_kv_cache_write", "Slots K KCache KScale V VCache VScale"),
            (P.kv_cache_write(3, 1, 576, 4, 64, cache_dtype="float8_e4m3"), "tl_b200_kv_cache_write", "Slots K KCache KScale"),
            (P.kv_cache_read(3, 2, 64, 4, 16, 32), "tl_b200_kv_cache_read", "Slots KCache KScale K VCache VScale V"),
            (P.attn_decode_paged_int4(2, 1, 8, 2, 128, 9, 16, 4), "tl_b200_attn_decode_paged_int4",
             "Q KCache KScale VCache VScale BlockTable CacheSeqlens Out"),
            (P.gemm_epilogue(4, 8, 16, bias=True, activation="gelu", residual=True), "tl_b200_gemm_epilogue", "A B Bias Residual C")]:
        bound = bind(prog)
        assert bound.entry_point == entry and [b.name for b in prog.params] == names.split()
        assert bound.full_outputs == (not entry.startswith("tl_b200_kv"))


def test_sizes_at_the_ends_of_the_ranges():
    assert write(page=2 ** 31, pages=0) == -1 and "too large" in N.last_error()
    assert write(pages=0, kc=None, ks=None) == 0                 # no slot lies in a cache without pages
    big = 2 ** 24 - 1                                            # the product of all three wraps 64 bits
    assert attn(batch=big, s_q=big, h_q=65536) == -1 and "too large" in N.last_error()
    assert N.load().tl_b200_attn_decode_paged_int4_workspace_bytes(big, big, 65536, 2, 64) == 0
    assert gemm(n=2 ** 31 - 8) == -1 and "2^31" in N.last_error()
