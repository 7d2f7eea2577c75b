"""The quantised cache: rows written into 4 bits or e4m3 and read back, against the formats' definition."""
import pytest
import torch

import oracle.ops as O
from tilelang import ops, workloads

pytestmark = pytest.mark.gpu
BF, HF, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def bits(t):
    return t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.uint8 if t.element_size() == 1 else torch.int32)


def u4g_cache(pages, heads, page, dim, group, dtype, dev):
    """A cache full of a pattern, so that a stray write shows."""
    return (torch.full((pages, heads, page, dim // 2), 0xA5, dtype=torch.uint8, device=dev),
            torch.full((pages, heads, page, dim // group, 2), 7.0, dtype=dtype, device=dev))


def rows(tokens, heads, dim, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, heads, dim, generator=g) * torch.exp2(torch.randint(-6, 7, (tokens, heads, 1), generator=g).float())
    return (x + 3 * torch.randn(tokens, heads, 1, generator=g)).to(dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 128)])
@pytest.mark.parametrize("tokens,heads,page", [(1, 1, 1), (5, 3, 7), (67, 8, 16), (130, 2, 48)])
def test_u4g_write_and_read(cuda_device, dtype, dim, group, tokens, heads, page):
    k, v = rows(tokens, heads, dim, dtype, tokens + dim), rows(tokens, heads, dim, dtype, tokens + group)
    pages = tokens // page + 4
    g = torch.Generator().manual_seed(tokens)
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    dev = cuda_device
    kc, ks = u4g_cache(pages, heads, page, dim, group, dtype, dev)
    vc, vs = u4g_cache(pages, heads, page, dim, group, dtype, dev)
    assert ops.kv_cache_write(slots.to(dev), k.to(dev), kc, ks, v.to(dev), vc, vs) == 0
    ko, vo = (torch.full((tokens, heads, dim), -1.0, dtype=dtype, device=dev) for _ in range(2))
    assert ops.kv_cache_read(slots.to(dev), kc, ks, ko, vc, vs, vo) == 0
    at = (slots // page, slice(None), slots % page)
    for x, cache, scale, out in ((k, kc, ks, ko), (v, vc, vs, vo)):
        codes, sc = O.quantise_u4g(x, group)
        want_c, want_s = (t.cpu() for t in u4g_cache(pages, heads, page, dim, group, dtype, "cpu"))
        want_c[at], want_s[at] = codes, sc
        assert torch.equal(cache.cpu(), want_c)                                   # codes and every row that was not written
        assert torch.equal(bits(scale.cpu()), bits(want_s))
        val = O.values_u4g(codes, sc)
        # s * code is exact in fp32; one fp32 rounding of the sum, then half a step of the 16-bit type (2^-25 where it is subnormal)
        tol = (torch.finfo(dtype).eps / 2 + 2.0 ** -23) * val.abs() + 2.0 ** -22 * sc.double().abs().amax(-1).repeat_interleave(group, -1) \
            + (2.0 ** -25 if dtype == HF else 0.0)
        assert ((out.cpu().double() - val).abs() <= tol).all()
        # what the format promises: half a step, and at the top what the rounding of the step takes away (15 steps of it)
        step = sc[..., 0].double().repeat_interleave(group, -1)
        lim = step * (0.5 + 15 * torch.finfo(dtype).eps) + 2.0 ** -22 * x.double().abs() + (15 * 2.0 ** -25 if dtype == HF else 0.0)
        assert ((val - x.double()).abs() <= lim).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tokens,dim,page", [(1, 8, 1), (3, 576, 64), (77, 320, 24), (20, 576, 64), (9, 1024, 16), (10, 640, 5)])
def test_e4m3_write_and_read(cuda_device, dtype, tokens, dim, page):
    x = rows(tokens, 1, dim, dtype, dim)[:, 0].contiguous()
    pages = tokens // page + 3
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(dim))[:tokens]
    dev = cuda_device
    cache = torch.full((pages, page, dim), 0x3A, dtype=torch.uint8, device=dev).view(F8)
    scale = torch.full((pages, page), 7.0, device=dev)
    assert ops.kv_cache_write(slots.to(dev), x.to(dev), cache, scale) == 0
    out = torch.empty(tokens, dim, dtype=dtype, device=dev)
    assert ops.kv_cache_read(slots.to(dev), cache, scale, out) == 0
    b8, sc = O.quantise_row_e4m3(x)
    want = torch.full((pages * page, dim), 0x3A, dtype=torch.uint8)
    want[slots] = b8.view(torch.uint8)
    assert torch.equal(cache.view(torch.uint8).cpu().reshape(-1, dim), want)
    ws = torch.full((pages * page,), 7.0)
    ws[slots] = sc
    assert torch.equal(scale.cpu().reshape(-1), ws)
    assert torch.equal(bits(out.cpu()), bits((b8.float() * sc[:, None]).to(dtype)))      # one fp32 product, one rounding: bit for bit
    old8, old_s = workloads.quantise_tokens_e4m3(x.float())                               # the framework's own quantiser agrees
    assert torch.equal(old8.view(torch.uint8), b8.view(torch.uint8)) and torch.equal(old_s, sc)


def test_padding_and_slots_outside_the_cache_are_skipped(cuda_device):
    dev, dim, page, pages = cuda_device, 64, 16, 3
    x = rows(6, 2, dim, BF, 1)
    slots = torch.tensor([5, -1, pages * page, 40, -2 ** 40, 2 ** 40])
    kc, ks = u4g_cache(pages, 2, page, dim, 32, BF, dev)
    before = kc.clone()
    ops.kv_cache_write(slots.to(dev), x.to(dev), kc, ks)
    changed = (kc != before).any(-1).any(1).cpu().reshape(-1)
    assert changed.nonzero().flatten().tolist() == [5, 40]
    out = torch.full((6, 2, dim), -3.0, dtype=BF, device=dev)
    ops.kv_cache_read(slots.to(dev), kc, ks, out)
    assert (out[[1, 2, 4, 5]] == -3.0).all() and (out[[0, 3]] != -3.0).any()
    c8, s8 = torch.zeros(pages, page, dim, dtype=torch.uint8, device=dev).view(F8), torch.zeros(pages, page, device=dev)
    ops.kv_cache_write(slots.to(dev), x[:, 0].contiguous().to(dev), c8, s8)
    assert (s8.reshape(-1) != 0).nonzero().flatten().tolist() == [5, 40]
    # a slot may be read more than once; no tokens at all is fine
    twice = torch.empty(3, 2, dim, dtype=BF, device=dev)
    ops.kv_cache_read(torch.tensor([5, 40, 5], device=dev), kc, ks, twice)
    assert torch.equal(bits(twice[0]), bits(twice[2])) and torch.equal(bits(twice[0]), bits(out[0]))
    assert ops.kv_cache_write(slots[:0].to(dev), x[:0].to(dev), kc, ks) == 0


@pytest.mark.parametrize("dtype", [BF, HF])
def test_constant_tiny_and_non_finite_groups(cuda_device, dtype):
    dev, dim = cuda_device, 128
    fi = torch.finfo(dtype)
    x = torch.randn(8, 1, dim, generator=torch.Generator().manual_seed(3)).to(dtype)
    x[0] = 2.5                                     # constant: step 0
    x[1] = 0
    x[2] = torch.linspace(-fi.max, fi.max, dim).to(dtype)
    x[3] = torch.linspace(0, 1, dim).to(dtype) * fi.tiny
    x[4, 0, 5] = float("nan")
    x[5, 0, 5] = float("inf")
    x[6, 0, 5] = float("-inf")
    x[7] = -0.0
    kc, ks = u4g_cache(1, 1, 8, dim, 64, dtype, dev)
    slots = torch.arange(8, device=dev)
    ops.kv_cache_write(slots, x.to(dev), kc, ks)
    out = torch.empty(8, 1, dim, dtype=dtype, device=dev)
    ops.kv_cache_read(slots, kc, ks, out)
    out = out.cpu()
    assert (out[0] == 2.5).all() and (out[1] == 0).all() and (out[7] == 0).all()
    for r in (4, 5, 6):                            # the group that holds it is NaN, the other one is as it was
        assert out[r, 0, :64].isnan().all() and not out[r, 0, 64:].isnan().any()
    codes, sc = O.quantise_u4g(x[:4], 64)
    assert torch.equal(kc.cpu()[0, 0, :4], codes[:, 0])
    # row 2 of the bf16 case spans more than fp32 holds (linspace itself gives NaN there): any NaN is as good as another
    assert torch.allclose(ks.cpu()[0, 0, :4].float(), sc[:, 0].float(), rtol=0, atol=0, equal_nan=True)
    c8, s8 = torch.zeros(1, 8, dim, dtype=torch.uint8, device=dev).view(F8), torch.zeros(1, 8, device=dev)
    ops.kv_cache_write(slots, x[:, 0].contiguous().to(dev), c8, s8)
    flat = torch.empty(8, dim, dtype=dtype, device=dev)
    ops.kv_cache_read(slots, c8, s8, flat)
    flat = flat.cpu()
    assert flat[4:7].isnan().all() and (flat[1] == 0).all() and not flat[[0, 1, 3, 7]].isnan().any()


def test_rows_of_a_wider_projection(cuda_device):
    """Keys and values as slices of one QKV output (token stride wider than the row), and read back into such slices."""
    dev, heads, dim = cuda_device, 2, 64
    qkv = torch.randn(33, (4 + 2 * heads) * dim, generator=torch.Generator().manual_seed(5)).to(BF).to(dev)
    k, v = (qkv[:, o:o + heads * dim].unflatten(1, (heads, dim)) for o in (4 * dim, (4 + heads) * dim))
    slots = torch.randperm(48, generator=torch.Generator().manual_seed(6))[:33].to(dev)
    a, b = [u4g_cache(3, heads, 16, dim, 32, BF, dev) for _ in range(2)], [u4g_cache(3, heads, 16, dim, 32, BF, dev) for _ in range(2)]
    ops.kv_cache_write(slots, k, *a[0], v, *a[1])
    ops.kv_cache_write(slots, k.contiguous(), *b[0], v.contiguous(), *b[1])
    for (c, s), (c2, s2) in zip(a, b):
        assert torch.equal(c, c2) and torch.equal(bits(s), bits(s2))
    back = torch.zeros_like(qkv)
    ko = back[:, 4 * dim:(4 + heads) * dim].unflatten(1, (heads, dim))
    ops.kv_cache_read(slots, *a[0], ko)
    assert (back[:, :4 * dim] == 0).all() and (back[:, (4 + heads) * dim:] == 0).all()
    dense = torch.empty(33, heads, dim, dtype=BF, device=dev)
    ops.kv_cache_read(slots, *a[0], dense)
    assert torch.equal(bits(ko), bits(dense))


def test_written_rows_feed_the_mla_decode(cuda_device):
    """The e4m3 writer fills the cache that mla_decode_paged reads: same attention as over the quantiser's own bytes."""
    dev = cuda_device
    w = workloads.mla_fp8_paged(batch=2, heads=16, d=576, dv=512, min_len=50, max_len=150, seed=4)
    x = torch.randn(w["kv_cache"].shape, generator=torch.Generator().manual_seed(8)).to(BF)
    c8, sc = O.quantise_row_e4m3(x)
    cache, scale = torch.zeros_like(c8, device=dev), torch.zeros(sc.shape, device=dev)
    n = x.shape[0] * x.shape[1]
    ops.kv_cache_write(torch.arange(n, device=dev), x.reshape(n, -1).to(dev), cache, scale)
    outs = []
    for c, s in ((cache, scale), (c8.to(dev), sc.to(dev))):
        out = torch.empty(2, 16, 512, dtype=BF, device=dev)
        ops.mla_decode_paged(w["q"].view(2, 16, 576).to(dev), c, s, w["block_table"].to(dev), w["cache_seqlens"].to(dev), out)
        outs.append(out.cpu())
    assert torch.equal(bits(outs[0]), bits(outs[1]))


def test_offsets_beyond_32_bits(cuda_device):
    """The last rows of a cache of more than 2^32 bytes of codes."""
    dev, page, dim = cuda_device, 4096, 256
    pages = (2 ** 32 // (dim // 2)) // page + 2
    cache = torch.zeros(pages, 1, page, dim // 2, dtype=torch.uint8, device=dev)
    scale = torch.zeros(pages, 1, page, 2, 2, dtype=BF, device=dev)
    x = rows(3, 1, dim, BF, 2)
    total = pages * page
    slots = torch.tensor([total - 1, 3, total - page])
    ops.kv_cache_write(slots.to(dev), x.to(dev), cache, scale)
    codes, sc = O.quantise_u4g(x, 128)
    assert torch.equal(cache.view(total, -1)[slots.to(dev)].cpu(), codes[:, 0])
    out = torch.empty(3, 1, dim, dtype=BF, device=dev)
    ops.kv_cache_read(slots.to(dev), cache, scale, out)
    assert torch.equal(bits(out.cpu()), bits(O.values_u4g(codes, sc).float().to(BF)))


def test_on_another_stream_and_in_a_graph(cuda_device):
    dev = cuda_device
    x = rows(40, 2, 128, BF, 9).to(dev)
    slots = torch.arange(40, device=dev)
    kc, ks = u4g_cache(3, 2, 16, 128, 128, BF, dev)
    out = torch.empty_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.kv_cache_write(slots, x, kc, ks)
        ops.kv_cache_read(slots, kc, ks, out)
    for seed in (1, 2):
        x.copy_(rows(40, 2, 128, BF, seed))
        graph.replay()
        torch.cuda.synchronize()
        codes, sc = O.quantise_u4g(x.cpu(), 128)
        assert torch.equal(bits(out.cpu()), bits(O.values_u4g(codes, sc).float().to(BF)))
