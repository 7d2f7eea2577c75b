"""Attention over the 4-bit paged cache against the definition in 64 bits."""
import pytest
import torch

import oracle.ops as O
from tilelang import ops

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def problem(lens, s_q, h_q, h_kv, dim, group, page, dtype, seed, spread=1.0, spare=3):
    g = torch.Generator().manual_seed(seed)
    lens = torch.tensor(lens, dtype=torch.int32)
    count = (lens.clamp(min=0) + page - 1) // page
    pages = int(count.sum()) + spare
    perm = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.zeros(len(lens), max(1, int(count.max())), dtype=torch.int32)
    at = 0
    for i, n in enumerate(count.tolist()):
        table[i, :n] = perm[at:at + n]
        at += n
    w = {"block_table": table, "cache_seqlens": lens}
    for s in "kv":
        x = torch.randn(pages, h_kv, page, dim, generator=g) * spread
        x[..., :3] *= 4                                             # a few wide channels
        w[s + "_cache"], w[s + "_scale"] = O.quantise_u4g(x.to(dtype), group)
    w["q"] = torch.randn(len(lens), s_q, h_q, dim, generator=g).to(dtype)
    return w


def run(w, dev, scale=None, **other):
    w = {**w, **other}
    t = {k: v.to(dev) if not v.is_cuda else v for k, v in w.items()}
    out = torch.full(t["q"].shape, float("nan"), dtype=t["q"].dtype, device=dev)
    assert ops.attn_decode_paged_int4(t["q"], t["k_cache"], t["k_scale"], t["v_cache"], t["v_scale"], t["block_table"], t["cache_seqlens"], out,
                                      softmax_scale=scale) == 0
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    return out.cpu()


def reference(w, scale=None):
    return O.attn_decode_paged_u4g(w["q"], w["k_cache"], w["k_scale"], w["v_cache"], w["v_scale"], w["block_table"], w["cache_seqlens"],
                                   w["q"].shape[-1] ** -0.5 if scale is None else scale)


def tolerance(w, ref, scale=None):
    """What the roundings can add up to.  Scores: products with codes offset by 128 are summed in fp32, 2^-22 of the sum of
    their magnitudes; a score that is d off moves its weight by d, and the output by 2 d of the largest value.  Weights times
    steps are rounded to 11 bits (2^-11) or, where they are subnormal, by 2^-25 of the largest, once per key, against at most
    8 steps and their middle; the output once more to its type."""
    d = w["q"].shape[-1]
    scale = abs(d ** -0.5 if scale is None else scale)
    live = torch.isfinite(w["k_scale"].float()).all(-1) & torch.isfinite(w["v_scale"].float()).all(-1)
    ks, vs = w["k_scale"].double()[live], w["v_scale"].double()[live]
    kmax, vmax = float((144 * ks[:, 0] + ks[:, 1].abs()).max()), float((15 * vs[:, 0]).max() + vs[:, 1].abs().max())
    off = 2.0 ** -22 * scale * float(w["q"].double().abs().sum(-1).max()) * kmax
    n = max(1, int(w["cache_seqlens"].max()))
    return torch.finfo(w["q"].dtype).eps / 2 * ref.abs() + 2 * off * vmax + (2.0 ** -11 + n * 2.0 ** -25 + 2.0 ** -16) * vmax


def check(w, dev, scale=None):
    out, ref = run(w, dev, scale), reference(w, scale)
    assert not out.isnan().any()
    err = (out.double() - ref).abs()
    assert (err <= tolerance(w, ref, scale)).all(), float((err / tolerance(w, ref, scale)).max())
    return out


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)])
def test_dims_groups_and_types(cuda_device, dtype, dim, group):
    check(problem([1, 130, 0, 77], 1, 8, 2, dim, group, 16, dtype, dim + group), cuda_device)


@pytest.mark.parametrize("s_q,h_q,h_kv", [(1, 1, 1), (1, 7, 7), (1, 8, 1), (1, 16, 2), (1, 14, 2), (2, 8, 2), (5, 6, 2), (4, 16, 2), (3, 24, 1),
                                          (1, 64, 1), (2, 64, 1), (40, 4, 2)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_head_layouts_and_query_tokens(cuda_device, s_q, h_q, h_kv, dim):
    check(problem([200, 3, 65, 0], s_q, h_q, h_kv, dim, 64, 32, BF, s_q + h_q), cuda_device)


@pytest.mark.parametrize("page", [1, 3, 16, 24, 64, 100, 256])
def test_pages_that_end_inside_a_tile(cuda_device, page):
    check(problem([1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257], 1, 4, 1, 64, 32, page, HF, page), cuda_device)


@pytest.mark.parametrize("lens", [[3000], [2999, 1, 0, 1500], [5000] + [17] * 30, [40] * 200])
@pytest.mark.parametrize("s_q", [1, 3])
def test_long_ragged_and_many(cuda_device, lens, s_q):
    check(problem(lens, s_q, 8, 2, 128, 128, 64, BF, len(lens)), cuda_device)


def test_peaked_scores_and_other_scales(cuda_device):
    """Scores of hundreds, rising and falling along the keys: the running maximum is replaced late and early."""
    for seed, scale in ((1, 2.0), (2, -1.0), (3, 0.0), (4, 1e-3)):
        w = problem([700, 33], 1, 4, 1, 64, 64, 16, BF, seed, spread=3.0)
        check(w, cuda_device, scale)


@pytest.mark.parametrize("dtype,spread", [(HF, 2.0 ** -12), (HF, 2.0 ** 8), (BF, 2.0 ** -60), (BF, 2.0 ** 40)])
def test_small_and_large_values(cuda_device, dtype, spread):
    """Steps far from 1, where weights times steps would leave the range of 16 bits if they were not scaled."""
    w = problem([300, 5], 1, 8, 2, 128, 64, 16, dtype, 11)
    for s in ("v_scale",):
        w[s] = (w[s].float() * spread).to(dtype)
    check(w, cuda_device)


def test_steps_of_very_different_size(cuda_device):
    """Tokens whose steps differ by 2^16, small ones first, then large ones, then small ones again."""
    for dtype in (BF, HF):
        w = problem([96 * 16], 1, 4, 1, 64, 32, 16, dtype, 12)
        pg = w["block_table"][0].long()
        for a, b in ((0, 40), (60, 96)):
            w["v_scale"][pg[a:b]] = (w["v_scale"][pg[a:b]].float() * 2.0 ** -10).to(dtype)
        check(w, cuda_device)
        w["v_scale"][:] = 0                                          # all values zero
        assert (run(w, cuda_device) == 0).all()


def test_rows_behind_the_last_token_may_hold_anything(cuda_device):
    w = problem([37, 100, 0], 2, 8, 2, 128, 32, 64, BF, 21)
    ref = run(w, cuda_device)
    seen = torch.zeros(w["k_cache"].shape[0], 64, dtype=torch.bool)
    for i, n in enumerate(w["cache_seqlens"].tolist()):
        for t in range(n):
            seen[int(w["block_table"][i, t // 64]), t % 64] = True
    for s in "kv":
        w[s + "_cache"].transpose(1, 2)[~seen] = 0xFF
        w[s + "_scale"].transpose(1, 2)[~seen] = float("nan")
    assert torch.equal(run(w, cuda_device).view(torch.int16), ref.view(torch.int16))


def test_non_finite_values_that_are_seen(cuda_device):
    w = problem([50, 50], 1, 4, 2, 64, 32, 16, BF, 22)
    pg = int(w["block_table"][0, 1])
    w["v_scale"][pg, 0, 3] = float("nan")                            # sequence 0, token 19, kv head 0
    out = run(w, cuda_device)
    assert out[0, 0, :2].isnan().all() and not out[0, 0, 2:].isnan().any() and not out[1].isnan().any()
    w = problem([50, 50], 1, 4, 2, 64, 32, 16, BF, 22)
    w["k_scale"][pg, 1, 3] = float("nan")
    out = run(w, cuda_device)
    assert out[0, 0, 2:].isnan().all() and not out[0, 0, :2].isnan().any() and not out[1].isnan().any()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_queries_of_very_different_size(cuda_device, dtype):
    """Heads of one kv head 2^10 (fp16) or 2^40 (bf16) apart: each against a tolerance of its own."""
    w = problem([150], 1, 4, 1, 128, 64, 16, dtype, 26)
    factor = torch.tensor([1.0, 2.0 ** -5, 2.0 ** -10, 2.0 ** 4] if dtype == HF else [1.0, 2.0 ** -20, 2.0 ** -40, 2.0 ** 4])
    w["q"] = (w["q"].float() * factor[None, None, :, None]).to(dtype)
    out, ref = run(w, cuda_device), reference(w)
    for h in range(4):
        one = {**w, "q": w["q"][:, :, h:h + 1]}
        assert ((out[:, :, h].double() - ref[:, :, h]).abs() <= tolerance(one, ref[:, :, h])).all()


def test_non_finite_queries(cuda_device):
    w = problem([90], 1, 4, 1, 64, 32, 16, BF, 27)
    ref = run(w, cuda_device)
    w["q"][0, 0, 1, 3] = float("nan")
    w["q"][0, 0, 2, 5] = float("inf")
    out = run(w, cuda_device)
    assert out[0, 0, 1].isnan().all() and out[0, 0, 2].isnan().all()             # infinity meets keys of both signs
    assert torch.equal(out[0, 0, [0, 3]].view(torch.int16), ref[0, 0, [0, 3]].view(torch.int16))


def test_bad_pages_and_lengths(cuda_device):
    """Ids outside the cache mask their tokens; a length beyond the table is cut to it, a negative one is empty."""
    w = problem([160, 160, 160, 64], 2, 8, 2, 64, 64, 16, BF, 23)
    w["block_table"][0, 3] = -1
    w["block_table"][0, 9] = 2 ** 31 - 1
    w["block_table"][1, :] = w["k_cache"].shape[0]
    w["cache_seqlens"][2] = 10 ** 6
    w["cache_seqlens"][3] = -5
    out = check(w, cuda_device)
    assert (out[1] == 0).all() and (out[3] == 0).all()


def test_a_page_of_two_sequences(cuda_device):
    """A shared prefix: two sequences, and one sequence twice over, name the same pages."""
    w = problem([96, 80], 1, 4, 1, 64, 32, 16, HF, 24)
    w["block_table"][1, :4] = w["block_table"][0, :4]
    w["block_table"][0, 5] = w["block_table"][0, 0]
    check(w, cuda_device)


def test_query_slices_and_streams(cuda_device):
    """q as a slice of a QKV projection; the call on a side stream."""
    dev = cuda_device
    w = problem([70, 9], 3, 8, 2, 64, 32, 16, BF, 25)
    qkv = torch.randn(2, 3, (8 + 4) * 64, generator=torch.Generator().manual_seed(1)).to(BF).to(dev)
    q = qkv[:, :, :512].unflatten(2, (8, 64))
    a = run(w, dev, q=q)
    b = run(w, dev, q=q.contiguous())
    assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(run(w, dev, q=q).view(torch.int16), a.view(torch.int16))


def test_two_graphs_and_eager_calls_at_once(cuda_device):
    """Two graphs captured on one stream and replayed on two, with eager calls between: no scratch is shared, and the
    answer is the same every time."""
    dev = cuda_device
    probs = [problem([4000, 11, 900], 1, 8, 2, 128, 128, 64, BF, s) for s in (31, 32)]
    t = [{k: v.to(dev) for k, v in w.items()} for w in probs]
    refs = [run(w, dev) for w in t]
    outs = [torch.zeros(w["q"].shape, dtype=BF, device=dev) for w in t]
    cap = torch.cuda.Stream()
    graphs = []
    for w, o in zip(t, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=cap):
            ops.attn_decode_paged_int4(w["q"], w["k_cache"], w["k_scale"], w["v_cache"], w["v_scale"], w["block_table"], w["cache_seqlens"], o)
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(20):
        for o in outs:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = run(t[rep % 2], dev)
        torch.cuda.synchronize()
        for o, r in zip(outs, refs):
            assert torch.equal(o.cpu().view(torch.int16), r.view(torch.int16))
        assert torch.equal(eager.view(torch.int16), refs[rep % 2].view(torch.int16))


def test_offsets_beyond_32_bits(cuda_device):
    """Pages behind the first 2^32 bytes of codes."""
    dev, page, dim = cuda_device, 1024, 128
    pages = 2 ** 32 // (page * dim // 2) + 3
    w = problem([300], 1, 2, 1, dim, 128, page, BF, 41, spare=0)
    big = {"q": w["q"], "block_table": torch.tensor([[pages - 1]], dtype=torch.int32), "cache_seqlens": w["cache_seqlens"]}
    for s in "kv":
        for n, shape in (("_cache", (pages, 1, page, dim // 2)), ("_scale", (pages, 1, page, 1, 2))):
            big[s + n] = torch.zeros(shape, dtype=w[s + n].dtype, device=dev)
            big[s + n][pages - 1] = w[s + n][0].to(dev)
    assert torch.equal(run(big, dev).view(torch.int16), run(w, dev).view(torch.int16))


def test_no_sequences_and_no_pages(cuda_device):
    w = problem([5], 1, 2, 1, 64, 32, 16, BF, 42)
    assert run(w, cuda_device, q=w["q"][:0], block_table=w["block_table"][:0], cache_seqlens=w["cache_seqlens"][:0]).shape[0] == 0
    empty = {k: w[k][:0] for k in ("k_cache", "k_scale", "v_cache", "v_scale")}
    assert (run(w, cuda_device, **empty) == 0).all()
    assert (run(w, cuda_device, block_table=w["block_table"][:, :0]) == 0).all()


def test_a_decode_step_with_all_of_them(cuda_device):
    """Projection with bias -> write keys and values -> attention -> projection added to the residual stream, twice, as one
    captured step, against the same in 64 bits on what each operator was given."""
    dev, b, h_q, h_kv, dim, width, page = cuda_device, 5, 8, 2, 64, 256, 16
    g = torch.Generator().manual_seed(51)
    wqkv = (torch.randn((h_q + 2 * h_kv) * dim, width, generator=g) * width ** -0.5).to(BF).to(dev)
    bias = torch.randn((h_q + 2 * h_kv) * dim, generator=g).to(BF).to(dev)
    wo = (torch.randn(width, h_q * dim, generator=g) * (h_q * dim) ** -0.5).to(BF).to(dev)
    w = problem([30, 1, 16, 100, 64], 1, h_q, h_kv, dim, 32, page, BF, 52)
    t = {k: v.to(dev) for k, v in w.items()}
    x = torch.randn(b, width, generator=g).to(BF).to(dev)
    start = x.clone()
    qkv = torch.empty(b, wqkv.shape[0], dtype=BF, device=dev)
    att = torch.empty(b, 1, h_q, dim, dtype=BF, device=dev)
    last = (t["cache_seqlens"] - 1).long()
    slots = t["block_table"].gather(1, (last // page)[:, None])[:, 0].long() * page + last % page

    def step():
        ops.gemm_epilogue(x, wqkv, qkv, bias=bias, transpose_b=True)
        k = qkv[:, h_q * dim:(h_q + h_kv) * dim].unflatten(1, (h_kv, dim))
        v = qkv[:, (h_q + h_kv) * dim:].unflatten(1, (h_kv, dim))
        ops.kv_cache_write(slots, k, t["k_cache"], t["k_scale"], v, t["v_cache"], t["v_scale"])
        ops.attn_decode_paged_int4(qkv[:, None, :h_q * dim].unflatten(2, (h_q, dim)), t["k_cache"], t["k_scale"], t["v_cache"], t["v_scale"],
                                   t["block_table"], t["cache_seqlens"], att)
        ops.gemm_epilogue(att.view(b, -1), wo, x, residual=x, transpose_b=True)

    step()
    x.copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(2):
        before = x.cpu()
        graph.replay()
        torch.cuda.synchronize()
        host = {k: v.cpu() for k, v in t.items()}
        ref_qkv = O.gemm_epilogue(before, wqkv.cpu(), bias=bias.cpu(), transpose_b=True)
        assert torch.allclose(qkv.cpu().double(), ref_qkv, rtol=2.0 ** -8, atol=1e-4)
        kc, ks = O.quantise_u4g(qkv.cpu()[:, h_q * dim:(h_q + h_kv) * dim].unflatten(1, (h_kv, dim)), 32)
        at = (slots.cpu() // page, slice(None), slots.cpu() % page)
        assert torch.equal(host["k_cache"][at], kc) and torch.equal(host["k_scale"][at].view(torch.int16), ks.view(torch.int16))
        host["q"] = qkv.cpu()[:, None, :h_q * dim].unflatten(2, (h_q, dim))
        ref = reference(host)
        assert ((att.cpu().double() - ref).abs() <= tolerance(host, ref)).all()
        ref_x = O.gemm_epilogue(att.cpu().view(b, -1), wo.cpu(), residual=before, transpose_b=True)
        assert torch.allclose(x.cpu().double(), ref_x, rtol=2.0 ** -8, atol=1e-4)


def test_the_same_through_compiled_programs(cuda_device):
    """Write, attention and projection as library programs with host tensors: the same bits as the operators."""
    import tilelang
    from tilelang import programs as P
    dev, h_q, h_kv, dim, page = cuda_device, 8, 2, 64, 16
    w = problem([40, 7], 1, h_q, h_kv, dim, 32, page, BF, 61)
    pages, tokens = w["k_cache"].shape[0], 2
    g = torch.Generator().manual_seed(62)
    k, v = (torch.randn(tokens, h_kv, dim, generator=g).to(BF) for _ in range(2))
    last = (w["cache_seqlens"] - 1).long()
    slots = w["block_table"].gather(1, (last // page)[:, None])[:, 0].long() * page + last % page
    t = {n: x.to(dev) for n, x in w.items()}
    ops.kv_cache_write(slots.to(dev), k.to(dev), t["k_cache"], t["k_scale"], v.to(dev), t["v_cache"], t["v_scale"])
    ref = run(t, dev)
    write = tilelang.compile(P.kv_cache_write(tokens, h_kv, dim, pages, page, 32), out_idx=[2, 3, 5, 6], target="b200")
    assert write(slots, k, w["k_cache"], w["k_scale"], v, w["v_cache"], w["v_scale"]) == 0
    for n in ("k_cache", "v_cache"):
        assert torch.equal(w[n], t[n].cpu())
    attn = tilelang.compile(P.attn_decode_paged_int4(2, 1, h_q, h_kv, dim, pages, page, w["block_table"].shape[1], 32), out_idx=-1, target="b200")
    out = torch.zeros_like(w["q"])
    assert attn(w["q"], w["k_cache"], w["k_scale"], w["v_cache"], w["v_scale"], w["block_table"], w["cache_seqlens"], out) == 0
    assert torch.equal(out.view(torch.int16), ref.view(torch.int16))
    read = tilelang.compile(P.kv_cache_read(tokens, h_kv, dim, pages, page, 32), out_idx=[3, 6], target="b200")
    ko, vo = torch.zeros_like(k), torch.zeros_like(v)
    assert read(slots, w["k_cache"], w["k_scale"], ko, w["v_cache"], w["v_scale"], vo) == 0
    codes, sc = O.quantise_u4g(k, 32)
    assert torch.equal(ko.view(torch.int16), O.values_u4g(codes, sc).float().to(BF).view(torch.int16))
    wo = (torch.randn(96, h_q * dim, generator=g) * 0.05).to(BF)
    res, bias, c = torch.randn(2, 96, generator=g).to(BF), torch.randn(96, generator=g).to(BF), torch.zeros(2, 96, dtype=BF)
    proj = tilelang.compile(P.gemm_epilogue(2, 96, h_q * dim, bias=True, activation="silu", residual=True, transpose_b=True), out_idx=-1, target="b200")
    assert proj(out.view(2, -1), wo, bias, res, c) == 0
    assert torch.allclose(c.double(), O.gemm_epilogue(out.view(2, -1), wo, bias, "silu", res, True), rtol=2.0 ** -8, atol=1e-4)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_long_sequences_keep_the_precision_of_their_output(cuda_device, dtype):
    """Errors of one sign must not add up over a long sequence.  Relative to the output in the 2-norm, its own rounding is uniform
    within half a step at most, 2^-11 / sqrt 3 for fp16 (2^-8 / sqrt 3 for bf16), and the weights' (2^-11 each, of either sign,
    so they add up like the values themselves) 2^-11 / sqrt 3 again: together 2^-11 sqrt(2/3).  A bf16 output's weights meet
    codes of one sign, at most twice the values about zero."""
    g = torch.Generator(device=cuda_device).manual_seed(4)
    n, d, page, batch, h_q = 100000, 64, 64, 60, 8
    pages = (n + page - 1) // page
    w = {"block_table": torch.arange(pages, dtype=torch.int32, device=cuda_device).repeat(batch, 1),       # one cache, 60 queries
         "cache_seqlens": torch.full((batch,), n, dtype=torch.int32, device=cuda_device)}
    for s in "kv":
        x = torch.randn(pages * page, 1, d, generator=g, device=cuda_device).to(dtype)
        w[s + "_cache"] = torch.empty(pages, 1, page, d // 2, dtype=torch.uint8, device=cuda_device)
        w[s + "_scale"] = torch.empty(pages, 1, page, 1, 2, dtype=dtype, device=cuda_device)
        ops.kv_cache_write(torch.arange(pages * page, device=cuda_device), x, w[s + "_cache"], w[s + "_scale"])
    w["q"] = torch.randn(batch, 1, h_q, d, generator=g, device=cuda_device).to(dtype)
    out = run(w, cuda_device).double().flatten(0, 2)
    k, v = (O.values_u4g(w[s + "_cache"].cpu(), w[s + "_scale"].cpu()).double().reshape(-1, d)[:n].to(cuda_device) for s in "kv")
    ref = (torch.softmax(w["q"].double().reshape(-1, d) @ k.T * d ** -0.5, -1) @ v).cpu()
    bound = 2.0 ** -11 * (2 / 3) ** 0.5 if dtype is HF else (2.0 ** -16 / 3 + 4 * 2.0 ** -22 / 3) ** 0.5
    err = float((out - ref).norm() / ref.norm())
    assert err <= bound, (err, bound)
