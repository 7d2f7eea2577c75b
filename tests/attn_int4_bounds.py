"""Attention over a 4-bit cache in 64 bits, with what the kernel's roundings may add up to for every single element."""
import torch

import oracle.ops as O


def reference(w, scale=None, leave_out=None):
    """(out, tolerance, rms): the definition in 64 bits, the largest error that an element may have, and the root mean square of
    the error that independent roundings give it.  `leave_out(sequence, tokens)`: a mask of tokens to forget, for a check of the bounds.

    A weight times its step, p s, is rounded to 11 bits (2^-11) and has a smallest unit 2^-25 / f, where f brings the largest p s
    of the query, of that group of columns, to 2^4 at least: 2^-29 of it.  It meets a code less 8, at most 8 in size; the value's
    middle, lo + 8 s, and both sums are in fp32 (the tensor core's truncation included: 2^-16).  A score is off by 2^-22 of
    sum |q| (15 s + |lo|), which moves a weight by as much, and the output by that of sum p (|v| + |out|)."""
    q = w["q"]
    b, s_q, h_q, d = q.shape
    pages, h_kv, page, _ = w["k_cache"].shape
    groups, per, n_max = w["k_scale"].shape[3], h_q // h_kv, w["block_table"].shape[1] * page
    scale = d ** -0.5 if scale is None else scale
    out, tol, var = (torch.zeros(b, s_q, h_q, d, dtype=torch.float64) for _ in range(3))
    unit, least = torch.finfo(q.dtype).eps / 2, 2.0 ** -25 if q.dtype == torch.float16 else 0.0         # half a step of subnormals
    for i in range(b):
        n = max(0, min(int(w["cache_seqlens"][i]), n_max))
        at = torch.arange(n)
        pg = w["block_table"][i].long()[at // page] if n else at
        ok = (pg >= 0) & (pg < pages)
        if leave_out is not None:
            ok &= ~leave_out(i, at)
        pg = pg.clamp(0, max(pages - 1, 0))
        for h in range(h_kv):
            ks, vs = (w[s + "_scale"][pg, h, at % page].double() for s in "kv")
            k, v = (O.values_u4g(w[s + "_cache"][pg, h, at % page], w[s + "_scale"][pg, h, at % page]) for s in "kv")
            size = (15 * ks[..., 0].abs() + ks[..., 1].abs()).nan_to_num(0, 0, 0)                      # (n, groups)
            step = vs[..., 0].abs()
            for t in range(s_q):
                see = ok & (at < n - s_q + t + 1)
                if not see.any():
                    continue
                rows = slice(h * per, (h + 1) * per)
                qq = q[i, t, rows].double()
                p = torch.softmax(qq @ k[see].t() * scale, -1)                                          # (per, keys)
                o = p @ v[see]
                off = 2.0 ** -22 * abs(scale) * (qq.abs().unflatten(-1, (groups, -1)).sum(-1) @ size[see].t()).amax(-1, keepdim=True)
                st, mid = step[see], (vs[see][..., 1] + 8 * vs[see][..., 0]).abs()
                wide = lambda x: x.repeat_interleave(d // groups, -1)
                in_mma, beside = wide(p @ (8 * st)), wide(p @ mid)
                unit_w = wide(8 * 2.0 ** -29 * (p[:, :, None] * st[None]).amax(1))                      # of the largest p s, per key
                shift = off * (p @ v[see].abs() + o.abs())
                out[i, t, rows] = o
                tol[i, t, rows] = unit * o.abs() + least + 2 * shift + 2.0 ** -11 * in_mma + 2.0 ** -16 * (in_mma + beside) + int(see.sum()) * unit_w
                about = (v[see] - wide(vs[see][..., 1] + 8 * vs[see][..., 0])) ** 2                    # (s (c - 8))^2
                var[i, t, rows] = ((unit * o.abs()) ** 2 + least ** 2) / 3 + 2.0 ** -22 / 3 * (p ** 2 @ about) + (2 * shift + 2.0 ** -16 * (in_mma + beside)) ** 2 \
                    + int(see.sum()) * unit_w ** 2 / 3
    return out, tol, var.sqrt()


def excess(out, ref, tol, rms):
    """How far `out` is beyond the bounds: the largest error in tolerances, and the largest row's norm in twice its expected
    one (a row has 64 roundings or more, so its norm is near that).  Both are at most 1 for a right answer."""
    err = (out.double() - ref).abs()
    finite = torch.isfinite(ref)
    assert torch.isfinite(out[finite]).all() and not torch.isfinite(out[~finite]).any()
    ratio = torch.where(finite & (err > 0), err / tol, torch.zeros_like(err))
    e, r = torch.where(finite, err, torch.zeros_like(err)).norm(dim=-1), torch.where(finite, rms, torch.zeros_like(rms)).norm(dim=-1)
    norm = torch.where(e > 0, e / (2 * r), torch.zeros_like(e))
    return float(ratio.max()), float(norm.max())


def problem(lens, s_q, h_q, h_kv, dim, group, page, dtype, seed, spare=3):
    """Caches of normal rows, pages in any order."""
    g = torch.Generator().manual_seed(seed)
    lens = torch.tensor(lens, dtype=torch.int32)
    count = (lens + page - 1) // page
    pages = int(count.sum()) + spare
    perm = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.zeros(len(lens), max(1, int(count.max())), dtype=torch.int32)
    at = 0
    for i, n in enumerate(count.tolist()):
        table[i, :n] = perm[at:at + n]
        at += n
    w = {"block_table": table, "cache_seqlens": lens}
    for s in "kv":
        w[s + "_cache"], w[s + "_scale"] = O.quantise_u4g(torch.randn(pages, h_kv, page, dim, generator=g).to(dtype), group)
    w["q"] = torch.randn(len(lens), s_q, h_q, dim, generator=g).to(dtype)
    return w


def rows_of(w, sequence, tokens):
    """(page, row) of tokens of a sequence."""
    page = w["k_cache"].shape[2]
    tokens = torch.as_tensor(tokens)
    return w["block_table"][sequence].long()[tokens // page], tokens % page


def run(w, dev, scale=None):
    from tilelang import ops
    t = {k: v.to(dev) for k, v in w.items()}
    out = torch.full(t["q"].shape, float("nan"), dtype=t["q"].dtype, device=dev)
    ops.attn_decode_paged_int4(t["q"], t["k_cache"], t["k_scale"], t["v_cache"], t["v_scale"], t["block_table"], t["cache_seqlens"], out,
                               softmax_scale=scale)
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    return out.cpu()
