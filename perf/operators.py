"""Cases of the serving operators around a quantised key/value cache, in plain form and as the framework's calls.

Operators: `kv_cache_write` / `kv_cache_read` (a paged cache held as 4-bit codes with a scale and a minimum per group, or
as e4m3 rows with one scale each), `attn_decode_paged_int4` (attention over the 4-bit cache) and `gemm_epilogue` (matrix
product with bias, activation and residual in its epilogue).

The 4-bit cache: codes (pages, kv heads, page, dim / 2) uint8, the value of an even column in the low four bits of a
byte; scale (pages, kv heads, page, dim / group, 2) in the 16-bit type of the model, a group's step s and its minimum lo;
a value is s * code + lo.  The e4m3 cache: (pages, page, dim) with an fp32 scale per row, (pages, page).
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one new token for each of 64 sequences, as every decode step writes them: a latency
        dict(name="write int4 64 tokens", op="write", fmt="int4", tokens=64, heads=8, dim=128, group=128, page=64, dtype="bf16"),
        # the prompt of a prefill step: keys and values of 8192 tokens at 8 heads of 128
        dict(name="write int4 8192 tokens", op="write", fmt="int4", tokens=8192, heads=8, dim=128, group=64, page=64, dtype="bf16"),
        # the same for a latent cache (512 + 64 columns a row), a ragged number of tokens
        dict(name="write e4m3 8179 tokens", op="write", fmt="e4m3", tokens=8179, heads=1, dim=576, group=576, page=64, dtype="bf16"),
        # a shared prefix read back in 16 bits for a prefill on top of it: small heads, fine groups
        dict(name="read int4 32771 tokens", op="read", fmt="int4", tokens=32771, heads=4, dim=64, group=32, page=32, dtype="fp16"),
        # the same for the latent cache
        dict(name="read e4m3 65500 tokens", op="read", fmt="e4m3", tokens=65500, heads=1, dim=576, group=576, page=64, dtype="bf16"),
        # one short conversation: a latency
        dict(name="attn 1 x 777", op="attn", batch=1, s_q=1, q_heads=32, heads=8, dim=128, group=128, page=64, min_len=777, max_len=777,
             dtype="bf16"),
        # a full decode batch of mixed lengths
        dict(name="attn 64 x 2k-12k", op="attn", batch=64, s_q=1, q_heads=32, heads=8, dim=128, group=128, page=64, min_len=2048,
             max_len=12288, dtype="bf16"),
        # one long document
        dict(name="attn 1 x 131077", op="attn", batch=1, s_q=1, q_heads=32, heads=8, dim=128, group=64, page=128, min_len=131077,
             max_len=131077, dtype="bf16"),
        # several tokens a sequence are verified at once; new sequences (some still empty) beside long ones
        dict(name="attn 24 x 4 tokens 0-5k", op="attn", batch=24, s_q=4, q_heads=16, heads=2, dim=64, group=32, page=16, min_len=0,
             max_len=5000, dtype="fp16"),
        # projection of a small decode batch with its bias
        dict(name="gemm 16 bias", op="gemm", m=16, n=6144, k=4096, bias=True, act="none", residual=False, trans_b=True, dtype="bf16"),
        # down projection of a decode batch, added to the residual stream
        dict(name="gemm 61 residual", op="gemm", m=61, n=4096, k=14336, bias=False, act="none", residual=True, trans_b=True, dtype="bf16"),
        # up projection of a prefill step with bias and GELU, weights as (inputs, outputs)
        dict(name="gemm 8192 bias gelu", op="gemm", m=8192, n=14336, k=4096, bias=True, act="gelu", residual=False, trans_b=False,
             dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "attn", "attn", "gemm", "gemm"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op in ("write", "read"):
        tokens = _log(rng, 1, 8192 if op == "write" else 32768)
        page = rng.choice([16, 24, 64, 128])
        if rng.random() < 0.35:
            return dict(op=op, fmt="e4m3", tokens=tokens, heads=1, dim=rng.choice([128, 320, 576]), group=0, page=page, dtype=dtype)
        dim = rng.choice([64, 128, 256])
        return dict(op=op, fmt="int4", tokens=tokens, heads=rng.choice([1, 2, 5, 8]), dim=dim, group=rng.choice([g for g in (32, 64, 128) if g <= dim]),
                    page=page, dtype=dtype)
    if op == "attn":
        heads = rng.choice([1, 2, 4, 8])
        dim = rng.choice([64, 128, 128, 256])
        batch = _log(rng, 1, 64)
        most = min(131072, 64 * 7000 * 8 * 128 // (batch * heads * dim))     # no more of the cache than the largest listed case
        max_len = _log(rng, 1, most)
        s_q = rng.choice([1, 1, 1, 2, 5])
        return dict(op="attn", batch=batch, s_q=s_q, q_heads=heads * rng.choice([1, 2, 4, 7, 8]), heads=heads, dim=dim,
                    group=rng.choice([g for g in (32, 64, 128) if g <= dim]), page=rng.choice([16, 24, 64, 128]),
                    min_len=rng.choice([0, max_len // 2, max_len]), max_len=max_len, dtype=dtype)
    trans_b = rng.random() < 0.7
    m, k = _log(rng, 1, 8192), 8 * _log(rng, 8, 1024)
    n = _log(rng, 64, 14336)
    if not trans_b:
        n = (n + 7) // 8 * 8
    return dict(op="gemm", m=m, n=n, k=k, bias=rng.random() < 0.6, act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]),
                residual=rng.random() < 0.5, trans_b=trans_b, dtype=dtype)


def _group(case):
    return case["group"] or case["dim"]


# ------------------------------------------------------------------------------------------------- inputs
def _activations(g, shape, dtype):
    """Keys or values: normal, with a few channels of larger spread, as projections give them."""
    spread = 1.0 + 3.0 * (torch.rand(shape[-2:], generator=g, device="cuda") > 0.95).float()
    return (torch.randn(shape, generator=g, device="cuda") * spread).to(dtype)


def _random_int4(g, pages, heads, page, dim, group, dtype):
    """A cache already filled: codes, and steps and minima as normal rows have them."""
    codes = torch.randint(0, 256, (pages, heads, page, dim // 2), generator=g, device="cuda", dtype=torch.uint8)
    shape = (pages, heads, page, dim // group)
    step = 0.25 + 0.15 * torch.rand(shape, generator=g, device="cuda")
    lo = -7.5 * step + 0.4 * torch.randn(shape, generator=g, device="cuda")
    return codes, torch.stack((step, lo), -1).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]
    op = case["op"]
    s = {"case": case, "op": op}
    if op in ("write", "read"):
        t, h, d, page = case["tokens"], case["heads"], case["dim"], case["page"]
        pages = t // page + 9
        # the tokens of a sequence fill a page in order; pages come in any order
        order = torch.randperm(pages, generator=g, device="cuda")
        at = torch.arange(t, device="cuda")
        s["slots"] = order[at // page] * page + at % page
        if case["fmt"] == "int4":
            grp = _group(case)
            for w in "kv":
                if op == "write":
                    s[w] = _activations(g, (t, h, d), dt)
                    s[w + "_cache"] = torch.zeros(pages, h, page, d // 2, dtype=torch.uint8, device="cuda")
                    s[w + "_scale"] = torch.zeros(pages, h, page, d // grp, 2, dtype=dt, device="cuda")
                else:
                    s[w + "_cache"], s[w + "_scale"] = _random_int4(g, pages, h, page, d, grp, dt)
                s[w + "_out"] = torch.empty(t, h, d, dtype=dt, device="cuda")
        else:
            if op == "write":
                s["k"] = _activations(g, (t, d), dt)
                s["k_cache"] = torch.zeros(pages, page, d, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
                s["k_scale"] = torch.zeros(pages, page, dtype=torch.float32, device="cuda")
            else:
                x = torch.randn(pages, page, d, generator=g, device="cuda")
                s["k_scale"] = x.abs().amax(-1) / 448.0
                s["k_cache"] = (x / s["k_scale"][..., None]).to(torch.float8_e4m3fn)
            s["k_out"] = torch.empty(t, d, dtype=dt, device="cuda")
        return s
    if op == "attn":
        b, h, d, page = case["batch"], case["heads"], case["dim"], case["page"]
        lens = torch.randint(case["min_len"], case["max_len"] + 1, (b,), generator=g, device="cuda")
        if b > 1 and case["min_len"] < case["max_len"]:
            lens[0], lens[1] = case["min_len"], case["max_len"]
        per = -(-case["max_len"] // page)
        count = (lens + page - 1) // page
        # every sequence has pages of its own, in any order; table entries behind a sequence's last page are 0
        pages = int(count.sum()) + 5
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        first = torch.cumsum(count, 0) - count
        at = torch.arange(per, device="cuda")
        table = torch.where(at[None] < count[:, None], order[(first[:, None] + at[None]).clamp(max=pages - 1)], 0).to(torch.int32)
        s["block_table"], s["cache_seqlens"] = table.contiguous(), lens.to(torch.int32)
        for w in "kv":
            s[w + "_cache"], s[w + "_scale"] = _random_int4(g, pages, h, page, d, _group(case), dt)
        s["q"] = torch.randn(b, case["s_q"], case["q_heads"], d, generator=g, device="cuda").to(dt)
        s["out"] = torch.empty_like(s["q"])
        return s
    m, n, k = case["m"], case["n"], case["k"]
    s["a"] = torch.randn(m, k, generator=g, device="cuda").to(dt)
    s["b"] = (torch.randn((n, k) if case["trans_b"] else (k, n), generator=g, device="cuda") * k ** -0.5).to(dt)
    s["bias"] = torch.randn(n, generator=g, device="cuda").to(dt) if case["bias"] else None
    s["residual"] = torch.randn(m, n, generator=g, device="cuda").to(dt) if case["residual"] else None
    s["c"] = torch.empty(m, n, dtype=dt, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------- plain forms
def _unpacked(codes):
    return torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()


def _values(codes, scale, dim):
    """Values of 4-bit rows (..., dim / 2) with (..., groups, 2), in 32 bits."""
    groups = scale.shape[-2]
    c = _unpacked(codes).unflatten(-1, (groups, dim // groups))
    sc = scale.float()
    return (c * sc[..., :1] + sc[..., 1:]).flatten(-2)


def _plain_write_int4(x, page_at, row, cache, scale):
    groups = scale.shape[-2]
    xf = x.float().unflatten(-1, (groups, x.shape[-1] // groups))
    lo = xf.amin(-1, keepdim=True)
    step = ((xf.amax(-1, keepdim=True) - lo) / torch.full_like(lo, 15.0)).to(x.dtype).float()     # by a tensor: a division, not a reciprocal
    code = torch.where(step > 0, torch.round((xf - lo) / step), torch.zeros_like(xf)).clamp(0, 15).to(torch.uint8).flatten(-2)
    cache[page_at, :, row] = code[..., 0::2] | (code[..., 1::2] << 4)
    scale[page_at, :, row] = torch.cat((step, lo), -1).to(scale.dtype)


def _plain_write_e4m3(x, page_at, row, cache, scale):
    xf = x.float()
    sc = xf.abs().amax(-1).clamp(min=1e-4)
    sc = sc / torch.full_like(sc, 448.0)
    cache.view(torch.uint8)[page_at, row] = (xf / sc[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
    scale[page_at, row] = sc


def _plain_cache(s):
    c = s["case"]
    dt = _DTYPES[c["dtype"]]
    page_at, row = s["slots"] // c["page"], s["slots"] % c["page"]
    if c["fmt"] == "e4m3":
        if s["op"] == "write":
            _plain_write_e4m3(s["k"], page_at, row, s["k_cache"], s["k_scale"])
        return (s["k_cache"].view(torch.uint8)[page_at, row].view(torch.float8_e4m3fn).float() * s["k_scale"][page_at, row][..., None]).to(dt)
    if s["op"] == "write":
        _plain_write_int4(s["k"], page_at, row, s["k_cache"], s["k_scale"])
        _plain_write_int4(s["v"], page_at, row, s["v_cache"], s["v_scale"])
    return (_values(s["k_cache"][page_at, :, row], s["k_scale"][page_at, :, row], c["dim"]).to(dt),
            _values(s["v_cache"][page_at, :, row], s["v_scale"][page_at, :, row], c["dim"]).to(dt))


def _plain_attn(s):
    q, table, lens = s["q"], s["block_table"].long(), s["cache_seqlens"].long()
    b, s_q, hq, d = q.shape
    h = s["k_cache"].shape[1]
    k = _values(s["k_cache"][table].transpose(1, 2).flatten(2, 3), s["k_scale"][table].transpose(1, 2).flatten(2, 3), d)
    qh = q.float().view(b, s_q, h, hq // h, d).permute(0, 2, 1, 3, 4).flatten(2, 3)              # (b, h, s_q * group, d)
    logits = torch.matmul(qh, k.transpose(-1, -2)) * d ** -0.5
    del k
    seen = lens[:, None] - s_q + torch.arange(s_q, device=q.device)[None] + 1                    # keys that token i of a sequence sees
    hidden = torch.arange(logits.shape[-1], device=q.device)[None, None] >= seen[..., None]      # (b, s_q, keys)
    hidden = hidden.repeat_interleave(hq // h, 1)[:, None]
    logits = logits.masked_fill(hidden, float("-inf"))
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    v = _values(s["v_cache"][table].transpose(1, 2).flatten(2, 3), s["v_scale"][table].transpose(1, 2).flatten(2, 3), d)
    o = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    return o.view(b, h, s_q, hq // h, d).permute(0, 2, 1, 3, 4).reshape(b, s_q, hq, d).to(q.dtype)


def _plain_gemm(s):
    b = s["b"].float()
    x = torch.matmul(s["a"].float(), b.t() if s["case"]["trans_b"] else b)
    if s["bias"] is not None:
        x = x + s["bias"].float()
    act = s["case"]["act"]
    if act == "relu":
        x = torch.where(x > 0, x, torch.zeros_like(x))
    elif act == "silu":
        x = x / (1 + torch.exp(-x))
    elif act == "gelu":
        x = 0.5 * x * (1 + torch.erf(x * 0.7071067811865476))
    elif act == "gelu_tanh":
        x = 0.5 * x * (1 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x)))
    if s["residual"] is not None:
        x = x + s["residual"].float()
    return x.to(s["a"].dtype)


# ------------------------------------------------------------------------------------------------- one pass
def run(s):
    op = s["op"]
    if not own:
        return _plain_cache(s) if op in ("write", "read") else _plain_attn(s) if op == "attn" else _plain_gemm(s)
    ops = _ops()
    if op in ("write", "read"):
        if s["case"]["fmt"] == "e4m3":
            if op == "write":
                ops.kv_cache_write(s["slots"], s["k"], s["k_cache"], s["k_scale"])
            ops.kv_cache_read(s["slots"], s["k_cache"], s["k_scale"], s["k_out"])
            return s["k_out"]
        if op == "write":
            ops.kv_cache_write(s["slots"], s["k"], s["k_cache"], s["k_scale"], s["v"], s["v_cache"], s["v_scale"])
        ops.kv_cache_read(s["slots"], s["k_cache"], s["k_scale"], s["k_out"], s["v_cache"], s["v_scale"], s["v_out"])
        return s["k_out"], s["v_out"]
    if op == "attn":
        ops.attn_decode_paged_int4(s["q"], s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"], s["block_table"], s["cache_seqlens"],
                                   s["out"])
        return s["out"]
    ops.gemm_epilogue(s["a"], s["b"], s["c"], bias=s["bias"], activation=s["case"]["act"], residual=s["residual"],
                      transpose_b=s["case"]["trans_b"])
    return s["c"]


def _ops():
    import sys
    if "tilelang-tpu_b200" not in sys.path:
        sys.path.insert(0, "tilelang-tpu_b200")
    from tilelang import ops
    return ops


# ------------------------------------------------------------------------------------------------- floors
def work(case):
    op = case["op"]
    if op in ("write", "read"):
        t, h, d = case["tokens"], case["heads"], case["dim"]
        if case["fmt"] == "int4":
            rows, code, wide = 2 * t * h, d // 2 + 4 * (d // _group(case)), 2 * d           # keys and values
        else:
            rows, code, wide = t, d + 4, 2 * d
        n = rows * (code + wide) + 8 * t
        # a write case is two operators, each with what it reads and what it writes: 16 bits -> cache, cache -> 16 bits
        return {"bytes": 2 * n if op == "write" else n, "flops": rows * d * (5 if op == "write" else 2)}
    if op == "attn":
        b, h, hq, d, s_q = case["batch"], case["heads"], case["q_heads"], case["dim"], case["s_q"]
        keys = b * (case["min_len"] + case["max_len"]) / 2                                   # the mean of the lengths that are drawn
        row = 2 * (d // 2 + 4 * (d // _group(case)))
        return {"bytes": int(keys * h * row + 4 * b * s_q * hq * d + 4 * keys / case["page"] + 4 * b), "flops": int(4 * keys * s_q * hq * d)}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": 2 * (m * k + n * k + m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)), "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------------------- 64 bits
def _exact_rows_int4(codes, scale):
    c = codes.long()
    c = torch.stack((c % 16, torch.div(c, 16, rounding_mode="floor")), -1).flatten(-2).double()
    sc = scale.double().repeat_interleave(c.shape[-1] // scale.shape[-2], -2)
    return c * sc[..., 0] + sc[..., 1]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("write", "read"):
        slots, page = s["slots"], case["page"]
        if case["fmt"] == "e4m3":
            if op == "read":
                rows = s["k_cache"].view(torch.uint8).reshape(-1, case["dim"])[slots].view(torch.float8_e4m3fn)
                return rows.double() * s["k_scale"].reshape(-1)[slots].double()[:, None]
            x = s["k"].double()
            sc = (x.abs().max(1, keepdim=True).values.clamp_min(1e-4) / 448).float().double()       # the scale that is kept is fp32
            return (x / sc).to(torch.float8_e4m3fn).double() * sc

        def rows_of(w):
            if op == "read":
                at = (slots // page, slice(None), slots % page)
                return _exact_rows_int4(s[w + "_cache"][at], s[w + "_scale"][at])
            x = s[w].double().reshape(case["tokens"], case["heads"], -1, _group(case))
            lo, hi = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
            step = ((hi - lo) / 15).to(s[w].dtype).double()                                          # the step that is kept is 16-bit
            code = torch.clamp(torch.round((x - lo) / torch.where(step > 0, step, 1.0)), 0, 15) * (step > 0)
            return (code * step + lo).flatten(-2)

        return rows_of("k"), rows_of("v")
    if op == "attn":
        q, h = s["q"], case["heads"]
        per = case["q_heads"] // h
        out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        for i in range(case["batch"]):
            n = int(s["cache_seqlens"][i])
            at = torch.arange(n, device="cuda")
            pg, row = s["block_table"][i][at // case["page"]].long(), at % case["page"]
            for j in range(h):
                k = _exact_rows_int4(s["k_cache"][pg, j, row], s["k_scale"][pg, j, row])
                v = _exact_rows_int4(s["v_cache"][pg, j, row], s["v_scale"][pg, j, row])
                for t in range(case["s_q"]):
                    see = n - case["s_q"] + t + 1
                    if see > 0:
                        w = torch.softmax(q[i, t, j * per:(j + 1) * per].double() @ k[:see].t() / math.sqrt(case["dim"]), -1)
                        out[i, t, j * per:(j + 1) * per] = w @ v[:see]
        return out
    b = s["b"].double()
    x = s["a"].double() @ (b.t() if case["trans_b"] else b)
    if s["bias"] is not None:
        x += s["bias"].double()
    f = {"none": lambda z: z, "relu": torch.nn.functional.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
         "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}[case["act"]]
    x = f(x)
    return x if s["residual"] is None else x + s["residual"].double()
