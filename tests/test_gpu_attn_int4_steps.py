"""Steps of values that are infinite, or far above the others: they reach the outputs that see them, in their group of columns, and
leave all others as exact as they are without them."""
import pytest
import torch

from attn_int4_bounds import excess, problem, reference, rows_of, run

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
SHAPES = [(64, 32, 2), (64, 64, 1), (128, 32, 2), (128, 64, 2), (128, 128, 2), (256, 32, 2), (256, 128, 1)]      # dim, group, kv heads


def check(w, dev, scale=None):
    out = run(w, dev, scale)
    element, norm = excess(out, *reference(w, scale))
    assert element <= 1 and norm <= 1, (element, norm)
    return out


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim,group,h_kv", SHAPES)
def test_an_infinite_step_reaches_its_group_alone(cuda_device, dtype, dim, group, h_kv):
    """As kv_cache_write stores a group with an infinity: an infinite step, codes 0, and the group's minimum."""
    w = problem([300, 90], 1, 4 * h_kv, h_kv, dim, group, 16, dtype, dim + group)
    pg, row = rows_of(w, 0, 19)
    w["v_scale"][pg, 0, row, 0] = torch.tensor([float("inf"), -1.0]).to(dtype)
    w["v_cache"][pg, 0, row, :group // 2] = 0
    out = run(w, cuda_device)
    ref, tol, rms = reference(w)
    assert ref[0, 0, :4, :group].isnan().all() and torch.isfinite(ref[0, 0, :4, group:]).all() and torch.isfinite(ref[1]).all()
    element, norm = excess(out, ref, tol, rms)
    assert element <= 1 and norm <= 1, (element, norm)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("h_q", [2, 4, 16])
@pytest.mark.parametrize("dim,group,h_kv", SHAPES[:5])
def test_an_infinite_step_that_earlier_queries_do_not_see(cuda_device, dtype, h_q, dim, group, h_kv):
    w = problem([260, 37, 4], 4, h_q, 1, dim, group, 16, dtype, h_q + dim)
    for i, n in enumerate((260, 37, 4)):
        pg, row = rows_of(w, i, n - 1)
        w["v_scale"][pg, 0, row, :, 0] = float("inf")
        w["v_cache"][pg, 0, row] = 0
    out = run(w, cuda_device)
    ref, tol, rms = reference(w)
    assert ref[:, 3].isnan().all() and torch.isfinite(ref[:, :3]).all()
    element, norm = excess(out, ref, tol, rms)
    assert element <= 1 and norm <= 1, (element, norm)


@pytest.mark.parametrize("dim,group,h_kv", SHAPES)
def test_groups_whose_steps_are_far_apart(cuda_device, dim, group, h_kv):
    w = problem([300, 90], 1, 4 * h_kv, h_kv, dim, group, 16, BF, dim + group)
    groups = dim // group
    for g in range(groups):
        w["v_scale"][:, :, :, g] = (w["v_scale"][:, :, :, g].float() * 2.0 ** (40 - 23 * g)).to(BF)
    check(w, cuda_device)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim,group,h_kv", SHAPES)
def test_large_values_that_are_not_seen_or_hardly_weigh(cuda_device, dtype, dim, group, h_kv):
    """A value far above the others: hidden from the earlier query tokens, or with next to no weight for some queries and
    all of it for others, before, between and after the ordinary tokens."""
    n = 400
    small = 1.0 if dtype is BF else 2.0 ** -12
    for where in ([n - 1], [n - 2, n - 3], [0], [150, 151], [5, 6, 7, 390], list(range(128, 256))):
        up = 2.0 ** 25 if dtype is HF else 2.0 ** 60 if where[0] > n - 4 else 2.0 ** 30
        w = problem([n], 4, 4, 1, dim, group, 16, dtype, len(where) + where[0])
        w["v_scale"] = (w["v_scale"].float() * small).to(dtype)
        pg, row = rows_of(w, 0, where)
        w["v_scale"][pg, 0, row] = (w["v_scale"][pg, 0, row].float() * up).to(dtype)
        # the keys of those tokens: q of head 0 and 1 against them gives about -25 and 25 (head 0: a weight of 2^-70 or so)
        k = torch.ones(dim)
        w["k_cache"][pg, 0, row] = 0
        w["k_scale"][pg, 0, row] = torch.tensor([0.0, 1.0]).to(dtype)
        w["q"][:, :, 0] = (w["q"][:, :, 0].float() * 0.2 - 3.0 * 8 / dim ** 0.5).to(dtype)
        w["q"][:, :, 1] = (w["q"][:, :, 1].float() * 0.2 + 3.0 * 8 / dim ** 0.5).to(dtype)
        check(w, cuda_device)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_the_lowest_value_of_the_type(cuda_device, dtype):
    """Rows of the type's lowest value behind what a query sees, as a padded batch may leave them, written by kv_cache_write."""
    from tilelang import ops
    dev = cuda_device
    w = problem([200, 21], 3, 8, 2, 128, 64, 16, dtype, 5)
    t = {k: v.to(dev) for k, v in w.items()}
    low = torch.randn(4, 2, 128, generator=torch.Generator().manual_seed(3)).to(dtype)
    low[:, :, ::3] = torch.finfo(dtype).min
    slots = torch.tensor([int(pg) * 16 + int(row) for i, n in ((0, 200), (1, 21)) for pg, row in [rows_of(w, i, n - 2), rows_of(w, i, n - 1)]])
    ops.kv_cache_write(slots.to(dev), low.abs().clamp(max=1).to(dev), t["k_cache"], t["k_scale"], low.to(dev), t["v_cache"], t["v_scale"])
    host = {k: v.cpu() for k, v in t.items()}
    out = run(host, dev)
    ref, tol, rms = reference(host)
    element, norm = excess(out[:, :1], ref[:, :1], tol[:, :1], rms[:, :1])      # the first query token sees neither of the two
    assert element <= 1 and norm <= 1, (element, norm)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_steps_that_rise_and_fall(cuda_device, dtype):
    """From token to token 2^-20 to 2^4 in both directions, and zero steps between; the small ones weigh more."""
    w = problem([700, 65], 1, 8, 2, 128, 64, 16, dtype, 9)
    g = torch.Generator().manual_seed(1)
    low, high = (-24, 8) if dtype is BF else (-8, 4)
    e = torch.exp2(torch.randint(low, high, w["v_scale"].shape[:3], generator=g).float())
    e[torch.rand(e.shape, generator=g) < 0.1] = 0
    w["v_scale"] = (w["v_scale"].float() * e[..., None, None]).to(dtype)
    # a key along q where the step is small
    w["k_scale"] = (w["k_scale"].float() * torch.where(e > 2.0 ** (low + 4), 0.1, 2.0)[..., None, None]).to(dtype)
    check(w, cuda_device)
