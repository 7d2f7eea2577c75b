"""Sequences that many teams share, against bounds that no missing part of a sequence passes (the CPU test shows it)."""
import pytest
import torch

from attn_int4_bounds import excess, problem, reference, run

BF, HF = torch.bfloat16, torch.float16
CASES = [([5000] + [17] * 30, 1, 128, 128), ([5000] + [17] * 30, 3, 128, 128), ([2999, 1, 0, 1500], 3, 128, 64), ([3000], 1, 64, 32)]


@pytest.mark.parametrize("lens,s_q,dim,group", CASES)
def test_the_bounds_notice_a_unit_or_a_share_left_out(lens, s_q, dim, group):
    w = problem(lens, s_q, 8, 2, dim, group, 64, BF, len(lens))
    ref, tol, rms = reference(w)
    element, norm = excess(ref.to(BF), ref, tol, rms)
    assert element <= 1 and norm <= 1
    for leave_out in (lambda i, at: (i == 0) & (at // 128 == 5),                          # a unit
                      lambda i, at: (i == 0) & (at // 128 >= at.numel() // 128 - 1),      # the last, in part
                      lambda i, at: (i == 0) & (at // 128 % 13 == 12),                    # a team in thirteen
                      lambda i, at: (i == 0) & (at // 16 == 77)):                         # one warp's tile
        out = reference(w, leave_out=leave_out)[0].to(BF)
        assert max(excess(out, ref, tol, rms)) > 2


@pytest.mark.gpu
@pytest.mark.parametrize("lens,s_q,dim,group", CASES)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_long_and_ragged(cuda_device, lens, s_q, dim, group, dtype):
    w = problem(lens, s_q, 8, 2, dim, group, 64, dtype, len(lens))
    element, norm = excess(run(w, cuda_device), *reference(w))
    assert element <= 1 and norm <= 1, (element, norm)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,group", [(64, 64), (128, 128), (256, 64)])
@pytest.mark.parametrize("units", [1, 2, 11, 12, 13, 24, 25, 36, 37, 100, 157])
@pytest.mark.parametrize("before", [0, 3])
def test_every_number_of_teams_to_a_segment(cuda_device, dim, group, units, before):
    """Up to as many units as there are teams, each team has one: `units` teams share the segment (two kv heads), added up in
    groups of twelve; the shorter sequences move the segment's first team."""
    lens = [100] * before + [128 * units - 5]
    w = problem(lens, 1, 8, 2, dim, group, 32, BF, units + before)
    element, norm = excess(run(w, cuda_device), *reference(w))
    assert element <= 1 and norm <= 1, (element, norm)


@pytest.mark.gpu
def test_segments_that_begin_and_end_inside_teams(cuda_device):
    """More units than teams: several units a team, segments of 40 units that begin anywhere in them."""
    w = problem([5100, 4000, 70, 5119, 2000] * 3, 1, 8, 8, 64, 64, 64, BF, 3)
    element, norm = excess(run(w, cuda_device), *reference(w))
    assert element <= 1 and norm <= 1, (element, norm)
