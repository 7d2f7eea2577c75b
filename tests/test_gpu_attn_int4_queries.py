"""Queries of any finite size."""
import pytest
import torch

from attn_int4_bounds import excess, problem, reference, run

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("dim,group", [(64, 32), (128, 128), (256, 64)])
@pytest.mark.parametrize("h_q", [4, 16])
def test_queries_up_to_the_largest_number(cuda_device, dim, group, h_q):
    """Keys small enough that the scores are ordinary ones; beside them an ordinary query and one of zeros, whose scores vanish."""
    w = problem([300, 20], 1, h_q, 1, dim, group, 16, BF, dim + h_q)
    w["k_scale"] = (w["k_scale"].float() * 2.0 ** -118).to(BF)
    size = torch.ones(h_q)
    size[0], size[1], size[2], size[3] = 2.0 ** 125, 2.0 ** 116, 2.0 ** 119, 0
    w["q"] = (w["q"].float().clamp(-3.9, 3.9) * size[None, None, :, None]).to(BF)
    w["q"][1, 0, 0] = torch.finfo(BF).max * torch.sign(w["q"][1, 0, 0].float())
    assert torch.isfinite(w["q"]).all()
    element, norm = excess(run(w, cuda_device, 2.0 ** -4), *reference(w, 2.0 ** -4))
    assert element <= 1 and norm <= 1, (element, norm)


def test_large_queries_with_large_keys(cuda_device):
    """Scores near 2^122 that decide for one key, and a query of the other end of the range beside them."""
    w = problem([90], 1, 4, 1, 64, 64, 16, BF, 8)
    w["q"][0, 0, 1] = (w["q"][0, 0, 1].float() * 2.0 ** 118).to(BF)
    w["q"][0, 0, 2] = (w["q"][0, 0, 2].float() * 2.0 ** -110).to(BF)
    element, norm = excess(run(w, cuda_device), *reference(w))
    assert element <= 1 and norm <= 1, (element, norm)
