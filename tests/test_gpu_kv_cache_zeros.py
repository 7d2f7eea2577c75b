"""The e4m3 bytes of zeros of both signs, and of what rounds to them."""
import pytest
import torch

import oracle.ops as O
from tilelang import ops

pytestmark = pytest.mark.gpu
BF, HF, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 576, 1024])
def test_the_sign_of_zero_is_kept(cuda_device, dtype, dim):
    x = torch.randn(5, dim, generator=torch.Generator().manual_seed(dim)).to(dtype)
    x[0, ::3], x[0, 1::3] = -0.0, 0.0
    x[1] = -0.0
    x[2, ::2] = -torch.finfo(dtype).tiny                   # far below half of the smallest e4m3 step: a zero of its sign
    x[3] = torch.finfo(dtype).tiny
    x[4, 1::2] *= 2.0 ** -12
    cache = torch.zeros(1, 5, dim, dtype=torch.uint8, device=cuda_device).view(F8)
    scale = torch.zeros(1, 5, device=cuda_device)
    ops.kv_cache_write(torch.arange(5, device=cuda_device), x.to(cuda_device), cache, scale)
    want, s = O.quantise_row_e4m3(x)
    assert (want.view(torch.uint8)[1] == 0x80).all() and (want.view(torch.uint8)[0, 1::3] == 0).all()
    assert torch.equal(cache.view(torch.uint8).cpu()[0], want.view(torch.uint8)) and torch.equal(scale.cpu()[0], s)
