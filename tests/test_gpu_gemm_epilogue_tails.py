"""Activations far below zero, where the value is a small fraction of its argument."""
import pytest
import torch

from tilelang import ops

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def value(x, act):
    """In 64 bits without a difference of near numbers."""
    if act == "gelu":
        return 0.5 * x * torch.special.erfc(-x * 0.5 ** 0.5)
    z = 2 * (2 / torch.pi) ** 0.5 * (x + 0.044715 * x ** 3) if act == "gelu_tanh" else x
    return x * torch.exp(-torch.nn.functional.softplus(-z))


def slope(x, act):
    """By how much a relative error of 2^-24 of the argument of erfc or exp grows in their values."""
    if act == "gelu":
        return x * x + 1                                      # erfc(t) ~ exp(-t^2), t^2 = x^2 / 2
    return (2 * (2 / torch.pi) ** 0.5 * (x + 0.044715 * x ** 3).abs() if act == "gelu_tanh" else x.abs()) + 1


@pytest.mark.parametrize("act,low", [("gelu", -13.0), ("gelu_tanh", -9.9), ("silu", -100.0)])
@pytest.mark.parametrize("dtype,out", [(BF, BF), (BF, F32), (HF, HF), (HF, F32), (F32, F32)])
@pytest.mark.parametrize("m", [5, 300, 1100])
def test_values_keep_their_precision(cuda_device, act, low, dtype, out, m):
    """A product with the unit matrix, so that the activation's argument is exact; every kernel by its rows."""
    n = 264
    x = torch.linspace(low, 3.0, m * n).reshape(m, n).to(dtype)
    c = torch.empty(m, n, dtype=out, device=cuda_device)
    ops.gemm_epilogue(x.to(cuda_device), torch.eye(n, dtype=dtype, device=cuda_device), c, activation=act, transpose_b=True)
    xd = x.double()
    ref = value(xd, act)
    # six roundings of the argument and of the value (constants, products, the function's own few units); exp and the products of
    # the smallest values are subnormal in fp32: half their step times |x|
    tol = (torch.finfo(out).eps / 2 + 6 * 2.0 ** -24 * slope(xd, act)) * ref.abs() + (xd.abs() + 1) * 2.0 ** -149
    # below a 16-bit type's normal range a rounding is off by half its smallest step: 2^-24 for fp16 (normal from 2^-14, 11 bits),
    # 2^-133 for bf16 (normal from 2^-126, 8 bits), whatever the value
    tol = tol + {HF: 2.0 ** -25, BF: 2.0 ** -134, F32: 0.0}[out]
    err = (c.cpu().double() - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_the_ends(cuda_device, act):
    """Arguments whose exponential over- or underflows: the argument itself, or a zero, and never NaN."""
    x = torch.tensor([-3e38, -1e20, -1000.0, -120.0, -0.0, 0.0, 120.0, 1e20, 3e38])
    a = torch.zeros(9, 8)
    a[:, 0] = x
    b = torch.zeros(1, 8)
    b[0, 0] = 1
    c = torch.empty(9, 1, device=cuda_device)
    ops.gemm_epilogue(a.to(cuda_device), b.to(cuda_device), c, activation=act, transpose_b=True)
    assert torch.equal(c.cpu()[:, 0], torch.where(x > 0, x, torch.zeros(())))
