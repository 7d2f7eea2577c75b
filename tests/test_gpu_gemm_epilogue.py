"""Matrix product with bias, activation and residual in its epilogue, against the definition in 64 bits."""
import pytest
import torch

import oracle.ops as O
from tilelang import ops

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]


def make(m, n, k, dtype, trans, seed):
    g = torch.Generator().manual_seed(seed)
    a = torch.randn(m, k, generator=g).to(dtype)
    b = (torch.randn((n, k) if trans else (k, n), generator=g) * 1.5 * k ** -0.5).to(dtype)
    return a, b, torch.randn(n, generator=g).to(dtype), torch.randn(m, n, generator=g).to(dtype)


def check(dev, m, n, k, dtype, trans, act, bias, residual, out=None, seed=0, rows=None):
    a, b, bi, re = make(m, n, k, dtype, trans, seed + m + n + k)
    bi, re = bi if bias else None, re if residual else None
    c = torch.full((m, n), float("nan"), dtype=out or dtype, device=dev)
    assert ops.gemm_epilogue(a.to(dev), b.to(dev), c, bias=None if bi is None else bi.to(dev), activation=act,
                             residual=None if re is None else re.to(dev), transpose_b=trans) == 0
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    sel = slice(None) if rows is None else rows
    ref = O.gemm_epilogue(a[sel], b, bi, act, None if re is None else re[sel], trans)
    mag = a[sel].double().abs() @ (b.double().abs().t() if trans else b.double().abs())
    # fp32 sums of k products (2^-24 of the magnitudes each, sqrt(k) of them and a factor 8 for order and truncation); no
    # activation is steeper than 1.13; expf, erff and tanhf are a few ulp of values below the magnitude of x; one rounding at the end
    pre = O.gemm_epilogue(a[sel], b, bi, None, None, trans).abs()
    tol = 1.13 * (8 * k ** 0.5 * 2.0 ** -24) * mag + 2.0 ** -20 * pre + torch.finfo(c.dtype).eps / 2 * (ref.abs() + 2.0 ** -20)
    if dtype == HF and c.dtype == HF:
        tol = tol + 2.0 ** -25                                       # subnormal results
    err = (c.cpu()[sel].double() - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())
    return c


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("dtype,trans,m,n,k", [(BF, True, 16, 256, 512), (HF, False, 130, 264, 200), (BF, False, 5, 136, 64), (F32, True, 9, 33, 21)])
def test_epilogues(cuda_device, dtype, trans, m, n, k, act, bias, residual):
    check(cuda_device, m, n, k, dtype, trans, act, bias, residual)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("trans", [True, False])
@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 100, 128, 129, 200, 256, 257, 300])
def test_few_rows(cuda_device, dtype, trans, m):
    check(cuda_device, m, 328, 520, dtype, trans, "silu", True, True)


@pytest.mark.parametrize("trans,m,n,k", [(True, 3, 1, 8), (True, 17, 129, 8), (True, 64, 1000, 4096), (True, 1, 4096, 4096), (False, 1, 4096, 1032),
                                         (True, 48, 6144, 1024), (False, 33, 8, 64), (True, 31, 127, 14336), (False, 60, 2056, 1000),
                                         (True, 500, 1001, 264), (True, 1024, 2048, 512), (False, 2049, 2056, 136), (True, 2500, 4100, 72)])
def test_odd_sizes(cuda_device, trans, m, n, k):
    check(cuda_device, m, n, k, BF, trans, "gelu", True, True)
    check(cuda_device, m, n, k, BF, trans, None, False, False, out=F32)


@pytest.mark.parametrize("dtype,trans,m,n,k", [(BF, True, 33, 47, 13), (HF, False, 17, 9, 5), (BF, False, 70, 129, 40), (F32, False, 1, 1, 1),
                                               (F32, True, 130, 70, 200)])
def test_sizes_without_tensor_maps(cuda_device, dtype, trans, m, n, k):
    check(cuda_device, m, n, k, dtype, trans, "gelu_tanh", True, True)
    check(cuda_device, m, n, k, dtype, trans, "relu", True, False, out=F32)


def test_full_sizes_on_sampled_rows(cuda_device):
    check(cuda_device, 2048, 14336, 4096, BF, False, "gelu", True, False, rows=[0, 1, 127, 128, 255, 256, 1000, 2047])
    check(cuda_device, 61, 4096, 14336, BF, True, None, False, True)


@pytest.mark.parametrize("m,n,k", [(4, 512, 1024), (61, 328, 520), (300, 520, 264)])
def test_residual_in_place(cuda_device, m, n, k):
    """c += a b^T, m of every kernel: the residual is the output's own buffer."""
    a, b, bi, re = make(m, n, k, BF, True, 5)
    dev = cuda_device
    apart = torch.empty(m, n, dtype=BF, device=dev)
    ops.gemm_epilogue(a.to(dev), b.to(dev), apart, residual=re.to(dev), transpose_b=True)
    c = re.to(dev)
    ops.gemm_epilogue(a.to(dev), b.to(dev), c, residual=c, transpose_b=True)
    assert torch.equal(c.view(torch.int16), apart.view(torch.int16))


@pytest.mark.parametrize("m", [3, 64, 300])
def test_same_bits_every_time_and_neighbours_untouched(cuda_device, m):
    dev, n, k = cuda_device, 1001, 2048
    a, b, bi, re = (t.to(dev) for t in make(m, n, k, BF, True, 6))
    pad = torch.full((m + 2, n), 5.0, dtype=BF, device=dev)
    first = None
    for _ in range(5):
        ops.gemm_epilogue(a, b, pad[1:m + 1], bias=bi, activation="gelu", residual=re, transpose_b=True)
        first = pad.clone() if first is None else first
        assert torch.equal(pad.view(torch.int16), first.view(torch.int16))
    assert (pad[0] == 5).all() and (pad[-1] == 5).all()


@pytest.mark.parametrize("m", [2, 40, 300])
def test_non_finite_inputs(cuda_device, m):
    """NaN and infinity reach exactly the rows and columns they belong to; relu keeps NaN."""
    dev = cuda_device
    a, b, bi, _ = make(m, 264, 128, BF, True, 7)
    a[1, 3] = float("nan")
    bi[5] = float("inf")
    for act in (None, "relu", "silu", "gelu", "gelu_tanh"):
        c = torch.empty(m, 264, dtype=BF, device=dev)
        ops.gemm_epilogue(a.to(dev), b.to(dev), c, bias=bi.to(dev), activation=act, transpose_b=True)
        c = c.cpu()
        assert c[1].isnan().all()
        keep = torch.arange(m) != 1
        assert (c[keep][:, 5] == float("inf")).all()
        assert torch.isfinite(c[keep][:, torch.arange(264) != 5]).all()


def test_two_streams_and_a_graph(cuda_device):
    dev = cuda_device
    sets = [tuple(t.to(dev) for t in make(12, 4096, 2048, BF, True, s)) for s in (1, 2)]
    refs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for a, b, bi, re in sets:
        c = torch.empty(12, 4096, dtype=BF, device=dev)
        ops.gemm_epilogue(a, b, c, bias=bi, residual=re, transpose_b=True)
        refs.append(c)
        outs.append(torch.zeros_like(c))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        a, b, bi, re = sets[0]
        ops.gemm_epilogue(a, b, outs[0], bias=bi, residual=re, transpose_b=True)
    for _ in range(10):
        outs[0].zero_()
        outs[1].zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            graph.replay()
        with torch.cuda.stream(streams[1]):
            a, b, bi, re = sets[1]
            ops.gemm_epilogue(a, b, outs[1], bias=bi, residual=re, transpose_b=True)
        torch.cuda.synchronize()
        assert all(torch.equal(o.view(torch.int16), r.view(torch.int16)) for o, r in zip(outs, refs))
