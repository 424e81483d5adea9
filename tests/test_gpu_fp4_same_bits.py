"""A 4-bit layer's output is the same with gradients and without, whichever way its rows are quantized."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _uneven(rows, cols, g):
    """Normal values whose blocks of 32 columns lie up to 2^12 apart: what an fp32 sum of them drops depends on its order."""
    size = torch.exp2(torch.randint(-6, 7, (rows, cols // 32), generator=g, device=DEV).float())
    return torch.randn(rows, cols, generator=g, device=DEV) * size.repeat_interleave(32, -1) * 0.05


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", [
    (32, 1536, 65536), (17, 2048, 65536), (16, 4096, 131072), (9, 8192, 131072), (4, 4096, 131072), (1, 1536, 65536),  # a vocabulary's columns
    (32, 2048, 4096), (32, 2048, 4112), (32, 2080, 4096), (17, 1536, 8192), (33, 512, 512),  # where rows stop being quantized inside the product
    (16, 8192, 16384), (16, 8192, 16400), (16, 8224, 4096), (5, 1440, 16400),
    (2, 1728, 5024), (16, 96, 264), (32, 160, 1000), (1, 32, 8),
])
def test_linear(m, k, n, dtype):
    from kohakuwullm_amd.kernels.mxfp4 import mxfp4_linear, mxfp4_matmul_pq, quantize_mxfp4
    from kohakuwullm_amd.kernels.mxfp8 import quantize_mx

    g = torch.Generator(device=DEV).manual_seed(m + k + n)
    x = _uneven(m, k, g).to(dtype)
    pair = quantize_mxfp4(_uneven(n, k, g).to(dtype))
    weight = torch.zeros(n, k, device=DEV, dtype=dtype, requires_grad=True)
    with torch.no_grad():
        served = mxfp4_linear(x, pair)
        masters = mxfp4_linear(x.float(), pair) if dtype == torch.bfloat16 else None  # fp32 computes in fp32: another output type
    trained = mxfp4_linear(x, pair, weight)
    assert trained.requires_grad and torch.equal(served, trained)
    assert torch.equal(served, mxfp4_matmul_pq(*quantize_mx(x), *pair, dtype))
    if masters is not None:
        assert torch.equal(masters.to(dtype), mxfp4_linear(x.float(), pair, weight.detach().float().requires_grad_()).to(dtype))


@pytest.mark.parametrize("m,k,n", [(32, 1536, 65536), (16, 4096, 32768), (8, 1440, 1000)])
def test_rounded_masters(m, k, n):
    """Rows in fp32 under autocast are rounded to its type first, on either way."""
    from kohakuwullm_amd.kernels.mxfp4 import mxfp4_linear, quantize_mxfp4

    g = torch.Generator(device=DEV).manual_seed(n)
    x = _uneven(m, k, g)
    pair = quantize_mxfp4(_uneven(n, k, g))
    weight = torch.zeros(n, k, device=DEV, requires_grad=True)
    with torch.autocast("cuda", torch.bfloat16):
        trained = mxfp4_linear(x, pair, weight)
        with torch.no_grad():
            served = mxfp4_linear(x, pair)
    assert served.dtype == torch.bfloat16 and torch.equal(served, trained) and torch.equal(served, mxfp4_linear(x.bfloat16(), pair))
