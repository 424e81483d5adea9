"""Products with MXFP4 weights whose last round of tiles is cut along K, for every kernel that cuts and every way to fetch scales: that
they are cut shows in the workspace, whose fp32 tiles the slices write."""

import pytest
import torch

from tests.fp4_checks import assert_product, values64

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _rand(*shape, seed, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(torch.bfloat16)


def _some(rows):
    """Rows on both sides of tile borders, and some of every tile."""
    picked = {0, rows - 1, *range(0, rows, max(1, rows // 200))}
    picked |= {r for border in range(128, rows, max(128, rows // 16 // 128 * 128)) for r in (border - 1, border)}
    return torch.tensor(sorted(picked))


CUT = [
    (8, 300, 1536, 8192), (4, 300, 1536, 8192), (8, 130, 136, 16896), (4, 130, 136, 16896),  # the stream; the last two: slices of two lengths
    (8, 300, 1537, 8192), (4, 300, 1537, 8192), (8, 130, 130, 16384), (4, 130, 130, 16384),  # small tiles, scales by the 16
    (8, 300, 1000, 8320), (4, 300, 1000, 8320),                                              # ... by the 4
    (8, 300, 1000, 8224), (4, 300, 1000, 8224), (8, 124, 1936, 2784),                        # ... by the byte, K ends inside a stage
    (8, 20736, 4096, 8192), (4, 20736, 4096, 8192),                                          # large tiles, by the 16
    (8, 4352, 4360, 12416), (4, 4352, 4360, 12416),                                          # ... by the 4
    (8, 4352, 4360, 12320), (4, 4352, 4360, 12320),                                          # ... by the byte
]


@pytest.mark.parametrize("bits,m,n,k", CUT)
def test_cut_along_k(bits, m, n, k):
    from kohakuwullm_amd import _lib
    from kohakuwullm_amd.kernels.mxfp4 import mxfp4_matmul_pq, quantize_mxfp4
    from kohakuwullm_amd.kernels.mxfp8 import quantize_mx

    # blocks of K of different sizes: a slice's scales in another's place do not go unseen
    size = torch.exp2((torch.arange(k // 32, device=DEV) * 5 % 7 - 3).float()).repeat_interleave(32)
    x = (_rand(m, k, seed=m + n).float() * size).to(torch.bfloat16)
    aq, sa = quantize_mx(x) if bits == 8 else quantize_mxfp4(x)
    bq, sb = quantize_mxfp4(_rand(n, k, seed=k, std=0.02))
    fmt = _lib.MX_E4M3 if bits == 8 else _lib.MX_E2M1
    rows = _some(m)
    a, b = values64(aq.cpu()[rows], sa.cpu()[rows]), values64(bq, sb)
    space = _lib.gemm_workspace(aq)
    for dtype in (torch.bfloat16, torch.float32):
        own = torch.full((space.numel() // 4,), float("nan"), device=DEV)
        got, whole = (torch.full((m, n), float("nan"), device=DEV, dtype=dtype) for _ in range(2))
        for out, at, room in ((got, own.data_ptr(), space.numel()), (whole, None, 0)):
            _lib.call("mx_fp4_gemm_nt", 0.0, aq, aq.data_ptr(), sa.data_ptr(), fmt, bq.data_ptr(), sb.data_ptr(), out.data_ptr(), _lib.MX_DTYPE[dtype],
                      m, n, k, aq.shape[1], k // 32, k // 2, k // 32, n, at, room)
        written = int((~own.isnan()).sum())
        assert written and written % (128 * 128) == 0, "no tile was cut along K"
        for out, what in ((got, "cut"), (whole, "whole")):
            assert not out.isnan().any()
            assert_product(out[rows.to(DEV)], a, b, bits, f"{m}x{n}x{k}, A in {bits} bits, {dtype}, {what}")
        assert torch.equal(got, mxfp4_matmul_pq(aq, sa, bq, sb, dtype))
