"""Offsets that are no prefix sum: nothing outside the operands is read or written, however many tiles they seem to ask for."""

import pytest
import torch

from tests.fp4_checks import assert_product, values64

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("experts,rows,n,k", [
    (1024, 1 << 22, 384, 512),  # the stream: 2^24 row tiles by three, past what its division by a reciprocal takes
    (64, 40000, 384, 512),
    (64, 40000, 384, 96),       # tiles with scales by the byte
    (2000, 30000, 100, 96),     # more experts than tables hold
    (8, 40, 100, 512),          # a few rows
])
def test_offsets_that_go_up_and_down(experts, rows, n, k):
    """Every other expert claims all rows; all have one weight, so every row that is written is the product with it."""
    from kohakuwullm_amd.kernels.mxfp4 import grouped_mxfp4_gemm, quantize_mxfp4

    g = torch.Generator(device=DEV).manual_seed(rows)
    few = torch.randint(0, 120, (1 << 12, k), generator=g, device=DEV, dtype=torch.uint8)  # finite codes of e4m3, above zero
    xq = few[torch.arange(rows, device=DEV) % len(few)].view(torch.float8_e4m3fn)
    xs = torch.randint(120, 128, (rows, k // 32), generator=g, device=DEV, dtype=torch.uint8)
    wq, ws = quantize_mxfp4(torch.randn(n, k, generator=g, device=DEV, dtype=torch.bfloat16) * 0.02)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=DEV)
    offsets[1::2] = rows
    room = torch.full((rows + 2, n + 64), float("nan"), dtype=torch.bfloat16, device=DEV)
    out = room[1:-1, 32:-32]
    got = grouped_mxfp4_gemm(xq, xs, wq.expand(experts, n, k // 2), ws.expand(experts, n, k // 32), offsets, out=out)
    torch.cuda.synchronize()
    assert got is out
    for edge in (room[0], room[-1], room[:, :32], room[:, -32:]):
        assert edge.isnan().all()
    assert not out.isnan().any()
    some = torch.cat([torch.arange(0, rows, max(1, rows // 300)), torch.tensor([rows - 1])])
    assert_product(out[some.to(DEV)], values64(xq[some.to(DEV)], xs[some.to(DEV)]), values64(wq, ws), 8, f"{experts} experts")
