"""Products of rows sorted by expert with MXFP4 expert weights, with a variable row count per expert.

The arguments are :func:`~kohakuwullm_amd.kernels.mxfp8.grouped.grouped_mxfp8_gemm`'s (``grouped.py:254-327`` of the reference);
``offsets`` stays on the device and is never read on the host.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from kohakuwullm_amd import _lib, host
from kohakuwullm_amd.kernels.mxfp4.quantize import PAIR, _check_scales, _code_format, code_rows, scale_rows
from kohakuwullm_amd.kernels.mxfp8.grouped import _check_index, _check_offsets, grouped_mxfp8_wgrad, quantize_mx_cols_grouped
from kohakuwullm_amd.kernels.mxfp8.linear import gradient_dtype
from kohakuwullm_amd.kernels.mxfp8.quantize import BLOCK_SCALE, aligned_rows, quantize_mx


def _stacked(t: torch.Tensor, alignment: int) -> torch.Tensor:
    """A stack of matrices with unit stride along the row whose matrices and rows start ``alignment`` bytes apart, or a copy that is."""
    matrix, row, unit = t.stride()
    fits = unit == 1 and row >= t.shape[2] and matrix >= 0 and row % alignment == 0 and matrix % alignment == 0 and t.data_ptr() % alignment == 0
    return t if fits else t.clone(memory_format=torch.contiguous_format)


def grouped_mxfp4_gemm(
    xq: torch.Tensor,
    x_scale: torch.Tensor,
    wq: torch.Tensor,
    w_scale: torch.Tensor,
    offsets: torch.Tensor,
    index: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
    rows: int | None = None,
    out: torch.Tensor | None = None,
    zero_rest: bool = False,
) -> torch.Tensor:
    """``out[m] = xq[index[m]] @ wq[e(m)].T`` for expert-sorted rows, the weights in MXFP4.

    Args:
        xq / x_scale: ``(R, K)`` e4m3 or ``(R, K//2)`` uint8 of two e2m1, and ``(R, K//32)`` ue8m0.
        wq / w_scale: ``(E, N, K//2)`` uint8 of two e2m1 and ``(E, N, K//32)`` ue8m0.
        offsets: ``(E+1,)`` int32 exclusive prefix sum of per-expert row counts.  Never read on the host.
        index: ``(M,)`` int32 source row per sorted position, each below ``R``, or ``None`` for the identity.
        rows: output row count ``M`` when it differs from ``xq``'s / ``index``'s; at most that.
        out: destination, or ``None`` to allocate.
        zero_rest: set rows outside every expert's range to zero.  Without it they are not written.
    """
    if rows is None and out is None:
        made = host.fp4_grouped(xq, x_scale, wq, w_scale, offsets, index, out_dtype, zero_rest)
        if made is not None:
            return made
    if wq.dim() != 3 or wq.dtype != torch.uint8:
        raise ValueError(f"wq must be uint8 (E, N, K//2), got {wq.dtype} {tuple(wq.shape)}")
    if xq.dim() != 2:
        raise ValueError(f"xq must be a matrix, got {tuple(xq.shape)}")
    num_experts, n, _ = wq.shape
    fmt, k = _code_format(xq, "xq")
    if k != wq.shape[2] * PAIR:
        raise ValueError(f"contraction mismatch: {k} columns of xq {tuple(xq.shape)}, {wq.shape[2] * PAIR} of wq {tuple(wq.shape)}")
    _check_scales(x_scale, xq, k, "x_scale")
    _check_scales(w_scale, wq, k, "w_scale")
    _check_offsets(offsets, num_experts)
    _check_index(index, "index")
    most = xq.shape[0] if index is None else index.numel()
    m = most if rows is None else rows
    if not 0 <= m <= most:
        raise ValueError(f"rows={m} must lie between 0 and the {most} source rows")
    if out is None:
        if out_dtype not in _lib.MX_DTYPE:
            raise ValueError(f"out_dtype={out_dtype} is not one of {tuple(_lib.MX_DTYPE)}")
        out = torch.empty(m, n, device=xq.device, dtype=out_dtype)
    elif out.shape != (m, n) or out.dtype not in _lib.MX_DTYPE or (n > 1 and out.stride(1) != 1) or (m > 1 and out.stride(0) < n):
        raise ValueError(f"out must be a ({m}, {n}) matrix of {tuple(_lib.MX_DTYPE)} with unit stride along its rows, got {out.dtype} "
                         f"{tuple(out.shape)} {out.stride()}")
    _lib.require_gpu(xq, "xq")
    _lib.require_same_device(xq, x_scale=x_scale, wq=wq, w_scale=w_scale, offsets=offsets, index=index, out=out)
    if m and n:
        if not xq.shape[0]:
            raise ValueError("index names rows of an empty xq")
        x, sx, w, sw = code_rows(xq), scale_rows(x_scale), _stacked(wq, 16), _stacked(w_scale.view(torch.uint8), 1)
        _lib.call(
            "mx_fp4_grouped_gemm_nt", 2.0 * m * n * k, xq,
            x.data_ptr(), sx.data_ptr(), fmt, x.shape[0], max(x.stride(0), x.shape[1]), sx.stride(0), 0 if index is None else index.data_ptr(),
            w.data_ptr(), sw.data_ptr(), w.stride(0), w.stride(1), sw.stride(0), sw.stride(1),
            offsets.data_ptr(), num_experts, out.data_ptr(), _lib.MX_DTYPE[out.dtype], max(out.stride(0), n), m, n, k, 1 if zero_rest else 0)
    return out


class _GroupedMXFP4Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, wq, ws, wqt, wst, offsets):
        xq, xs = quantize_mx(x)
        wgrad = weight is not None and ctx.needs_input_grad[1]
        xt = quantize_mx_cols_grouped(aligned_rows(x), offsets, x.shape[0], stage_major=True) if wgrad and x.shape[0] else (None, None)
        ctx.save_for_backward(*xt, wqt, wst, offsets)
        ctx.dw_dtype = None if weight is None else gradient_dtype(weight, x.dtype)
        ctx.dw_shape = None if weight is None else weight.shape
        return grouped_mxfp4_gemm(xq, xs, wq, ws, offsets, out_dtype=x.dtype, zero_rest=True)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        xtq, xts, wqt, wst, offsets = ctx.saved_tensors
        dx = dw = None
        rows = dout.shape[0]
        if ctx.needs_input_grad[0]:
            dx = grouped_mxfp4_gemm(*quantize_mx(dout), wqt, wst, offsets, out_dtype=dout.dtype, zero_rest=True)
        if ctx.needs_input_grad[1]:
            if rows:
                dt = quantize_mx_cols_grouped(aligned_rows(dout), offsets, rows, stage_major=True)
                dw = grouped_mxfp8_wgrad(*dt, xtq, xts, offsets, rows, ctx.dw_dtype)
            else:
                dw = torch.zeros(ctx.dw_shape, device=dout.device, dtype=ctx.dw_dtype)
        return dx, dw, None, None, None, None, None


def grouped_mxfp4_linear(x: torch.Tensor, operands, offsets: torch.Tensor, weight: torch.Tensor | None = None) -> torch.Tensor:
    """``out[m] = x[m] @ W[e(m)].T`` for 16-bit rows sorted by expert, with gradients: the experts' weights in MXFP4, the rows quantized
    to MXFP8 on the way.

    Args:
        x: ``(M, K)`` bf16 or fp16.
        operands: ``(q, s)`` of ``quantize_mxfp4(W)``, or ``mxfp4_operands(W)``, which the gradient of ``x`` needs.
        offsets: as in :func:`grouped_mxfp4_gemm`.  Rows outside every expert's range come out as zeros, and get a gradient of zero.
        weight: the ``(E, N, K)`` parameter that receives the weights' gradient; its values are not read.
    """
    if _lib.elsewhere(x):
        with torch.cuda.device(x.device):
            return grouped_mxfp4_linear(x, operands, offsets, weight)
    if len(operands) not in (2, 4):
        raise ValueError(f"operands are (q, s) or (q, s, qT, sT), got {len(operands)} tensors")
    wq, ws = operands[:2]
    if x.dim() != 2 or x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"x must be a 16-bit matrix, got {x.dtype} {tuple(x.shape)}")
    if wq.dim() != 3 or x.shape[1] != PAIR * wq.shape[2]:
        raise ValueError(f"x {tuple(x.shape)} does not match the codes {tuple(wq.shape)}")
    _lib.require_gpu(x, "x")
    shape = (wq.shape[0], wq.shape[1], x.shape[1])
    if weight is not None and weight.shape != shape:
        raise ValueError(f"weight {tuple(weight.shape)} does not match the quantized one {shape}")
    recorded = _lib.recorded(x, weight)
    if not recorded and not _lib.forward_mode():
        return grouped_mxfp4_gemm(*quantize_mx(x), wq, ws, offsets, out_dtype=x.dtype, zero_rest=True)
    if recorded and shape[1] % BLOCK_SCALE:
        raise ValueError(f"gradients need a multiple of {BLOCK_SCALE} output columns, got {shape[1]}")
    wqt, wst = operands[2:] if len(operands) == 4 else (None, None)
    if recorded and x.requires_grad and wqt is None:
        raise ValueError("the gradient of x needs the weights quantized along their output axis too: pass mxfp4_operands(weight)")
    return _GroupedMXFP4Linear.apply(x, weight, wq, ws, wqt, wst, offsets)
