"""A linear layer whose weight is held in MXFP4: activations in MXFP8, FPROP and DGRAD against 4-bit codes, WGRAD in MXFP8.

The surface is :class:`~kohakuwullm_amd.kernels.mxfp8.linear.MXFP8Linear`'s (``src/kohakuwullm/kernels/mxfp8/linear.py:77-126`` of the
reference), so ``swap_mxfp8(model, linear_cls=MXFP4Linear)`` and ``refresh_mxfp8_weights`` take it.  Gradients are those of the
product with the quantized weight (straight through both quantizers): ``dX = Q8(dY) W4``, with the weight quantized along its
output axis, ``dW = Q8(dY)^T Q8(X)`` with blocks of 32 tokens.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from kohakuwullm_amd import _lib, host
from kohakuwullm_amd.kernels.mxfp4.quantize import PAIR, check_source, mxfp4_matmul_pq, quantize_mxfp4, quantize_mxfp4_cols
from kohakuwullm_amd.kernels.mxfp8.linear import compute_dtype, gradient_dtype
from kohakuwullm_amd.kernels.mxfp8.quantize import BLOCK_SCALE, activation_matrix, mxfp8_matmul_pq, quantize_mx, quantize_tokens


def mxfp4_operands(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Both quantized copies ``(q, s, qT, sT)`` of a weight ``(out, in)``, or of a stack ``(E, out, in)``.

    ``(q, s)``, blocks along ``in``, is what the forward multiplies with, ``(qT, sT)``, blocks along ``out`` (padded with zeros to a
    multiple of 32), what the gradient of the input does.
    """
    check_source(weight, "weight", (2, 3))
    with torch.no_grad():
        extra = -weight.shape[-2] % BLOCK_SCALE
        return *quantize_mxfp4(weight), *quantize_mxfp4_cols(F.pad(weight, (0, 0, 0, extra)) if extra else weight)


def quantized_activation(x2d: torch.Tensor, compute: torch.dtype, token_axis: bool):
    """``(q, s, qT, sT)`` of an activation matrix as :func:`activation_matrix` returns it; without ``token_axis`` the last two are None."""
    if x2d.shape[0] and (token_axis or x2d.dtype != compute):
        return quantize_tokens(x2d, compute, token_axis=token_axis)
    return *quantize_mx(x2d.to(compute)), None, None


class _MXFP4Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, wq, ws, wqt, wst):
        compute = compute_dtype(x)
        wgrad = weight is not None and ctx.needs_input_grad[1]
        made = host.fp4_linear(x, compute, wq, ws, wgrad)
        if made is None:
            xq, xs, xtq, xts = quantized_activation(activation_matrix(x, compute), compute, wgrad)
            out = mxfp4_matmul_pq(xq, xs, wq, ws, compute).reshape(*x.shape[:-1], wq.shape[0])
        else:
            out, xtq, xts = made
        ctx.save_for_backward(xtq, xts, wqt, wst)
        ctx.out_features, ctx.x_shape, ctx.x_dtype, ctx.compute = wq.shape[0], x.shape, x.dtype, compute
        ctx.dw_dtype = None if weight is None else gradient_dtype(weight, compute)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        xtq, xts, wqt, wst = ctx.saved_tensors
        n, compute, inp = ctx.out_features, ctx.compute, ctx.x_shape[-1]
        need_dx, need_dw = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        made = host.fp4_linear_backward(dout, compute, xtq, xts, wqt, wst, need_dx, need_dw, ctx.x_dtype, ctx.dw_dtype or compute)
        if made is not None:
            return *made, None, None, None, None
        d2d = dout.reshape(-1, n)
        cols = n + -n % BLOCK_SCALE
        dx = dw = None
        if need_dw and xtq is None:  # no tokens
            dw = torch.zeros(n, inp, device=dout.device, dtype=ctx.dw_dtype)
        if not d2d.shape[0]:
            return (dout.new_zeros(ctx.x_shape, dtype=ctx.x_dtype) if need_dx else None), dw, None, None, None, None
        # rows of a width the quantizer cannot fetch 16 bytes at a time are padded here
        d2d = activation_matrix(F.pad(d2d, (0, cols - n)) if n % 8 else d2d, compute)
        if need_dw:
            dq, ds, dtq, dts = quantize_tokens(d2d, compute, cols)
            dw = mxfp8_matmul_pq(dtq, dts, xtq, xts, ctx.dw_dtype)[:n]
        elif need_dx:
            d2d = d2d.to(compute)
            dq, ds = quantize_mx(F.pad(d2d, (0, cols - d2d.shape[1])) if cols != d2d.shape[1] else d2d)
        if need_dx:
            dx = mxfp4_matmul_pq(dq, ds, wqt, wst, ctx.x_dtype).reshape(ctx.x_shape)
        return dx, dw, None, None, None, None


def mxfp4_linear(x: torch.Tensor, operands, weight: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ W.T`` with ``W`` in MXFP4 and ``x`` quantized to MXFP8 on the way, in the type ``nn.Linear`` would compute in.

    Args:
        x: ``(.., in)``.
        operands: ``(q, s)`` of :func:`quantize_mxfp4`, or the four tensors of :func:`mxfp4_operands`, which the gradient of ``x`` needs.
        weight: the ``(out, in)`` parameter that receives the weight's gradient; its values are not read.  ``None``: no such gradient.
    """
    if _lib.elsewhere(x):
        with torch.cuda.device(x.device):
            return mxfp4_linear(x, operands, weight)
    if len(operands) not in (2, 4):
        raise ValueError(f"operands are (q, s) or (q, s, qT, sT), got {len(operands)} tensors")
    wq, ws = operands[:2]
    recorded = _lib.recorded(x, weight)
    through = recorded or _lib.forward_mode()
    if not through and (weight is None or weight.shape == (wq.shape[0], x.shape[-1])):
        made = host.fp4_linear(x, compute_dtype(x), wq, ws, False)
        if made is not None:
            return made[0]
    if wq.dim() != 2 or x.dim() < 1 or x.shape[-1] != PAIR * wq.shape[1]:
        raise ValueError(f"x {tuple(x.shape)} does not match the codes {tuple(wq.shape)} of a weight of {PAIR * wq.shape[-1]} columns")
    if x.dtype not in _lib.MX_DTYPE:
        raise ValueError(f"x.dtype={x.dtype} is not one of {tuple(_lib.MX_DTYPE)}")
    _lib.require_gpu(x, "x")
    n, k = wq.shape[0], x.shape[-1]
    if weight is not None and weight.shape != (n, k):
        raise ValueError(f"weight {tuple(weight.shape)} does not match the quantized one ({n}, {k})")
    if not through:
        compute = compute_dtype(x)
        xq, xs, _, _ = quantized_activation(activation_matrix(x, compute), compute, False)
        return mxfp4_matmul_pq(xq, xs, wq, ws, compute).reshape(*x.shape[:-1], n)
    wqt, wst = operands[2:] if len(operands) == 4 else (None, None)
    if recorded and x.requires_grad and wqt is None:
        raise ValueError("the gradient of x needs the weight quantized along its output axis too: pass mxfp4_operands(weight)")
    if wqt is not None and wqt.shape != (k, (n + -n % BLOCK_SCALE) // PAIR):
        raise ValueError(f"qT {tuple(wqt.shape)} is not the transposed copy of a weight ({n}, {k})")
    return _MXFP4Linear.apply(x, weight, wq, ws, wqt, wst)


class MXFP4Linear(torch.nn.Module):
    """``nn.Linear`` (no bias) whose FPROP and DGRAD multiply MXFP8 activations with the weight in MXFP4.

    ``refresh_quantized_weight`` must be called after every optimizer step.  ``dw`` comes back in the compute dtype, or in fp32 for
    an fp32 master.
    """

    def __init__(self, in_features: int, out_features: int, dtype=torch.bfloat16):
        super().__init__()
        if in_features % BLOCK_SCALE:
            raise ValueError(f"in_features={in_features} must be a multiple of {BLOCK_SCALE}: it is FPROP's contraction axis")
        self.in_features = in_features
        self.out_features = out_features
        self.weight = torch.nn.Parameter(torch.empty(out_features, in_features, dtype=dtype))
        torch.nn.init.normal_(self.weight, std=in_features**-0.5)
        self._cache: tuple[torch.Tensor, ...] | None = None

    @torch.no_grad()
    def refresh_quantized_weight(self) -> None:
        with torch.inference_mode(False):  # copies made while serving may be saved for a backward later
            self._cache = mxfp4_operands(self.weight)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if self._cache is None:
            self.refresh_quantized_weight()
        return mxfp4_linear(x, self._cache, self.weight)

    def _apply(self, *args, **kwargs):
        """Any device or dtype transform drops the quantized cache; ``forward`` rebuilds it."""
        self._cache = None
        return super()._apply(*args, **kwargs)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, mxfp4=True"
