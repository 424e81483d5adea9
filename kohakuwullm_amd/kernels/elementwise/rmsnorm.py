"""RMSNorm that can hand the next projection its MXFP8 operand: ``(out, e4m3, ue8m0)`` from one pass.

Counterpart of ``src/kohakuwullm/kernels/elementwise/rmsnorm.py`` (``_RMSNorm`` :130-229,
``rms_norm`` :232-236, ``rms_norm_mx`` :239-246, ``rms_norm_mx_vendor`` :249-258).  The fp8 pair is
quantized from the fp32 normalized row, not from the rounded 16-bit ``out``, and carries no
gradient: dgrad reaches the norm through ``out``.

Differences from the reference, on purpose: the tensors must live on the GPU (there is no ATen
route here, so ``rms_norm`` on a CPU tensor raises instead of falling back), any row width that is
a multiple of 8 is taken (no 16384 cap), and the sum of squares is accumulated in fp64.
"""

from __future__ import annotations

import functools

import torch
from torch.autograd.function import once_differentiable

from kohakuwullm_amd import _lib, host
from kohakuwullm_amd.kernels.mxfp8.quantize import BLOCK_SCALE, aligned_rows

_FP8 = torch.float8_e4m3fn
_E8M0 = getattr(torch, "float8_e8m0fnu", torch.uint8)
_ACT = (torch.bfloat16, torch.float16)
# Partial weight-gradient rows = workgroups of the backward kernel.  The reference fixes 512 (rmsnorm.py:206); here the
# kernel holds three waves per SIMD, i.e. three workgroups per CU, and fewer leave a third of the latency hiding unused
# (32768 x 2048 bf16 on 256 CUs: 110 us with 512, 94 us with 768, 115 us with 1024, which runs a ragged second round).
BWD_WORKGROUPS_PER_CU = 3


@functools.lru_cache(maxsize=64)
def backward_partial_rows(device) -> int:
    return BWD_WORKGROUPS_PER_CU * torch.cuda.get_device_properties(device).multi_processor_count


def launch_rmsnorm(x2d, weight, eps: float, out, rstd, q, s) -> None:
    """One launch of ``mx_rmsnorm_quantize``; any of ``out``, ``rstd``, ``(q, s)`` may be ``None``."""
    m, k = x2d.shape
    written = (0 if out is None else x2d.element_size()) + (0 if q is None else 1 + 1 / BLOCK_SCALE)
    _lib.invoke(
        "mx_rmsnorm_quantize", m * k * (x2d.element_size() + written), x2d,
        x2d.data_ptr(), _lib.MX_DTYPE[x2d.dtype], m, k, x2d.stride(0),
        0 if weight is None else weight.data_ptr(), 0 if weight is None else _lib.MX_DTYPE[weight.dtype], float(eps),
        0 if out is None else out.data_ptr(), 0 if out is None else out.stride(0),
        0 if rstd is None else rstd.data_ptr(),
        0 if q is None else q.data_ptr(), 0 if q is None else q.stride(0),
        0 if s is None else s.data_ptr(), 0 if s is None else s.stride(0),
    )


def _check(x: torch.Tensor, weight: torch.Tensor | None, quant: bool) -> None:
    _lib.require_gpu(x, "x")
    k = x.shape[-1]
    if x.dtype not in _ACT:
        raise ValueError(f"x.dtype={x.dtype} is not one of {_ACT}")
    if weight is not None:
        _lib.require_gpu(weight, "weight")
        if weight.shape != (k,):
            raise ValueError(f"weight {tuple(weight.shape)} does not match the row width {k}")
        if weight.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"weight.dtype={weight.dtype} must be {x.dtype} or float32")
    if quant and k % BLOCK_SCALE:
        raise ValueError(f"quant needs n_cols % {BLOCK_SCALE} == 0, got {k}")


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, quant=False, write_out=True, swizzle=False):
        if not quant and write_out:
            made = host.rmsnorm_forward(x, weight, eps)
            if made is not None:
                out, x2d, rstd = made
                ctx.save_for_backward(x2d, weight, rstd)
                ctx.set_materialize_grads(False)
                return out
        _check(x, weight, quant)
        shape = x.shape
        x2d = x.reshape(-1, shape[-1]).contiguous()
        n_rows, n_cols = x2d.shape
        if swizzle and n_cols % (4 * BLOCK_SCALE):
            raise ValueError(f"swizzle needs n_cols % {4 * BLOCK_SCALE} == 0")
        if weight is not None:
            weight = weight.contiguous()
        dev = x2d.device
        rstd = torch.empty(n_rows, dtype=torch.float32, device=dev)
        out = torch.empty_like(x2d) if write_out else None
        q = s = None
        if quant:
            q = torch.empty(n_rows, n_cols, dtype=_FP8, device=dev)
            s = torch.empty(n_rows, n_cols // BLOCK_SCALE, dtype=torch.uint8, device=dev)
        if n_rows and n_cols:
            launch_rmsnorm(x2d, weight, eps, out, rstd, q, s)
        ctx.save_for_backward(x2d, weight, rstd)
        # without this autograd would fill zero "gradients" for the fp8 pair on every backward
        ctx.set_materialize_grads(False)
        if out is None:
            out = x2d.new_empty(0)
        elif write_out:
            out = out.reshape(shape)
        if not quant:
            return out
        if swizzle:
            from kohakuwullm_amd.kernels.mxfp8.interop import swizzle_mx_scales

            s = swizzle_mx_scales(s)  # flat, zero padded to whole 128-row tiles
        # the fp8 pair carries no gradient; dgrad reaches the norm through `out`
        ctx.mark_non_differentiable(q, s)
        return out, q, s

    @staticmethod
    def backward(ctx, dout, *_unused_fp8_grads):
        if dout is None:
            return None, None, None, None, None, None
        x2d, weight, rstd = ctx.saved_tensors
        made = host.rmsnorm_backward(dout, x2d, weight, rstd, ctx.needs_input_grad[1], backward_partial_rows(x2d.device))
        if made is not None:
            return *made, None, None, None, None
        shape = dout.shape
        dout2d = dout.reshape(-1, shape[-1]).contiguous()
        n_rows, n_cols = x2d.shape
        dx = torch.empty_like(x2d)
        has_w = weight is not None and ctx.needs_input_grad[1]
        parts = max(1, min((n_rows + 3) // 4, backward_partial_rows(x2d.device)))
        dw_part = torch.empty(parts, n_cols, dtype=torch.float32, device=x2d.device) if has_w else None
        if n_cols:
            _lib.invoke(
                "mx_rmsnorm_backward", n_rows * n_cols * 3 * x2d.element_size(), x2d,
                x2d.data_ptr(), _lib.MX_DTYPE[x2d.dtype], n_rows, n_cols, x2d.stride(0),
                0 if weight is None else weight.data_ptr(), 0 if weight is None else _lib.MX_DTYPE[weight.dtype],
                dout2d.data_ptr(), dout2d.stride(0), rstd.data_ptr(), dx.data_ptr(), dx.stride(0),
                0 if dw_part is None else dw_part.data_ptr(), parts,
            )
        dw = torch.empty(n_cols, dtype=weight.dtype, device=x2d.device) if has_w else None
        if has_w and n_cols:
            _lib.invoke("mx_rmsnorm_weight_grad", dw_part.numel() * 4, x2d, dw_part.data_ptr(), parts, n_cols, dw.data_ptr(),
                        _lib.MX_DTYPE[weight.dtype])
        return dx.reshape(shape), dw, None, None, None, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None, eps: float = 1e-6) -> torch.Tensor:
    """Fused RMSNorm on the GPU (no MXFP8 output)."""
    if host.unrecorded(x, weight):
        made = host.rmsnorm_forward(x, weight, eps)
        if made is not None:
            return made[0]
    return _RMSNorm.apply(x, weight, eps)


def rms_norm_mx(x: torch.Tensor, weight: torch.Tensor | None, eps: float = 1e-6):
    """Fused RMSNorm returning ``(out, e4m3, ue8m0)``, the fp8 pair K-blocked: ``(rows, K)``, ``(rows, K//32)``."""
    return _RMSNorm.apply(x, weight, eps, True, True)


def rms_norm_mx_vendor(x: torch.Tensor, weight: torch.Tensor | None, eps: float = 1e-6):
    """RMSNorm emitting scales in the flat ``SWIZZLE_32_4_4`` exchange layout (zero padded to 128-row tiles)."""
    out, q, s = _RMSNorm.apply(x, weight, eps, True, True, True)
    return out, q, s.view(_E8M0)


# The norm behind the residual sum of a block.  The reference adds first and norms the sum it has written (the ``rms_norm`` above);
# here the sum, which the residual stream needs anyway, is written by the kernel that norms it.

ADD_NORM_BACKWARD_MAX = 16384  # columns the backward holds in registers


def _check_add(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None, quant: bool) -> None:
    if not x.dim() or not x.shape[-1] or x.shape[-1] % 8:
        raise ValueError(f"x {tuple(x.shape)}: the row width must be a positive multiple of 8")
    if residual.shape != x.shape:
        raise ValueError(f"residual {tuple(residual.shape)} does not match x {tuple(x.shape)}")
    if residual.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"residual.dtype={residual.dtype} must be {x.dtype} or float32")
    _check(x, weight, quant)
    _lib.require_same_device(x, residual=residual, weight=weight)


def launch_add_rmsnorm(x, residual, weight, eps: float, write_out: bool, rstd: bool, quant: bool):
    """``(out, h, rstd, q, s)`` of one launch; what is not asked for is ``None``."""
    made = host.add_norm(x, residual, weight, eps, write_out, rstd, quant)
    if made is not None:
        return made
    _check_add(x, residual, weight, quant)
    shape, k = x.shape, x.shape[-1]
    rows = x.numel() // k
    dev = x.device
    h = torch.empty(shape, dtype=residual.dtype, device=dev)
    out = torch.empty(shape, dtype=x.dtype, device=dev) if write_out else None
    r = torch.empty(rows, dtype=torch.float32, device=dev) if rstd else None
    q = torch.empty(rows, k, dtype=_FP8, device=dev) if quant else None
    s = torch.empty(rows, k // BLOCK_SCALE, dtype=torch.uint8, device=dev) if quant else None
    if rows:
        x2d, r2d = aligned_rows(x.reshape(rows, k)), aligned_rows(residual.reshape(rows, k))
        w = None if weight is None else _vector(weight)
        written = h.element_size() + (x.element_size() if write_out else 0) + (1 + 1 / BLOCK_SCALE if quant else 0)
        _lib.call(
            "mx_add_rmsnorm_quantize", rows * k * (x.element_size() + h.element_size() + written), x,
            x2d.data_ptr(), _lib.MX_DTYPE[x.dtype], rows, k, max(x2d.stride(0), k), r2d.data_ptr(), _lib.MX_DTYPE[h.dtype], max(r2d.stride(0), k),
            0 if w is None else w.data_ptr(), 0 if w is None else _lib.MX_DTYPE[w.dtype], float(eps), h.data_ptr(), k,
            0 if out is None else out.data_ptr(), k, 0 if r is None else r.data_ptr(),
            0 if q is None else q.data_ptr(), k, 0 if s is None else s.data_ptr(), k // BLOCK_SCALE)
    return out, h, r, q, s


def _vector(weight: torch.Tensor) -> torch.Tensor:
    """A norm's weight as the kernels read it: one run that starts on a 16-byte boundary."""
    return weight if weight.is_contiguous() and weight.data_ptr() % 16 == 0 else weight.clone(memory_format=torch.contiguous_format)


class _AddRMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps, quant):
        out, h, rstd, q, s = launch_add_rmsnorm(x, residual, weight, eps, True, True, quant)
        ctx.save_for_backward(h, weight, rstd)
        ctx.x_dtype = x.dtype
        # Leaves keep their gradients, and of a tensor that is handed to two autograd gives one a copy: then it is written twice here.
        # Everywhere else it is passed on as it is.
        ctx.apart = x.dtype != residual.dtype or (x.is_leaf and residual.is_leaf)
        ctx.set_materialize_grads(False)
        if not quant:
            return out, h
        ctx.mark_non_differentiable(q, s)  # no gradient: dgrad reaches the norm through `out`
        return out, h, q, s

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dh, *_unused_fp8_grads):
        h, weight, rstd = ctx.saved_tensors
        need_x, need_r, need_w = ctx.needs_input_grad[:3]
        if dout is None:  # the norm's output is not used: the sum alone
            if dh is None:
                return None, None, None, None, None
            return dh.to(ctx.x_dtype) if need_x else None, dh if need_r else None, None, None, None
        made = host.add_norm_backward(dout, dh, h, weight, rstd, need_x, need_r, need_w, ctx.apart, backward_partial_rows(h.device))
        if made is not None:
            d, dr, dw = made
            return d if need_x else None, (d if dr is None else dr) if need_r else None, dw, None, None
        shape, k = h.shape, h.shape[-1]
        rows, dev, one = h.numel() // k, h.device, not (ctx.apart and need_x and need_r) and h.dtype == ctx.x_dtype
        dx = torch.empty(shape, dtype=ctx.x_dtype, device=dev) if need_x or (need_r and one) else None
        dr = torch.empty(shape, dtype=h.dtype, device=dev) if need_r and not one else None
        parts = max(1, min((rows + 3) // 4, backward_partial_rows(dev)))
        part = torch.empty(parts, k, dtype=torch.float32, device=dev) if need_w else None
        if rows:
            h2d, d2d = aligned_rows(h.reshape(rows, k)), aligned_rows(dout.reshape(rows, k))
            dh2d = None if dh is None else aligned_rows(dh.reshape(rows, k))
            w = None if weight is None else _vector(weight)
            _lib.call(
                "mx_add_rmsnorm_backward", rows * k * (2 * h.element_size() + 2 * dout.element_size()), h,
                h2d.data_ptr(), _lib.MX_DTYPE[h.dtype], rows, k, max(h2d.stride(0), k), 0 if w is None else w.data_ptr(),
                0 if w is None else _lib.MX_DTYPE[w.dtype], d2d.data_ptr(), _lib.MX_DTYPE[ctx.x_dtype], max(d2d.stride(0), k),
                0 if dh2d is None else dh2d.data_ptr(), k if dh2d is None else max(dh2d.stride(0), k), rstd.data_ptr(),
                0 if dx is None else dx.data_ptr(), k, 0 if dr is None else dr.data_ptr(), k, 0 if part is None else part.data_ptr(), parts)
        dw = None
        if need_w and not rows:
            dw = torch.zeros(k, dtype=weight.dtype, device=dev)
        elif need_w:
            dw = torch.empty(k, dtype=weight.dtype, device=dev)
            _lib.call("mx_rmsnorm_weight_grad", part.numel() * 4, part, part.data_ptr(), parts, k, dw.data_ptr(), _lib.MX_DTYPE[weight.dtype])
        return dx if need_x else None, (dx if one else dr) if need_r else None, dw, None, None


def _add_norm(x, residual, weight, eps, quant):
    recorded = _lib.recorded(x, residual, weight)
    if recorded and x.dim() and x.shape[-1] > ADD_NORM_BACKWARD_MAX:
        raise ValueError(f"gradients need a row width of {ADD_NORM_BACKWARD_MAX} at most, got {x.shape[-1]}")
    if recorded or _lib.forward_mode():
        return _AddRMSNorm.apply(x, residual, weight, eps, quant)
    out, h, _, q, s = launch_add_rmsnorm(x, residual, weight, eps, True, False, quant)
    return (out, h, q, s) if quant else (out, h)


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None, eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """``h = x + residual`` and its RMSNorm: ``(out, h)``, one pass over both.

    ``x``: bf16 or fp16, its last axis a multiple of 8.  ``residual``: of ``x``'s shape, in ``x``'s type or in fp32; ``h`` has its type, and
    the norm reads the rounded ``h``.  ``out`` has ``x``'s type; for a 16-bit stream it is ``rms_norm(h, weight, eps)`` bit for bit.
    ``weight``: the row's width in ``x``'s type or fp32, or ``None``.  Differentiable in all three
    (reverse mode).
    """
    return _add_norm(x, residual, weight, eps, False)


def add_rms_norm_mx(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None, eps: float = 1e-6):
    """:func:`add_rms_norm` that also hands the next projection its MXFP8 operand: ``(out, h, e4m3, ue8m0)``.

    The pair is quantized from the fp32 normalized row, K-blocked, ``(rows, K)`` and ``(rows, K//32)``, and carries no gradient.
    """
    return _add_norm(x, residual, weight, eps, True)
