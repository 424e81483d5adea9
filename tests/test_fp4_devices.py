"""Calls on tensors of a device that is not the current one make it current around their launches (no GPU: the devices are stood in for)."""

import contextlib

import pytest
import torch

BF, FP8, U8 = torch.bfloat16, torch.float8_e4m3fn, torch.uint8


def _e(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def _calls():
    from kohakuwullm_amd.kernels import mxfp4 as m
    from kohakuwullm_amd.kernels.elementwise import add_rms_norm, add_rms_norm_mx
    from kohakuwullm_amd.kernels.mxfp8.fused_act import add_rmsnorm_mx

    pair, four = (_e(32, 32, dtype=U8), _e(32, 2, dtype=U8)), (_e(32, 32, dtype=U8), _e(32, 2, dtype=U8), _e(64, 16, dtype=U8), _e(64, 1, dtype=U8))
    experts, offsets = (_e(3, 32, 32, dtype=U8), _e(3, 32, 2, dtype=U8)), torch.zeros(4, dtype=torch.int32)
    e4m3 = _e(4, 64, dtype=U8).view(FP8), _e(4, 2, dtype=U8)
    weight = _e(32, 64).requires_grad_()
    yield "mx_add_rmsnorm_quantize", lambda: add_rms_norm(_e(4, 64), _e(4, 64), None)
    yield "mx_add_rmsnorm_quantize", lambda: add_rms_norm_mx(_e(4, 64).requires_grad_(), _e(4, 64), _e(64))
    yield "mx_add_rmsnorm_quantize", lambda: add_rmsnorm_mx(_e(4, 64), _e(4, 64), _e(64))
    yield "mx_rmsnorm_weight_grad", lambda: add_rms_norm(_e(4, 64), _e(4, 64), _e(64).requires_grad_())[0].sum().backward()
    yield "mx_fp4_quantize_rows", lambda: m.quantize_mxfp4(_e(4, 64))
    yield "mx_fp4_quantize_cols", lambda: m.quantize_mxfp4(_e(64, 64).t())
    yield "mx_fp4_quantize_cols", lambda: m.quantize_mxfp4_cols(_e(64, 64))
    yield "mx_fp4_quantize_cols", lambda: m.mxfp4_operands(_e(3, 32, 64))
    yield "mx_dequantize_rows", lambda: m.dequantize_mx(*pair)
    yield "mx_turn_bytes", lambda: m.dequantize_mx(_e(32, 32, dtype=U8).t(), _e(32, 2, dtype=U8))
    yield "mx_fp4_gemm_nt", lambda: m.mxfp4_matmul_pq(*e4m3, *pair)
    yield "mx_fp4_gemm_nt", lambda: m.mxfp4_matmul(_e(4, 64), _e(8, 64))
    yield "mx_fp4_gemm_nt", lambda: m.mxfp4_linear(_e(4, 64), pair)
    yield "mx_fp4_gemm_nt", lambda: m.mxfp4_linear(_e(4, 64).requires_grad_(), four, weight)
    yield "mx_fp4_grouped_gemm_nt", lambda: m.grouped_mxfp4_gemm(*e4m3, *experts, offsets)
    yield "mx_fp4_grouped_gemm_nt", lambda: m.grouped_mxfp4_linear(_e(4, 64), experts, offsets)
    yield "mx_fp4_gemm_nt", lambda: m.MXFP4Linear(64, 32)(_e(4, 64))


CALLS = 17


@pytest.mark.parametrize("which", range(CALLS))
def test_launches_are_made_on_the_tensors_device(which, monkeypatch):
    from kohakuwullm_amd import _lib

    inside, launched, entered = [], [], []

    @contextlib.contextmanager
    def device(d):
        entered.append(d)
        inside.append(d)
        yield
        inside.pop()

    monkeypatch.setattr(_lib, "require_gpu", lambda t, name: None)
    monkeypatch.setattr(_lib, "elsewhere", lambda t: not inside)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(_lib, "gemm_workspace", lambda t: torch.empty(0, dtype=U8))
    monkeypatch.setattr(_lib, "invoke", lambda name, work, tensor, *args: launched.append((name, len(inside))))
    from kohakuwullm_amd.kernels.elementwise import rmsnorm

    monkeypatch.setattr(rmsnorm, "backward_partial_rows", lambda d: 1)
    last, call = list(_calls())[which]
    call()
    assert last in [name for name, _ in launched] and all(depth == 1 for _, depth in launched), launched
    assert entered and all(d == torch.device("cpu") for d in entered)


def test_number_of_calls():
    assert len(list(_calls())) == CALLS
