"""Forward-mode derivatives of the residual norm and the 4-bit layers: there are none, and a call says so (no GPU: launches are left out)."""

import pytest
import torch
from torch.autograd import forward_ad

BF, U8 = torch.bfloat16, torch.uint8


@pytest.fixture(autouse=True)
def no_launches(monkeypatch):
    from kohakuwullm_amd import _lib

    monkeypatch.setattr(_lib, "require_gpu", lambda t, name: None)
    monkeypatch.setattr(_lib, "invoke", lambda *args: None)
    monkeypatch.setattr(_lib, "gemm_workspace", lambda t: torch.empty(0, dtype=U8))


def _e(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def _calls():
    """Each function as one of a single tensor that could carry a tangent, and that tensor."""
    from kohakuwullm_amd.kernels.elementwise import add_rms_norm, add_rms_norm_mx
    from kohakuwullm_amd.kernels.mxfp4 import MXFP4Linear, grouped_mxfp4_linear, mxfp4_linear

    pair, experts = (_e(8, 32, dtype=U8), _e(8, 2, dtype=U8)), (_e(3, 8, 32, dtype=U8), _e(3, 8, 2, dtype=U8))
    offsets = torch.zeros(4, dtype=torch.int32)
    for norm in (add_rms_norm, add_rms_norm_mx):
        yield lambda t, norm=norm: norm(t, _e(4, 64), _e(64))[0], _e(4, 64)
        yield lambda t, norm=norm: norm(_e(4, 64), t, _e(64))[1], _e(4, 64)
        yield lambda t, norm=norm: norm(_e(4, 64), _e(4, 64), t)[0], _e(64)
    yield lambda t: mxfp4_linear(t, pair), _e(4, 64)
    yield lambda t: mxfp4_linear(_e(4, 64), pair, t), _e(8, 64)
    yield lambda t: grouped_mxfp4_linear(t, experts, offsets), _e(4, 64)
    yield lambda t: grouped_mxfp4_linear(_e(4, 64), experts, offsets, t), _e(3, 8, 64)
    layer = MXFP4Linear(64, 8)
    layer._cache = *pair, _e(64, 16, dtype=U8), _e(64, 1, dtype=U8)
    yield layer, _e(4, 64)


CALLS = 11


@pytest.mark.parametrize("which", range(CALLS))
@pytest.mark.parametrize("recorded", [True, False])
def test_a_tangent_is_refused(which, recorded):
    call, t = list(_calls())[which]
    with torch.set_grad_enabled(recorded), forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="jvp"):
            call(forward_ad.make_dual(t, torch.ones_like(t)))


@pytest.mark.parametrize("which", range(CALLS))
def test_a_call_without_one_goes_on(which):
    """Beside tangents of other tensors, and where no level is open."""
    call, t = list(_calls())[which]
    assert isinstance(call(t), torch.Tensor)
    with forward_ad.dual_level():
        other = forward_ad.make_dual(torch.ones(2), torch.ones(2))
        assert isinstance(call(t), torch.Tensor) and forward_ad.unpack_dual(other * 2).tangent.tolist() == [2.0, 2.0]


@pytest.mark.parametrize("which", range(CALLS))
def test_the_transform_is_refused(which):
    call, t = list(_calls())[which]
    with pytest.raises(RuntimeError):
        torch.func.jvp(call, (t,), (torch.ones_like(t),))


def test_an_open_level_asks_for_nothing_more():
    """A call without gradients takes what it takes elsewhere: no copy of the weight along its output axis, any width."""
    from kohakuwullm_amd.kernels.elementwise import add_rms_norm
    from kohakuwullm_amd.kernels.mxfp4 import grouped_mxfp4_linear, mxfp4_linear

    with torch.no_grad(), forward_ad.dual_level():
        assert mxfp4_linear(_e(4, 64).requires_grad_(), (_e(8, 32, dtype=U8), _e(8, 2, dtype=U8))).shape == (4, 8)
        pair = _e(3, 8, 32, dtype=U8), _e(3, 8, 2, dtype=U8)
        assert grouped_mxfp4_linear(_e(4, 64).requires_grad_(), pair, torch.zeros(4, dtype=torch.int32)).shape == (4, 8)
        assert add_rms_norm(_e(2, 16392).requires_grad_(), _e(2, 16392), None)[0].shape == (2, 16392)


def test_number_of_calls():
    assert len(list(_calls())) == CALLS
