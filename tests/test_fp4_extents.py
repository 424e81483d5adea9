"""Extents that the kernels' 32-bit arithmetic cannot carry past a matrix's end are refused before any pointer is followed."""

import pytest

MOST = (1 << 31) - 1024  # rows, columns and contraction of a product: stages, tiles and strides of a loop are added to them
PAST = [(MOST + 32, 32, 32), (32, MOST + 32, 32), (1, 16, MOST + 32), (1, 16, (1 << 31) - 32), ((1 << 31) - 1, 1, 32), (1, (1 << 31) - 1, 32)]


@pytest.mark.parametrize("m,n,k", PAST)
def test_product(m, n, k):
    from kohakuwullm_amd import _lib

    lib, at = _lib.load(), 1 << 20
    for fmt, row in ((_lib.MX_E4M3, k), (_lib.MX_E2M1, k // 2)):
        assert lib.mx_fp4_gemm_nt(at, at, fmt, at, at, at, 0, m, n, k, row, k // 32, k // 2, k // 32, n, None, 0, None) == _lib.MX_EUNSUPPORTED
    assert lib.mx_fp4_gemm_nt(at, at, 0, at, at, at, 0, m, n, 0, 0, 0, 0, 0, n, None, 0, None) == _lib.MX_EUNSUPPORTED or k > MOST


@pytest.mark.parametrize("m,n,k", PAST)
def test_experts(m, n, k):
    from kohakuwullm_amd import _lib

    lib, at = _lib.load(), 1 << 20
    call = lambda m, n, k, zero: lib.mx_fp4_grouped_gemm_nt(  # noqa: E731
        at, at, 0, m, k, k // 32, None, at, at, n * k // 2, k // 2, n * k // 32, k // 32, at, 2, at, 0, n, m, n, k, zero, None)
    expected = _lib.MX_EINVAL if m >= (1 << 31) - 1 else _lib.MX_EUNSUPPORTED
    assert call(m, n, k, 0) == expected and call(m, n, k, 1) == expected
    assert k > MOST or call(m, n, 0, 1) == expected


@pytest.mark.parametrize("m,n,k", PAST)
def test_activations(m, n, k):
    from kohakuwullm_amd import _lib

    lib, at = _lib.load(), 1 << 20
    assert lib.mx_fp4_activation_gemm_nt(at, 0, k, at, at, at, 0, m, n, k, k // 2, k // 32, n, None) == _lib.MX_EUNSUPPORTED

