"""Refusals of the residual norm and of the delta rule that need no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from taac_2026_amd import _native
from taac_2026_amd.api import residual_rms_norm, residual_rms_norm_fp8


@pytest.mark.parametrize("operator", [residual_rms_norm, residual_rms_norm_fp8])
def test_residual_norm_refuses(operator):
    x, w = torch.zeros(4, 8), torch.ones(8)
    with pytest.raises(ValueError, match="at least 2 dimensions"):
        operator(torch.zeros(8), torch.zeros(8), w)
    with pytest.raises(ValueError, match="residual shape"):
        operator(x, torch.zeros(1, 8), w)
    with pytest.raises(ValueError, match="1D"):
        operator(x, x, torch.ones(1, 8))
    with pytest.raises(ValueError, match="does not match weight size"):
        operator(x, x, torch.ones(7))
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        operator(x, x, w)


def test_residual_norm_entry_points_check_on_the_host():
    library = _native.load_library()
    fake = ctypes.c_void_p(256)
    bf16, invalid = _native.TAAC_BF16, _native.TAAC_ERR_INVALID_VALUE
    assert library.taac_residual_rmsnorm_fwd(fake, fake, fake, fake, fake, 4, 0, 1e-6, bf16, None) == invalid
    assert library.taac_residual_rmsnorm_fwd(fake, fake, fake, fake, fake, -1, 8, 1e-6, bf16, None) == invalid
    assert library.taac_residual_rmsnorm_fwd(fake, None, fake, fake, fake, 4, 8, 1e-6, bf16, None) == invalid
    assert library.taac_residual_rmsnorm_fwd(fake, fake, fake, fake, fake, 4, 8, 1e-6, 9, None) == invalid
    assert library.taac_residual_rmsnorm_fwd(None, None, None, None, None, 0, 8, 1e-6, bf16, None) == _native.TAAC_OK
    assert library.taac_residual_rmsnorm_fp8_fwd(fake, fake, fake, fake, fake, None, 4, 8, 1e-6, bf16, None) == invalid
    assert library.taac_residual_rmsnorm_bwd(fake, fake, fake, None, fake, fake, fake, 7, 4, 8, 1e-6, bf16, None) == invalid
    assert b"workspace" in library.taac_last_error()
    assert library.taac_residual_rmsnorm_bwd(fake, fake, None, None, fake, fake, fake, 1 << 20, 4, 8, 1e-6, bf16, None) == invalid
    # rows with maxima of their own: the checks of the tensor-wide form
    assert library.taac_linear_fp8_rows(fake, 16, fake, None, fake, None, None, fake, 16, 4, 16, 16, 0, 1, None) == invalid
    assert library.taac_linear_fp8_rows(fake, 24, fake, fake, fake, None, None, fake, 16, 4, 16, 16, 0, 1, None) == \
        _native.TAAC_ERR_UNSUPPORTED
