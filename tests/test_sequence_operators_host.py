"""Refusals of the residual norm and of the delta rule that need no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from taac_2026_amd import _native
from taac_2026_amd.api import gated_delta_rule, gated_delta_rule_step, linear_fp8, norm_linear_fp8, residual_rms_norm, residual_rms_norm_fp8


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


def _delta_inputs(batch=1, key_heads=1, heads=2, tokens=5, key_width=16, value_width=8):
    q, k = (torch.zeros(batch, key_heads, tokens, key_width, dtype=torch.bfloat16) for _ in range(2))
    v = torch.zeros(batch, heads, tokens, value_width, dtype=torch.bfloat16)
    return [q, k, v, torch.zeros(batch, heads, tokens), torch.zeros(batch, heads, tokens)]


@pytest.mark.parametrize("operator", [gated_delta_rule, lambda *a, **kw: gated_delta_rule_step(*a, torch.zeros(1, 2, 16, 8), **kw)])
def test_delta_rule_refuses(operator):
    q, k, v, g, b = _delta_inputs()
    with pytest.raises(ValueError, match="shape \\(batch, heads"):
        operator(q[0], k, v, g, b)
    with pytest.raises(ValueError, match="same shape"):
        operator(q[..., :8], k, v, g, b)
    with pytest.raises(ValueError, match="token dimensions"):
        operator(q, k, v[:, :, :4], g, b)
    with pytest.raises(ValueError, match="multiple of the key heads"):
        operator(q.expand(1, 3, 5, 16), k.expand(1, 3, 5, 16), v, g, b)
    with pytest.raises(ValueError, match="log_decay and beta"):
        operator(q, k, v, g[..., :4], b)
    with pytest.raises(ValueError, match="same dtype"):
        operator(q, k.float(), v, g, b)
    with pytest.raises(ValueError, match="same dtype"):
        operator(q, k, v, g, b.bfloat16())
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        operator(q, k, v, g, b)


def test_delta_step_refuses():
    inputs = _delta_inputs()
    with pytest.raises(ValueError, match="expects a state"):
        gated_delta_rule_step(*inputs, torch.zeros(1, 2, 8, 16))
    with pytest.raises(ValueError, match="in place"):
        gated_delta_rule_step(*inputs, torch.zeros(1, 2, 16, 8, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="in place"):
        gated_delta_rule_step(*inputs, torch.zeros(1, 2, 8, 16).transpose(2, 3))
    with pytest.raises(ValueError, match="without state_index"):
        gated_delta_rule_step(*inputs, torch.zeros(0, 2, 16, 8))
    for index in (torch.zeros(2, dtype=torch.int32), torch.zeros(1), torch.zeros(1, 1, dtype=torch.int64)):
        with pytest.raises(ValueError, match="state_index"):
            gated_delta_rule_step(*inputs, torch.zeros(1, 2, 16, 8), state_index=index)


def test_delta_entry_points_check_on_the_host():
    library = _native.load_library()
    fake, odd = ctypes.c_void_p(256), ctypes.c_void_p(258)
    strides = (ctypes.c_int64 * 3)
    invalid, unsupported, ok = _native.TAAC_ERR_INVALID_VALUE, _native.TAAC_ERR_UNSUPPORTED, _native.TAAC_OK
    f32, bf16, f16 = _native.TAAC_F32, _native.TAAC_BF16, _native.TAAC_F16

    def forward(**kw):
        a = dict(q=fake, lengths=None, final=None, states=None, misses=None, B=1, H=2, Hk=1, T=5, dk=16, dv=8, qs=strides(80, 80, 16), gs=strides(10, 5, 1), gate=f32,
                 ws=fake, bytes=1 << 20)
        a.update(kw)
        s = strides(80, 40, 8)
        return library.taac_delta_rule_fwd(a["q"], fake, fake, fake, fake, a["lengths"], fake, None, a["final"], a["states"], a["misses"], a["ws"], a["bytes"], a["B"], a["H"],
                                           a["Hk"], a["T"], a["dk"], a["dv"], a["qs"], strides(80, 80, 16), s, s, a["gs"], a["gs"], 1.0, a["gate"], None)

    assert forward(Hk=3) == invalid and b"multiple of the key heads" in library.taac_last_error()
    assert forward(H=0) == invalid and forward(B=-1) == invalid and forward(T=-1) == invalid
    assert forward(dk=12) == unsupported and forward(dv=136) == unsupported and b"multiples of 8" in library.taac_last_error()
    assert forward(gate=f16) == invalid and b"gates" in library.taac_last_error()
    assert forward(states=fake) == invalid and b"come together" in library.taac_last_error()
    assert forward(q=None) == invalid and forward(q=odd) == invalid
    assert forward(qs=strides(80, 80, 12)) == invalid and forward(gs=strides(10, 5, -1)) == invalid and forward(qs=None) == invalid
    assert forward(qs=strides(80, 80, 8)) == invalid and b"cover a row" in library.taac_last_error()
    assert forward(qs=strides(80, 80, 1 << 24)) == unsupported and forward(T=(1 << 30) + 1) == unsupported
    assert forward(B=0) == ok and forward(T=0) == ok
    need = library.taac_delta_rule_workspace_bytes(1, 2, 5, 16, 8)
    assert need > 0 and library.taac_delta_rule_workspace_bytes(1, 0, 5, 16, 8) == -1
    assert library.taac_delta_rule_workspace_bytes(4096, 8, 512, 32, 32) == 0  # many heads
    assert forward(bytes=need - 1) == invalid and b"workspace" in library.taac_last_error()
    assert forward(ws=None) == invalid and forward(ws=odd) == invalid

    def step(**kw):
        a = dict(state=fake, pool=4, slots=fake, B=1, H=2, Hk=1, T=1, dk=16, dv=8, dtype=bf16, gate=f32, qs=strides(16, 16, 16))
        a.update(kw)
        s = strides(16, 8, 8)
        return library.taac_delta_rule_step(fake, fake, fake, fake, fake, a["state"], a["pool"], a["slots"], 0, None, fake, a["B"], a["H"], a["Hk"], a["T"],
                                            a["dk"], a["dv"], a["qs"], s, s, s, s, s, 1.0, a["dtype"], a["gate"], None)

    assert step(Hk=4) == invalid and step(pool=-1) == invalid and step(state=None) == invalid and step(state=odd) == invalid
    assert step(dk=4) == unsupported and step(dtype=7) == invalid and step(gate=f16) == invalid
    assert step(slots=None, B=5) == invalid and b"without slots" in library.taac_last_error()
    assert step(qs=strides(16, -16, 16)) == invalid and step(qs=None) == invalid
    assert step(B=(1 << 28) + 1, H=1, pool=1 << 40) == unsupported and b"2^28" in library.taac_last_error()
    assert step(B=0) == ok and step(T=0) == ok


def test_linear_fp8_refuses_maxima_of_another_shape():
    """Read as one maximum, the first row's would dequantise them all."""
    x = torch.zeros(2, 3, 16).to(torch.float8_e4m3fn)
    weight, amax_w = torch.zeros(16, 16).to(torch.float8_e4m3fn), torch.ones(())
    for values, amax in ((x, (6,)), (x, (2, 3, 1)), (x, (3, 2)), (x, (3,)), (x.view(6, 16), (2, 3)), (x.view(6, 16), (6, 1)), (x.view(6, 16), (5,)), (x, (0,))):
        with pytest.raises(ValueError, match="one per row"):
            linear_fp8(values, weight, torch.ones(amax), amax_w)
    with pytest.raises(ValueError, match="float8_e4m3fn activations"):
        linear_fp8(x.bfloat16(), weight, torch.ones(2, 3), amax_w)
    for amax in ((2, 3), ()):
        with pytest.raises(ValueError, match="float32"):
            linear_fp8(x, weight, torch.ones(amax, dtype=torch.bfloat16), amax_w)
    for amax in ((2, 3), (), (1,), (1, 1)):  # as they should be: only the device is wrong
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            linear_fp8(x, weight, torch.ones(amax), amax_w)


def test_norm_linear_fp8_takes_one_maximum():
    """It quantises its rows itself: maxima of rows would be read as the first one."""
    x, weight = torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(64, 256).to(torch.float8_e4m3fn)
    for amax in (torch.ones(4), torch.ones(4, 1), torch.ones(0), torch.ones((), dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="float32 scalar"):
            norm_linear_fp8(x, weight, amax, torch.ones(()))
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        norm_linear_fp8(x, weight, torch.ones(1), torch.ones(()))
