"""Gated delta rule: a sequence mixer whose state has a fixed size, beside softmax attention.

Per sample and value head, with ``a_t = exp(log_decay_t)``, the state ``S`` (key width, value width; float32) follows

    S <- a_t S;   S <- S + k_t (beta_t (v_t - S^T k_t))^T;   o_t = scale S^T q_t

:func:`gated_delta_rule` runs whole histories in chunks on the matrix units (``taac_delta_rule_fwd`` / ``_bwd``), forward and
backward; :func:`gated_delta_rule_step` applies a few new tokens to states that a serving program keeps
(``taac_delta_rule_step``). The role of the reference's chunked gated delta rule
(src/taac2026/infrastructure/accelerators/attention/gated_delta_rule.py), on tensors laid out as :func:`flash_attention` takes
them, (batch, heads, tokens, width).
"""

from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd.function import once_differentiable

from taac_2026_amd import _native
from taac_2026_amd.accelerators.tensor_validation import require_cuda_tensors, require_inference, require_same_dtype

CHUNK = 64
MAX_WIDTH = 128
_Strides = ctypes.c_int64 * 3


def _check_shapes(name: str, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, beta: torch.Tensor) -> None:
    q_shape, k_shape, v_shape = q.shape, k.shape, v.shape
    if len(q_shape) != 4 or len(k_shape) != 4 or len(v_shape) != 4:
        raise ValueError(f"{name} expects q, k, and v with shape (batch, heads, tokens, width)")
    if q_shape != k_shape:
        raise ValueError(f"{name} requires q and k of the same shape, got {tuple(q_shape)} and {tuple(k_shape)}")
    if v_shape[0] != k_shape[0] or v_shape[2] != k_shape[2]:
        raise ValueError(f"{name} requires matching batch and token dimensions of k and v")
    if k_shape[1] == 0 or v_shape[1] == 0 or v_shape[1] % k_shape[1] != 0:
        raise ValueError(f"{name} requires a number of value heads that is a multiple of the key heads")
    if log_decay.shape != v_shape[:3] or beta.shape != v_shape[:3]:
        raise ValueError(f"{name} expects log_decay and beta with shape (batch, value heads, tokens)")
    if not q.dtype == k.dtype == v.dtype:
        require_same_dtype(f"{name} q, k, v", q, k, v)
    if log_decay.dtype != beta.dtype:
        require_same_dtype(f"{name} gates", log_decay, beta)


def _check_widths(name: str, key_width: int, value_width: int) -> None:
    if key_width <= 0 or value_width <= 0 or key_width % 8 != 0 or value_width % 8 != 0 or max(key_width, value_width) > MAX_WIDTH:
        raise RuntimeError(f"{name} is built for key and value widths that are multiples of 8, at most {MAX_WIDTH}")


def _lengths(name: str, key_lengths: torch.Tensor | None, batch: int, device: torch.device) -> torch.Tensor | None:
    if key_lengths is None:
        return None
    if key_lengths.shape != (batch,) or key_lengths.dtype.is_floating_point or key_lengths.dtype == torch.bool:
        raise ValueError(f"{name} key_lengths must hold one integer per sample")
    return key_lengths.to(device=device, dtype=torch.int32).contiguous()


@functools.lru_cache(maxsize=256)
def _stride_array(batch: int, head: int, token: int) -> ctypes.Array:
    return _Strides(batch, head, token)


def _strides(t: torch.Tensor) -> ctypes.Array:
    """Of (batch, head, token), for the library to read. The arrays are kept by value: a serving program repeats a few."""
    return _stride_array(*t.stride()[:3])


def _rows_view(t: torch.Tensor) -> torch.Tensor:
    """``t`` where the chunk kernels can read it in place (contiguous rows at 16-byte addresses, not overlapping and not too far apart), else a copy."""
    strides = t.stride()
    apart = t.shape[3] <= strides[2] < 1 << 24
    if strides[3] == 1 and apart and strides[0] % 8 == strides[1] % 8 == strides[2] % 8 == 0 and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _token_major(batch: int, heads: int, tokens: int, width: int, like: torch.Tensor) -> torch.Tensor:
    """(batch, heads, tokens, width) whose memory order is (batch, tokens, heads, width): the rows of the layers around it."""
    return like.new_empty_strided((batch, heads, tokens, width), (tokens * heads * width, width, heads * width, 1))


@functools.lru_cache(maxsize=256)
def _workspace_bytes(batch: int, heads: int, tokens: int, key_width: int, value_width: int) -> int:
    return _native.load_library().taac_delta_rule_workspace_bytes(batch, heads, tokens, key_width, value_width)


def _workspace(like: torch.Tensor, batch: int, heads: int, tokens: int, key_width: int, value_width: int) -> torch.Tensor:
    return like.new_empty(_workspace_bytes(batch, heads, tokens, key_width, value_width), dtype=torch.uint8)


def _forward(q, k, v, log_decay, beta, scale, lengths, initial_state, return_state, keep):
    batch, key_heads, tokens, key_width = k.shape
    heads, value_width = v.shape[1], v.shape[3]
    out = _token_major(batch, heads, tokens, value_width, v)
    final = v.new_empty(batch, heads, key_width, value_width, dtype=torch.float32) if return_state else None
    states = misses = None
    if keep:
        states = v.new_empty(batch, heads, (tokens + CHUNK - 1) // CHUNK, value_width, key_width)
        misses = v.new_empty(2, batch, heads, tokens, value_width)
    library = _native.load_library()
    workspace = _workspace(v, batch, heads, tokens, key_width, value_width)
    with _native.on_device(v.device):
        status = library.taac_delta_rule_fwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), beta.data_ptr(), _native.ptr(lengths), out.data_ptr(),
            _native.ptr(initial_state), _native.ptr(final), _native.ptr(states), _native.ptr(misses), _native.ptr(workspace),
            workspace.numel(), batch, heads, key_heads, tokens,
            key_width, value_width, _strides(q), _strides(k), _strides(v), _strides(out), _strides(log_decay), _strides(beta),
            float(scale), _native.dtype_code(beta.dtype), _native.current_stream(v.device))
    _native.check(status, "gated_delta_rule")
    return out, final, states, misses


class _GatedDeltaRuleFunction(torch.autograd.Function):
    """The forward keeps the state in front of every chunk in bf16 and what the state missed of every value in two parts of bf16;
    the backward makes the rest again from q, k and the gates."""

    @staticmethod
    def forward(ctx, q, k, v, log_decay, beta, scale: float, lengths, initial_state):
        q, k, v = _rows_view(q), _rows_view(k), _rows_view(v)
        out, _, states, misses = _forward(q, k, v, log_decay, beta, scale, lengths, initial_state, False, True)
        ctx.save_for_backward(q, k, log_decay, beta, lengths, states, misses)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        q, k, log_decay, beta, lengths, states, misses = ctx.saved_tensors
        batch, key_heads, tokens, key_width = k.shape
        heads, value_width = misses.shape[2], misses.shape[4]
        grad_out = _rows_view(grad_out)
        library = _native.load_library()
        with _native.on_device(k.device):
            grad_q, grad_k = (_token_major(batch, key_heads, tokens, key_width, k) for _ in range(2))
            grad_v = _token_major(batch, heads, tokens, value_width, k)
            grad_decay, grad_beta = (beta.new_empty_strided((batch, heads, tokens), (tokens * heads, 1, heads)) for _ in range(2))
            grad_states, workspace = torch.empty_like(states), _workspace(k, batch, heads, tokens, key_width, value_width)
            status = library.taac_delta_rule_bwd(
                q.data_ptr(), k.data_ptr(), log_decay.data_ptr(), beta.data_ptr(), _native.ptr(lengths), states.data_ptr(),
                misses.data_ptr(), grad_out.data_ptr(), grad_q.data_ptr(), grad_k.data_ptr(), grad_v.data_ptr(), grad_decay.data_ptr(),
                grad_beta.data_ptr(), grad_states.data_ptr(), workspace.data_ptr(), workspace.numel(), batch, heads, key_heads, tokens,
                key_width, value_width, _strides(q),
                _strides(k), _strides(log_decay), _strides(beta), _strides(grad_out), _strides(grad_q), _strides(grad_k),
                _strides(grad_v), _strides(grad_decay), _strides(grad_beta), ctx.scale, _native.dtype_code(beta.dtype),
                _native.current_stream(k.device))
        _native.check(status, "gated_delta_rule backward")
        return grad_q, grad_k, grad_v, grad_decay, grad_beta, None, None, None


def gated_delta_rule(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    log_decay: torch.Tensor,
    beta: torch.Tensor,
    *,
    scale: float | None = None,
    key_lengths: torch.Tensor | None = None,
    initial_state: torch.Tensor | None = None,
    return_state: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """The gated delta rule over ``q, k (batch, key heads, tokens, key width)``, ``v (batch, heads, tokens, value width)`` and the
    gates ``log_decay, beta (batch, heads, tokens)`` -> ``out (batch, heads, tokens, value width)``, whose memory order is
    (batch, tokens, heads, width).

    bfloat16 tokens, gates in bfloat16 or float32; widths that are multiples of 8, at most 128; value heads a multiple of the
    key heads (consecutive value heads share a key head). ``scale`` defaults to ``key width ** -0.5``. ``key_lengths`` (batch,):
    tokens at or beyond a sample's length are not read, get zeros and leave the state alone. Keys should have unit length at
    most (an :func:`rms_norm` over the head with weight ``key width ** -0.5``) and ``beta`` lie in [0, 1]; ``log_decay`` is normally
    below zero, and may have either sign as long as the sums of it within 64 tokens stay below 88 (``exp`` in float32). Infinities and NaN in a
    valid token reach every token of its chunk of 64, those in front of it too, and all behind it in the same sample and head.

    ``initial_state`` (batch, heads, key width, value width) float32 is the state in front of the first token, ``return_state``
    returns ``(out, state behind the last)``, which :func:`gated_delta_rule_step` continues. The state is kept in float32
    and everything that reaches it enters its products with 24 bits. Outputs and the gradient of v are rounded once, at the end
    (the outputs of keys wider than 64 also where the scores meet the values). The gradients of q, k and the gates, float32 gates
    among them, have the bfloat16 rounding of the states that the forward keeps in them, 1e-3 to 2.5e-3.

    Differentiable in q, k, v and the gates; the states are not, so that an ``initial_state`` that requires grad, and
    ``return_state`` where an input does, are refused."""
    name = "gated_delta_rule"
    _check_shapes(name, q, k, v, log_decay, beta)
    require_cuda_tensors(f"hip {name}", q, k, v, log_decay, beta, initial_state)
    _check_widths(name, k.shape[3], v.shape[3])
    if v.dtype != torch.bfloat16:
        raise RuntimeError(f"hip {name} does not support dtype {v.dtype}")
    if beta.dtype not in (torch.bfloat16, torch.float32):
        raise RuntimeError(f"hip {name} takes gates in bfloat16 or float32, got {beta.dtype}")
    lengths = _lengths(name, key_lengths, v.shape[0], v.device)
    if initial_state is not None:
        if initial_state.shape != (v.shape[0], v.shape[1], k.shape[3], v.shape[3]) or initial_state.dtype != torch.float32:
            raise ValueError(f"{name} initial_state must be float32 of shape (batch, heads, key width, value width)")
        require_inference(f"hip {name} initial_state", initial_state)
        initial_state = initial_state.contiguous()
    scale = k.shape[3] ** -0.5 if scale is None else float(scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or log_decay.requires_grad or beta.requires_grad):
        if return_state:
            raise RuntimeError(f"hip {name}: the returned state has no gradient: call it under torch.no_grad() or without return_state")
        return _GatedDeltaRuleFunction.apply(q, k, v, log_decay, beta, scale, lengths, initial_state)
    out, final, _, _ = _forward(_rows_view(q), _rows_view(k), _rows_view(v), log_decay, beta, scale, lengths, initial_state,
                                return_state, False)
    return (out, final) if return_state else out


def gated_delta_rule_step(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    log_decay: torch.Tensor,
    beta: torch.Tensor,
    state: torch.Tensor,
    *,
    scale: float | None = None,
    state_index: torch.Tensor | None = None,
    key_lengths: torch.Tensor | None = None,
) -> torch.Tensor:
    """One or a few new tokens of every sample: :func:`gated_delta_rule` on the same shapes, continuing states that are
    updated in place. ``state`` (slots, heads, key width, value width): contiguous float32; ``state_index`` (batch,) int32 or
    int64: the slot of each sample (without it sample b has slot b). Samples with the same slot are one sequence, their tokens
    applied in the order of the batch; an index outside the pool (-1 for a padded sample) touches no state and gives zeros.
    ``key_lengths`` (batch,): the tokens a sample really has, as in :func:`gated_delta_rule`. Tokens in float32, bfloat16 or
    float16, the gates in the same type or float32. Forward only."""
    name = "gated_delta_rule_step"
    _check_shapes(name, q, k, v, log_decay, beta)
    if state.ndim != 4 or state.shape[1:] != (v.shape[1], k.shape[3], v.shape[3]):
        raise ValueError(f"{name} expects a state of shape (slots, heads, key width, value width)")
    if state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError(f"{name} updates the state in place: it must be contiguous float32")
    batch, key_heads, tokens, key_width = k.shape
    if state_index is not None:
        if state_index.shape != (batch,) or state_index.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{name} state_index must hold one int32 or int64 per sample")
    elif batch > state.shape[0]:
        raise ValueError(f"{name}: {batch} samples without state_index and {state.shape[0]} slots")
    require_cuda_tensors(f"hip {name}", q, k, v, log_decay, beta, state, state_index)
    require_inference(f"hip {name}", q, k, v, log_decay, beta, state)
    _check_widths(name, key_width, v.shape[3])
    if beta.dtype not in (v.dtype, torch.float32):
        raise ValueError(f"{name} takes gates of the tokens' dtype or float32, got {beta.dtype}")
    lengths = _lengths(name, key_lengths, batch, v.device)
    q, k, v = (t if t.stride(-1) == 1 else t.contiguous() for t in (q, k, v))
    if state_index is not None:
        state_index = state_index.contiguous()
    scale = key_width ** -0.5 if scale is None else float(scale)
    out = _token_major(batch, v.shape[1], tokens, v.shape[3], v)
    library = _native.load_library()
    with _native.on_device(v.device):
        status = library.taac_delta_rule_step(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), beta.data_ptr(), state.data_ptr(), state.shape[0],
            _native.ptr(state_index), int(state_index is not None and state_index.dtype == torch.int64), _native.ptr(lengths),
            out.data_ptr(), batch, v.shape[1], key_heads, tokens, key_width, v.shape[3], _strides(q), _strides(k), _strides(v),
            _strides(out), _strides(log_decay), _strides(beta), scale, _native.dtype_code(v.dtype), _native.dtype_code(beta.dtype),
            _native.current_stream(v.device))
    _native.check(status, name)
    torch.autograd.graph.increment_version(state)
    return out


__all__ = ["gated_delta_rule", "gated_delta_rule_step"]
