"""RMSNorm of every head of the queries and keys with the rotation by their positions, in one pass (``taac_head_norm_rope_fwd`` / ``_bwd``).

:func:`qk_norm_rope` norms over the whole model width and rotates whole heads from position 0, as the reference's layers do
(experiments/tokenformer/model.py:149-192); here each head has its own norm, keys may have fewer heads than queries, a part of the head may be
rotated, in either pairing, and every sample or token stands at a position of its own, as serving event by event needs.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch
from torch.autograd.function import once_differentiable

from taac_2026_amd import _native
from taac_2026_amd.accelerators.tensor_validation import require_cuda_tensors, require_inference, require_no_tangents, require_same_dtype

MAX_HEAD_WIDTH = 512
MAX_COUNT = 2**31 - 1  # the library counts samples and tokens in 32 bits
_Strides3 = ctypes.c_int64 * 3
_Strides2 = ctypes.c_int64 * 2


@functools.lru_cache(maxsize=512)
def _strides3(batch: int, head: int, token: int, _: int) -> ctypes.Array:
    return _Strides3(batch, head, token)


def strides_of(t: torch.Tensor) -> ctypes.Array:
    """Of (batch, head, token), for the library to read. The arrays are kept by value: a serving program repeats a few."""
    return _strides3(*t.stride())


@functools.lru_cache(maxsize=64)
def _strides2(sample: int, token: int) -> ctypes.Array:
    return _Strides2(sample, token)


def token_major(shape: torch.Size, like: torch.Tensor, dtype: torch.dtype | None = None) -> torch.Tensor:
    """(batch, heads, tokens, width) whose memory order is (batch, tokens, heads, width): the rows of the layers around it."""
    batch, heads, tokens, width = shape
    row = heads * width
    return torch.empty_strided(shape, (tokens * row, width, row, 1), dtype=dtype or like.dtype, device=like.device)


def rotary_table(
    places: int,
    rotary_dim: int,
    base: float = 10000.0,
    *,
    factor: float = 1.0,
    trained_places: int | None = None,
    turns: tuple[float, float] = (1.0, 32.0),
    magnitude: float = 1.0,
    device: torch.device | str | None = None,
) -> torch.Tensor:
    """Float32 ``(places, rotary_dim / 2, 2)`` of ``magnitude (cos, sin)(position * frequency)`` with ``frequency_i = base ** (-2 i / rotary_dim)``, angles in 64
    bits, for :func:`head_norm_rope`, on ``device`` (torch's default).

    ``factor`` stretches positions for contexts longer than those a model was trained on: alone it divides every frequency. With ``trained_places``
    it does so by parts: frequencies that turn at most ``turns[0]`` times within them are divided, those that turn at least ``turns[1]`` times are kept, and the ones
    between are mixed in proportion. ``magnitude`` scales queries and keys alike, as some models do for long contexts."""
    places, rotary_dim = int(places), int(rotary_dim)
    if places < 0 or rotary_dim <= 0 or rotary_dim % 2 != 0:
        raise ValueError("rotary_table needs a number of places that is not negative and an even number of rotated features above zero")
    if not (base > 0.0 and factor > 0.0) or not math.isfinite(base) or not math.isfinite(factor):
        raise ValueError("rotary_table needs base and factor above zero")
    device = torch.get_default_device() if device is None else device
    frequencies = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device="cpu") / rotary_dim)
    if trained_places is None:
        frequencies = frequencies / factor
    else:
        low, high = turns
        if trained_places <= 0 or not low < high:
            raise ValueError("rotary_table needs trained_places above zero and turns in ascending order")
        kept = ((trained_places / (2.0 * math.pi) * frequencies - low) / (high - low)).clamp(0.0, 1.0)
        frequencies = frequencies * (kept + (1.0 - kept) / factor)
    angles = torch.arange(places, dtype=torch.float64, device=device)[:, None] * frequencies.to(device)
    return (magnitude * torch.stack((angles.cos(), angles.sin()), -1)).float()


def _arguments(q, k, q_out, k_out, weights, eps, table, places, interleaved):
    """The common arguments of both directions, from the sizes to the flags, in two halves around the strides of the gradients. ``places``: the positions'
    tensor or None, its strides for (sample, token), and whether the token's number is added."""
    positions, position_strides, add_token = places
    batch, heads, tokens, width = q.shape
    return (
        (batch, heads, k.shape[1], tokens, width, 0 if table is None else 2 * table.shape[1], strides_of(q), strides_of(k)),
        (strides_of(q_out), strides_of(k_out), _native.ptr(weights[0]), _native.ptr(weights[1]), eps, _native.ptr(table),
         0 if table is None else table.shape[0], _native.ptr(positions), positions is not None and positions.dtype == torch.int64, position_strides,
         add_token, interleaved, _native.dtype_code(q.dtype), _native.current_stream(q.device)),
    )


def _forward(q, k, weights, eps, table, places, interleaved):
    q_out, k_out = token_major(q.shape, q), token_major(k.shape, k)
    sizes, rest = _arguments(q, k, q_out, k_out, weights, eps, table, places, interleaved)
    library = _native.load_library()
    with _native.on_device(q.device):
        status = library.taac_head_norm_rope_fwd(q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), *sizes, *rest)
    _native.check(status, "head_norm_rope")
    return q_out, k_out


class _HeadNormRopeFunction(torch.autograd.Function):
    """Keeps the inputs; the backward makes each row's statistic again."""

    @staticmethod
    def forward(ctx, q, k, query_weight, key_weight, eps, table, positions, position_strides, add_token, interleaved):
        ctx.save_for_backward(*((q, k) if query_weight is not None else (None, None)), query_weight, key_weight, table, positions)
        ctx.options = eps, position_strides, add_token, interleaved
        return _forward(q, k, (query_weight, key_weight), eps, table, (positions, position_strides, add_token), interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_q_out, grad_k_out):
        q, k, query_weight, key_weight, table, positions = ctx.saved_tensors
        eps, position_strides, add_token, interleaved = ctx.options
        grad_q_out, grad_k_out = _rows(grad_q_out), _rows(grad_k_out)
        if q is None:  # a rotation alone does not read them
            q, k = grad_q_out, grad_k_out
        grad_q, grad_k = token_major(q.shape, q), token_major(k.shape, k)
        grad_weights, workspace, floats = (None, None), None, 0
        library = _native.load_library()
        if query_weight is not None:
            grad_weights = torch.empty_like(query_weight), torch.empty_like(key_weight)
            floats = library.taac_head_norm_rope_bwd_workspace_floats(q.shape[0], q.shape[1], k.shape[1], q.shape[2], q.shape[3])
            workspace = q.new_empty(floats, dtype=torch.float32)
        sizes, rest = _arguments(q, k, grad_q, grad_k, (query_weight, key_weight), eps, table, (positions, position_strides, add_token), interleaved)
        with _native.on_device(q.device):
            status = library.taac_head_norm_rope_bwd(
                q.data_ptr(), k.data_ptr(), grad_q_out.data_ptr(), grad_k_out.data_ptr(), grad_q.data_ptr(), grad_k.data_ptr(),
                _native.ptr(grad_weights[0]), _native.ptr(grad_weights[1]), _native.ptr(workspace), floats, *sizes,
                strides_of(grad_q_out), strides_of(grad_k_out), *rest)
        _native.check(status, "head_norm_rope backward")
        return grad_q, grad_k, *grad_weights, None, None, None, None, None, None


def _weight(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    return t if t.dtype == dtype and t.stride(0) == 1 else t.to(dtype).contiguous()


def _rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 else t.contiguous()


def head_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    query_weight: torch.Tensor | None = None,
    key_weight: torch.Tensor | None = None,
    *,
    eps: float = 1e-6,
    table: torch.Tensor | None = None,
    starts: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``q (batch, heads, tokens, width)`` and ``k (batch, key heads, tokens, width)`` normed and rotated, as new tensors whose memory order is
    (batch, tokens, heads, width).

    With weights ``(width,)`` (both or neither) every head becomes ``x rsqrt(mean(x^2) + eps) weight``. ``table`` (:func:`rotary_table`; float32
    ``(places, rotated / 2, 2)``) then rotates the first ``rotated`` features, in pairs ``(i, i + rotated / 2)`` or, ``interleaved``, ``(2 i, 2 i + 1)``, by the row of
    the token's position: its number, plus its sample's ``starts (batch,)``, or ``positions`` of shape (tokens,) or (batch, tokens). Both are int32 or
    int64; the rotated features of a token at a position that the table does not have come out as NaN.

    float32, bfloat16 or float16; a head has at most 512 features. Arithmetic in float32, rounded once. Differentiable in q, k and the
    weights, backwards; dual tensors are refused."""
    name = "head_norm_rope"
    q_shape, k_shape = q.shape, k.shape
    if len(q_shape) != 4 or len(k_shape) != 4:
        raise ValueError(f"{name} expects q and k with shape (batch, heads, tokens, width)")
    batch, heads, tokens, width = q_shape
    if batch != k_shape[0] or tokens != k_shape[2] or width != k_shape[3] or heads == 0 or k_shape[1] == 0 or width == 0:
        raise ValueError(f"{name} requires matching batch, tokens and width of q and k, got {tuple(q_shape)} and {tuple(k_shape)}")
    if q.dtype != k.dtype:
        require_same_dtype(f"{name} q, k", q, k)
    if (query_weight is None) != (key_weight is None):
        raise ValueError(f"{name} takes both norm weights or neither")
    if query_weight is None and table is None:
        raise ValueError(f"{name} needs norm weights, a table, or both")
    if query_weight is not None and (query_weight.shape != (width,) or key_weight.shape != (width,)):
        raise ValueError(f"{name} weights must hold one value per feature of a head")
    if not eps >= 0.0:
        raise ValueError(f"{name} eps must not be negative")
    if starts is not None and positions is not None:
        raise ValueError(f"{name} takes starts or positions, not both")
    place = starts if starts is not None else positions
    if place is not None:
        if table is None:
            raise ValueError(f"{name}: positions come with a table")
        if place.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{name} positions must be int32 or int64, got {place.dtype}")
        if starts is not None and place.shape != (batch,):
            raise ValueError(f"{name} starts must hold one position per sample")
        if positions is not None and place.shape not in ((tokens,), (batch, tokens)):
            raise ValueError(f"{name} positions must have shape (tokens,) or (batch, tokens)")
    if table is not None:
        if table.ndim != 3 or table.shape[2] != 2 or table.shape[1] == 0 or 2 * table.shape[1] > width:
            raise ValueError(f"{name} expects a table of shape (places, rotated / 2, 2) with at most the head's features")
        if table.dtype != torch.float32 or not table.is_contiguous():
            raise ValueError(f"{name} table must be contiguous float32")
    require_no_tangents(f"hip {name}", q, k, query_weight, key_weight, table)
    require_cuda_tensors(f"hip {name}", q, k, query_weight, key_weight, table, place)
    if q.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise RuntimeError(f"hip {name} does not support dtype {q.dtype}")
    if width > MAX_HEAD_WIDTH or batch > MAX_COUNT or tokens > MAX_COUNT:
        raise RuntimeError(f"hip {name} is built for heads of at most {MAX_HEAD_WIDTH} features, samples and tokens of at most 2^31 - 1")
    if table is not None and table.requires_grad:
        require_inference(f"hip {name} table", table)
    if query_weight is not None:
        query_weight, key_weight = _weight(query_weight, q.dtype), _weight(key_weight, q.dtype)
    position_strides = None
    if place is not None:
        strides = place.stride()
        position_strides = _strides2(strides[0], 0) if starts is not None else _strides2(*((0, *strides)[-2:]))
    q, k = _rows(q), _rows(k)
    eps, interleaved, add_token = float(eps), bool(interleaved), starts is not None
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or (query_weight is not None and (query_weight.requires_grad or key_weight.requires_grad))):
        return _HeadNormRopeFunction.apply(q, k, query_weight, key_weight, eps, table, place, position_strides, add_token, interleaved)
    return _forward(q, k, (query_weight, key_weight), eps, table, (place, position_strides, add_token), interleaved)


__all__ = ["head_norm_rope", "rotary_table"]
