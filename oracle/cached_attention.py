"""Per-head norm and rotation, the quantised cache's values and attention over them, in 64 bits, with the magnitudes that error bounds are made of. Tensors
laid out (batch, heads, tokens, width), on any device."""

from __future__ import annotations

import math

import torch


def rotation_angles(positions: torch.Tensor, rotary: int, base: float = 10000.0) -> torch.Tensor:
    """(..., rotary / 2) angles of integer positions."""
    return positions.double()[..., None] * base ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=positions.device) / rotary)


def _pairs(rotary: int, interleaved: bool) -> tuple[torch.Tensor, torch.Tensor]:
    i = torch.arange(rotary // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)


def head_norm_rope(x, weight, angles, *, eps=1e-6, interleaved=False, magnitude=False):
    """One of queries and keys; ``angles`` (batch or 1, tokens, pairs) or None. Differentiable. ``magnitude``: |a c| + |b s| in the place of every
    feature."""
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    if magnitude:
        y = y.abs()
    if angles is None:
        return y
    a, b = _pairs(2 * angles.shape[-1], interleaved)
    cos, sin = angles.cos()[:, None], angles.sin()[:, None]
    if magnitude:
        cos, sin, minus = cos.abs(), sin.abs(), 1.0
    else:
        minus = -1.0
    out = y.clone()
    out[..., a] = y[..., a] * cos + minus * y[..., b] * sin
    out[..., b] = y[..., a] * sin + y[..., b] * cos
    return out


def _grid(bits: int, device) -> torch.Tensor:
    if bits == 4:
        return torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=device)
    code = torch.arange(127, device=device)
    fraction, power = (code % 8).double() / 8.0, code // 8
    return torch.where(power == 0, fraction * 2.0**-6, torch.exp2(power.double() - 7.0) * (1.0 + fraction))


def cached_values(x, bits: int):
    """What a cache of 4 or 8 bits holds of finite ``x``: codes of the grid, nearest, ties to the even one, times the least power of two with which the largest
    of 32 features stays below 7 (464)."""
    grid = _grid(bits, x.device)
    blocks = x.double().unflatten(-1, (-1, 32))
    limit, least, most = (7.0, -117, 125) if bits == 4 else (464.0, -117, 119)
    exponent = torch.floor(torch.log2(blocks.abs().amax(-1, keepdim=True) / limit)) + 1.0
    scale = torch.exp2(exponent.clamp(least, most))
    size = (blocks / scale).abs()
    upper = torch.searchsorted(grid, size.contiguous()).clamp(1, len(grid) - 1)
    to_low, to_high = size - grid[upper - 1], grid[upper] - size
    down = (to_low < to_high) | ((to_low == to_high) & ((upper - 1) % 2 == 0))
    return (torch.copysign(torch.where(down, grid[upper - 1], grid[upper]), blocks) * scale).flatten(-2)


def visible(lengths, query_lengths, tokens: int, cached: int, window=None):
    """(batch, tokens, cached): the positions that a query sees."""
    place = (lengths - query_lengths).long()[:, None] + torch.arange(tokens, device=lengths.device)
    position = torch.arange(cached, device=lengths.device)
    seen = (position <= place[..., None]) & (torch.arange(tokens, device=lengths.device) < query_lengths[:, None])[..., None]
    if window is not None:
        seen &= position > place[..., None] - window
    return seen


def attention(q, k, v, seen, scale=None):
    """``(out, sum of p |v|, largest sum of |scale q k| of a visible pair)`` over visible pairs ``seen`` (batch, tokens, cached); rows that see nothing are zeros."""
    group = q.shape[1] // k.shape[1]
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    q, k, v = q.double(), (k.double().repeat_interleave(group, 1)), (v.double().repeat_interleave(group, 1))
    seen = seen[:, None]
    scores = torch.where(seen, scale * (q @ k.transpose(-1, -2)), -torch.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -torch.inf, 0.0, top))
    total = weights.sum(-1, keepdim=True)
    weights = torch.where(total > 0, weights / total, 0.0)
    sizes = torch.where(seen, abs(scale) * (q.abs() @ k.abs().transpose(-1, -2)), 0.0)
    largest = sizes.amax(-1) if sizes.shape[-1] else sizes.new_zeros(sizes.shape[:-1])
    return weights @ v, weights @ v.abs(), largest
