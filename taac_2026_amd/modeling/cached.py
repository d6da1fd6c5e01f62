"""Softmax attention for histories that grow event by event, over a quantised cache of keys and values, and the block around it: the peer of
:class:`GatedDeltaAttention`, whose state has a fixed size, for models that attend to every event."""

from __future__ import annotations

import torch
import torch.nn as nn

from taac_2026_amd.accelerators.attention import flash_attention
from taac_2026_amd.accelerators.head_rope import head_norm_rope, rotary_table
from taac_2026_amd.accelerators.kv_cache import CACHED_WIDTHS, KVCache, cached_attention, empty_kv_cache, kv_cache_write
from taac_2026_amd.accelerators.linear import linear
from taac_2026_amd.modeling.recurrent import PreNormBlock


class CachedAttention(nn.Module):
    """One projection to queries, keys and values -> RMSNorm of every head of queries and keys and the rotation by their positions -> causal attention -> out
    projection, in bfloat16. ``key_heads`` (a divisor of ``num_heads``) are shared by consecutive query heads; ``rotary_dim`` features of a head are rotated
    (default: all), for positions below ``max_tokens``; ``rotary_options`` go to :func:`rotary_table`. Training takes heads of at most 64 features, as the backward of
    :func:`flash_attention` does."""

    def __init__(self, d_model: int, num_heads: int, *, key_heads: int | None = None, head_dim: int | None = None, rotary_dim: int | None = None,
                 max_tokens: int = 4096, interleaved: bool = False, rotary_options: dict | None = None) -> None:
        super().__init__()
        self.num_heads = int(num_heads)
        self.key_heads = self.num_heads if key_heads is None else int(key_heads)
        if self.key_heads <= 0 or self.num_heads % self.key_heads != 0:
            raise ValueError("CachedAttention requires a number of heads that is a multiple of the key heads")
        self.head_dim = d_model // self.num_heads if head_dim is None else int(head_dim)
        if self.head_dim not in CACHED_WIDTHS:
            raise ValueError(f"CachedAttention is built for heads of {', '.join(map(str, CACHED_WIDTHS))} features, got {self.head_dim}")
        self.max_tokens, self.interleaved = int(max_tokens), bool(interleaved)
        self._rotary = (self.max_tokens, self.head_dim if rotary_dim is None else int(rotary_dim)), dict(rotary_options or {})
        self.inputs = nn.Linear(d_model, (self.num_heads + 2 * self.key_heads) * self.head_dim)
        self.query_weight, self.key_weight = (nn.Parameter(torch.ones(self.head_dim)) for _ in range(2))
        self.out = nn.Linear(self.num_heads * self.head_dim, d_model)
        self.register_buffer("table", rotary_table(*self._rotary[0], **self._rotary[1]), persistent=False)

    def _apply(self, fn, recurse: bool = True):
        kept = self.table
        super()._apply(fn, recurse)
        # Only the device follows: angles of far positions keep their digits whatever type the weights take, and a table is no part of a state that is loaded
        # into room without data.
        device = self.table.device
        self.table = rotary_table(*self._rotary[0], **self._rotary[1], device=device) if kept.is_meta and device.type != "meta" else kept.to(device)
        return self

    def empty_cache(self, pages: int, device: torch.device | str, *, bits: int = 4, page_tokens: int = 64) -> KVCache:
        """A pool of ``pages`` pages for the keys and values of this layer."""
        return empty_kv_cache(pages, self.key_heads, self.head_dim, bits=bits, page_tokens=page_tokens, device=device)

    def _project(self, tokens: torch.Tensor, starts: torch.Tensor | None = None) -> tuple[torch.Tensor, ...]:
        rows = linear(tokens, self.inputs.weight.to(tokens.dtype), self.inputs.bias.to(tokens.dtype))
        q, k, v = (t.transpose(1, 2) for t in rows.unflatten(-1, (-1, self.head_dim)).split((self.num_heads, self.key_heads, self.key_heads), 2))
        return *head_norm_rope(q, k, self.query_weight, self.key_weight, table=self.table, starts=starts, interleaved=self.interleaved), v

    def _require_positions(self, tokens: int) -> None:
        if tokens > self.max_tokens:
            raise ValueError(f"CachedAttention has positions for {self.max_tokens} tokens, got {tokens}")

    def _attend(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, key_lengths: torch.Tensor | None) -> torch.Tensor:
        self._require_positions(q.shape[2])
        group = self.num_heads // self.key_heads
        if group > 1:
            k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        if key_lengths is not None:
            key_lengths = key_lengths.to(torch.int32).contiguous()
        return flash_attention(q, k, v, key_lengths=key_lengths, is_causal=True, zero_padded_queries=key_lengths is not None)

    def _leave(self, mixed: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
        rows = mixed.transpose(1, 2).flatten(2)
        return linear(rows, self.out.weight.to(rows.dtype), self.out.bias.to(rows.dtype)).to(dtype)

    def forward(self, tokens: torch.Tensor, *, key_lengths: torch.Tensor | None = None) -> torch.Tensor:
        """(B, T, D) -> (B, T, D). Rows at or beyond a sample's length hold the out projection's bias."""
        return self._leave(self._attend(*self._project(tokens.to(torch.bfloat16)), key_lengths), tokens.dtype)

    def prefill(self, tokens: torch.Tensor, cache: KVCache, pages: torch.Tensor, *, key_lengths: torch.Tensor | None = None) -> torch.Tensor:
        """:meth:`forward` of histories that begin here, whose keys and values go into the cache's ``pages (B, pages of a sample)``. Forward only."""
        self._require_positions(tokens.shape[1])  # before anything is written
        q, k, v = self._project(tokens.to(torch.bfloat16))
        kv_cache_write(cache, k, v, pages, lengths=key_lengths)
        return self._leave(self._attend(q, k, v, key_lengths), tokens.dtype)

    def step(self, tokens: torch.Tensor, cache: KVCache, pages: torch.Tensor, starts: torch.Tensor, *, key_lengths: torch.Tensor | None = None) -> torch.Tensor:
        """The next tokens (B, t, D) of sequences that have ``starts (B,)`` tokens in the cache, to which these are added. Forward only."""
        if key_lengths is not None:
            key_lengths = key_lengths.clamp(0, tokens.shape[1])
        lengths = starts + (tokens.shape[1] if key_lengths is None else key_lengths)
        q, k, v = self._project(tokens.to(torch.bfloat16), starts)
        kv_cache_write(cache, k, v, pages, starts, lengths=key_lengths)
        return self._leave(cached_attention(q, cache, pages, lengths, query_lengths=key_lengths), tokens.dtype)


class CachedAttentionBlock(PreNormBlock):
    """Pre-norm :class:`CachedAttention` and SwiGLU feed-forward with residuals. No valid row reads a padded one; what padded rows hold is not specified."""

    def __init__(self, d_model: int, num_heads: int, hidden_mult: int, **options) -> None:
        super().__init__(d_model, CachedAttention(d_model, num_heads, **options), hidden_mult)

    def forward(self, tokens: torch.Tensor, *, key_lengths: torch.Tensor | None = None,
                fp8_weights: tuple[torch.Tensor, torch.Tensor] | None = None) -> torch.Tensor:
        """(B, T, D) -> (B, T, D) in bfloat16. ``fp8_weights`` (:meth:`fp8_weights`): the up projection runs on e4m3 operands, forward only."""
        tokens = tokens.to(torch.bfloat16)
        return self._feed_forward(self.attention(self.attn_norm(tokens), key_lengths=key_lengths), tokens, fp8_weights)

    def prefill(self, tokens: torch.Tensor, cache: KVCache, pages: torch.Tensor, *, key_lengths: torch.Tensor | None = None,
                fp8_weights: tuple[torch.Tensor, torch.Tensor] | None = None) -> torch.Tensor:
        tokens = tokens.to(torch.bfloat16)
        return self._feed_forward(self.attention.prefill(self.attn_norm(tokens), cache, pages, key_lengths=key_lengths), tokens, fp8_weights)

    def step(self, tokens: torch.Tensor, cache: KVCache, pages: torch.Tensor, starts: torch.Tensor, *, key_lengths: torch.Tensor | None = None,
             fp8_weights: tuple[torch.Tensor, torch.Tensor] | None = None) -> torch.Tensor:
        tokens = tokens.to(torch.bfloat16)
        return self._feed_forward(self.attention.step(self.attn_norm(tokens), cache, pages, starts, key_lengths=key_lengths), tokens, fp8_weights)


__all__ = ["CachedAttention", "CachedAttentionBlock"]
