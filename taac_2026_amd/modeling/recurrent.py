"""A token mixer with a state of fixed size, and the block around it: peers of the attention modules for histories that grow event by
event. A history is taken in chunks (:func:`gated_delta_rule`), and each new event costs one step on the user's state
(:func:`gated_delta_rule_step`), however long the history is."""

from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from taac_2026_amd.accelerators.delta_rule import MAX_WIDTH, gated_delta_rule, gated_delta_rule_step
from taac_2026_amd.accelerators.linear import linear, linear_fp8, quantize_fp8
from taac_2026_amd.accelerators.normalization import residual_rms_norm, residual_rms_norm_fp8, rms_norm
from taac_2026_amd.modeling.backbone import SwiGLUFeedForward
from taac_2026_amd.modeling.normalization import RMSNorm


class GatedDeltaAttention(nn.Module):
    """One projection to queries, keys, values and the gates -> queries and keys of unit length per head -> gated delta rule -> out
    projection, in bfloat16 with gates in float32. ``log_decay = -exp(decay_rate) softplus(gate + decay_bias)`` and
    ``beta = sigmoid(gate)`` per value head. ``key_heads`` (a divisor of ``num_heads``) are shared by consecutive value heads."""

    def __init__(self, d_model: int, num_heads: int, *, key_heads: int | None = None, key_width: int | None = None,
                 value_width: int | None = None) -> None:
        super().__init__()
        self.num_heads = int(num_heads)
        self.key_heads = self.num_heads if key_heads is None else int(key_heads)
        if self.key_heads <= 0 or self.num_heads % self.key_heads != 0:
            raise ValueError("GatedDeltaAttention requires a number of value heads that is a multiple of the key heads")
        self.key_width = d_model // self.num_heads if key_width is None else int(key_width)
        self.value_width = d_model // self.num_heads if value_width is None else int(value_width)
        for width in (self.key_width, self.value_width):
            if width <= 0 or width % 8 != 0 or width > MAX_WIDTH:
                raise ValueError(f"GatedDeltaAttention is built for key and value widths that are multiples of 8, at most {MAX_WIDTH}")
        keys, values = self.key_heads * self.key_width, self.num_heads * self.value_width
        self.sizes = (keys, keys, values, self.num_heads, self.num_heads)
        self.inputs = nn.Linear(d_model, -(-sum(self.sizes) // 8) * 8)  # dense layers come in multiples of eight features
        self.decay_rate = nn.Parameter(torch.empty(self.num_heads).uniform_(1.0, 16.0).log_())
        step = torch.empty(self.num_heads).uniform_(-6.9, -2.3).exp_()  # first decays of exp(-rate step)
        self.decay_bias = nn.Parameter(torch.log(torch.expm1(step)))
        self.out = nn.Linear(values, d_model)

    def empty_state(self, slots: int, device: torch.device | str) -> torch.Tensor:
        """A pool of ``slots`` states in front of a first token, float32 as the steps take them."""
        return torch.zeros(slots, self.num_heads, self.key_width, self.value_width, dtype=torch.float32, device=device)

    def _project(self, tokens: torch.Tensor) -> tuple[torch.Tensor, ...]:
        batch, count, _ = tokens.shape
        rows = linear(tokens, self.inputs.weight.to(tokens.dtype), self.inputs.bias.to(tokens.dtype))
        q, k, v, decay, beta = rows[..., : sum(self.sizes)].split(self.sizes, -1)
        # rows of length sqrt(width) from the norm, of length one with this weight
        unit = torch.full((self.key_width,), self.key_width ** -0.5, dtype=tokens.dtype, device=tokens.device)
        q, k = (rms_norm(t.reshape(batch, count, self.key_heads, self.key_width), unit).transpose(1, 2) for t in (q, k))
        v = v.unflatten(-1, (self.num_heads, self.value_width)).transpose(1, 2)
        log_decay = -self.decay_rate.float().exp() * F.softplus(decay.float() + self.decay_bias.float())
        return q, k, v, log_decay.transpose(1, 2), torch.sigmoid(beta.float()).transpose(1, 2)

    def _leave(self, mixed: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
        rows = mixed.transpose(1, 2).flatten(2)
        return linear(rows, self.out.weight.to(rows.dtype), self.out.bias.to(rows.dtype)).to(dtype)

    def forward(self, tokens: torch.Tensor, *, key_lengths: torch.Tensor | None = None) -> torch.Tensor:
        """(B, T, D) -> (B, T, D). Rows at or beyond a sample's length hold the out projection's bias."""
        return self._leave(gated_delta_rule(*self._project(tokens.to(torch.bfloat16)), key_lengths=key_lengths), tokens.dtype)

    def prefill(self, tokens: torch.Tensor, *, key_lengths: torch.Tensor | None = None, initial_state: torch.Tensor | None = None
                ) -> tuple[torch.Tensor, torch.Tensor]:
        """:meth:`forward` and the state (B, heads, key width, value width) behind each sample's last token. Forward only."""
        mixed, state = gated_delta_rule(*self._project(tokens.to(torch.bfloat16)), key_lengths=key_lengths,
                                        initial_state=initial_state, return_state=True)
        return self._leave(mixed, tokens.dtype), state

    def step(self, tokens: torch.Tensor, state: torch.Tensor, *, state_index: torch.Tensor | None = None,
             key_lengths: torch.Tensor | None = None) -> torch.Tensor:
        """The next tokens (B, t, D) of sequences whose states lie in a pool, which is updated in place. Forward only."""
        mixed = gated_delta_rule_step(*self._project(tokens.to(torch.bfloat16)), state, state_index=state_index,
                                      key_lengths=key_lengths)
        return self._leave(mixed, tokens.dtype)


class GatedDeltaBlock(nn.Module):
    """Pre-norm :class:`GatedDeltaAttention` and SwiGLU feed-forward with residuals; the first residual's addition and the norm in front
    of the feed-forward are one pass. No valid row reads a padded one; what padded rows hold is not specified."""

    def __init__(self, d_model: int, num_heads: int, hidden_mult: int, *, key_heads: int | None = None, key_width: int | None = None,
                 value_width: int | None = None) -> None:
        super().__init__()
        self.attn_norm = RMSNorm(d_model)
        self.attention = GatedDeltaAttention(d_model, num_heads, key_heads=key_heads, key_width=key_width, value_width=value_width)
        self.ffn_norm = RMSNorm(d_model)
        self.ffn = SwiGLUFeedForward(d_model, hidden_mult)

    def fp8_weights(self) -> tuple[torch.Tensor, torch.Tensor]:
        """The feed-forward's up projection as e4m3 and its maximum, for the caller to keep while the weights stay."""
        return quantize_fp8(self.ffn.up.weight.detach().to(torch.bfloat16))

    def _feed_forward(self, update: torch.Tensor, tokens: torch.Tensor, fp8_weights: tuple[torch.Tensor, torch.Tensor] | None
                      ) -> torch.Tensor:
        weight = self.ffn_norm.weight.to(tokens.dtype)
        if fp8_weights is None:
            normed, summed = residual_rms_norm(update, tokens, weight, self.ffn_norm.eps)
            return self.ffn(normed, residual=summed)
        values, row_amax, summed = residual_rms_norm_fp8(update, tokens, weight, self.ffn_norm.eps)
        dtype = tokens.dtype
        hidden = linear_fp8(values, fp8_weights[0], row_amax, fp8_weights[1], self.ffn.up.bias.to(dtype), swiglu=True,
                            gate_first=self.ffn.gate_first)
        return linear(hidden, self.ffn.down.weight.to(dtype), self.ffn.down.bias.to(dtype), residual=summed)

    def forward(self, tokens: torch.Tensor, *, key_lengths: torch.Tensor | None = None,
                fp8_weights: tuple[torch.Tensor, torch.Tensor] | None = None) -> torch.Tensor:
        """(B, T, D) -> (B, T, D) in bfloat16. ``fp8_weights`` (:meth:`fp8_weights`): the up projection runs on e4m3 operands, forward
        only."""
        tokens = tokens.to(torch.bfloat16)
        return self._feed_forward(self.attention(self.attn_norm(tokens), key_lengths=key_lengths), tokens, fp8_weights)

    def prefill(self, tokens: torch.Tensor, *, key_lengths: torch.Tensor | None = None, initial_state: torch.Tensor | None = None,
                fp8_weights: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        tokens = tokens.to(torch.bfloat16)
        update, state = self.attention.prefill(self.attn_norm(tokens), key_lengths=key_lengths, initial_state=initial_state)
        return self._feed_forward(update, tokens, fp8_weights), state

    def step(self, tokens: torch.Tensor, state: torch.Tensor, *, state_index: torch.Tensor | None = None,
             key_lengths: torch.Tensor | None = None, fp8_weights: tuple[torch.Tensor, torch.Tensor] | None = None) -> torch.Tensor:
        tokens = tokens.to(torch.bfloat16)
        update = self.attention.step(self.attn_norm(tokens), state, state_index=state_index, key_lengths=key_lengths)
        return self._feed_forward(update, tokens, fp8_weights)


__all__ = ["GatedDeltaAttention", "GatedDeltaBlock"]
