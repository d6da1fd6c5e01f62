"""The gated delta rule token by token in 64 bits, with the magnitudes that error bounds are made of. Tensors on the CPU, laid out
(batch, heads, tokens, width)."""

from __future__ import annotations

import torch


def delta_rule(q, k, v, log_decay, beta, *, scale=None, lengths=None, initial_state=None):
    """``(out, state, misses)`` of ``S <- a S; S <- S + k (beta (v - S^T k))^T; o = scale S^T q``; misses are ``v - S^T k``.
    Differentiable. Tokens at or beyond a sample's length are left out and have zeros."""
    group = v.shape[1] // q.shape[1]
    scale = k.shape[-1] ** -0.5 if scale is None else scale
    q, k = (t.double().repeat_interleave(group, 1) for t in (q, k))
    v, decay, beta = v.double(), log_decay.double().exp(), beta.double()
    batch, heads, tokens, _ = v.shape
    lengths = [tokens] * batch if lengths is None else [min(max(int(n), 0), tokens) for n in lengths]
    outs, finals, misses = [], [], []
    for b in range(batch):
        state = torch.zeros(heads, k.shape[-1], v.shape[-1], dtype=torch.float64)
        if initial_state is not None:
            state = initial_state[b].double()
        out, miss = [], []
        for t in range(lengths[b]):
            state = decay[b, :, t, None, None] * state
            m = v[b, :, t] - (k[b, :, t, :, None] * state).sum(1)
            state = state + k[b, :, t, :, None] * (beta[b, :, t, None] * m)[:, None]
            out.append(scale * (q[b, :, t, :, None] * state).sum(1))
            miss.append(m)
        pad = [torch.zeros(heads, v.shape[-1], dtype=torch.float64)] * (tokens - lengths[b])
        outs.append(torch.stack(out + pad, 1) if tokens else v[b])
        misses.append(torch.stack(miss + pad, 1) if tokens else v[b])
        finals.append(state)
    return torch.stack(outs), torch.stack(finals), torch.stack(misses)


def score_magnitudes(q, k, log_decay, beta, misses, *, scale=None):
    """``|P| |N|`` with ``P_ij = scale exp(G_i - G_j) (q_i . k_j) beta_j`` over all pairs j <= i: what one rounding of every P adds up to."""
    group = misses.shape[1] // q.shape[1]
    scale = k.shape[-1] ** -0.5 if scale is None else scale
    q, k = (t.double().repeat_interleave(group, 1) for t in (q, k))
    total = log_decay.double().clamp(min=-1e5).cumsum(-1)
    pairs = (q @ k.transpose(-1, -2)).abs() * (total[..., :, None] - total[..., None, :]).clamp(max=0.0).exp() * beta.double().abs()[..., None, :]
    return scale * pairs.tril() @ misses.abs()
