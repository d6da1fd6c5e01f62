"""The gated delta rule token by token in 64 bits, with the magnitudes that error bounds are made of. Tensors laid out (batch, heads, tokens,
width), on any device."""

from __future__ import annotations

import torch


def delta_rule(q, k, v, log_decay, beta, *, scale=None, lengths=None, initial_state=None):
    """``(out, state, misses)`` of ``S <- a S; S <- S + k (beta (v - S^T k))^T; o = scale S^T q``; misses are ``v - S^T k``.
    Differentiable. Tokens at or beyond a sample's length are left out and have zeros."""
    group = v.shape[1] // q.shape[1]
    scale = k.shape[-1] ** -0.5 if scale is None else scale
    q, k = (t.double().repeat_interleave(group, 1) for t in (q, k))
    v, decay, beta = v.double(), log_decay.double().exp(), beta.double()
    batch, heads, tokens, width = v.shape
    state = torch.zeros(batch, heads, k.shape[-1], width, dtype=torch.float64, device=v.device)
    if initial_state is not None:
        state = initial_state.double()
    if lengths is not None:
        lengths = torch.as_tensor(lengths, device=v.device).clamp(0, tokens)
    outs, misses = [], []
    for t in range(tokens):
        decayed = decay[:, :, t, None, None] * state
        miss = v[:, :, t] - (k[:, :, t, :, None] * decayed).sum(2)
        updated = decayed + k[:, :, t, :, None] * (beta[:, :, t, None] * miss)[:, :, None]
        out = scale * (q[:, :, t, :, None] * updated).sum(2)
        if lengths is not None:
            live = (t < lengths)[:, None, None]
            out, miss = torch.where(live, out, 0.0), torch.where(live, miss, 0.0)
            updated = torch.where(live[..., None], updated, state)
        state = updated
        outs.append(out)
        misses.append(miss)
    if tokens == 0:
        return v, state, v
    return torch.stack(outs, 2), state, torch.stack(misses, 2)


def _pair_decays(log_decay):
    """``exp(G_i - G_j)`` of the pairs j <= i, zero above."""
    total = log_decay.detach().double().clamp(min=-1e5).cumsum(-1)
    above = torch.ones(total.shape[-1], total.shape[-1], dtype=torch.bool, device=total.device).triu(1)
    return (total[..., :, None] - total[..., None, :]).masked_fill(above, -torch.inf).exp()


def score_magnitudes(q, k, log_decay, beta, misses, *, scale=None):
    """``|P| |N|`` with ``P_ij = scale exp(G_i - G_j) (q_i . k_j) beta_j`` over all pairs j <= i: what one rounding of every P adds up to."""
    group = misses.shape[1] // q.shape[1]
    scale = k.shape[-1] ** -0.5 if scale is None else scale
    q, k = (t.double().repeat_interleave(group, 1) for t in (q, k))
    pairs = (q @ k.transpose(-1, -2)).abs() * _pair_decays(log_decay) * beta.double().abs()[..., None, :]
    return scale * pairs @ misses.abs()


def gradient_magnitudes(q, k, log_decay, beta, misses, grad_out, grad_v, *, scale=None, initial_state=None):
    """For every gradient (q, k, v, log_decay, beta) the sum of the absolute values of the products that it is the sum of, over all pairs of
    tokens: with W_ij = exp(G_i - G_j) beta_j and dX = dv,
      dq_i = scale sum_j W_ij (dO_i . N_j) k_j,           dk_j gets scale sum_i W_ij (dO_i . N_j) q_i - sum_i W_ij (dX_i . N_j) k_i,
      dk_i gets -sum_j W_ij (dX_i . N_j) k_j,              dX = P^T dO - (products of P, k and dX, covered by |dX|),
      dlog_decay_t: the pairs i >= t > j of W_ij (scale (dO_i . N_j) q_i . k_j - (dX_i . N_j) k_i . k_j); dbeta_j: over i, without beta_j.
    The state in front of the first token counts as one more token for q, k and log_decay. Padded tokens have zeros in misses and grad_out."""
    group = misses.shape[1] // q.shape[1]
    scale = k.shape[-1] ** -0.5 if scale is None else scale
    q, k = (t.detach().double().repeat_interleave(group, 1).abs() for t in (q, k))
    n, do, dv, beta = (t.detach().double().abs() for t in (misses, grad_out, grad_v, beta))
    total = log_decay.detach().double().clamp(min=-1e5).cumsum(-1)
    tokens = n.shape[2]
    decay = _pair_decays(log_decay)
    weight = decay * beta[..., None, :]
    dx = dv + (scale * weight * (q @ k.transpose(-1, -2))).transpose(-1, -2) @ do
    from_out, from_x = scale * (do @ n.transpose(-1, -2)), (dx @ n.transpose(-1, -2)).tril(-1)
    mag_q = (weight * from_out) @ k
    mag_k = (weight * from_out).transpose(-1, -2) @ q + (weight * from_x) @ k + (weight * from_x).transpose(-1, -2) @ k
    pairs = decay * (from_out * (q @ k.transpose(-1, -2)) + from_x * (k @ k.transpose(-1, -2)))
    mag_beta = pairs.sum(-2)
    behind = (pairs * beta[..., None, :]).flip(-2).cumsum(-2).flip(-2).cumsum(-1)  # [t, j]: over i >= t and up to j
    mag_g = torch.cat([torch.zeros_like(behind[..., :1, 0]), behind.diagonal(-1, -2, -1)], -1) if tokens > 1 else torch.zeros_like(total)
    if initial_state is not None:
        start = initial_state.double().abs()
        grown = total.exp()[..., None]
        out_k, x_k = scale * grown * (do @ start.transpose(-1, -2)), grown * (dx @ start.transpose(-1, -2))
        mag_q, mag_k = mag_q + out_k, mag_k + x_k
        mag_g = mag_g + (q * out_k + k * x_k).sum(-1).flip(-1).cumsum(-1).flip(-1)
    fold = lambda t: t.unflatten(1, (-1, group)).sum(2)  # noqa: E731
    return fold(mag_q), fold(mag_k), dx, mag_g, mag_beta
