"""Linear attention with a decay for each head, and layer norm, in 64 bits, token by token as they are defined: test infrastructure.

    S_t = e^g S_{t-1} + k_t v_t^T        o_t = scale S_t^T q_t

(the reference's loop, lm_engine/modeling_utils/sequence_mixer_blocks/linear_attention/op.py:10-44, with a log-decay per head).  Gradients
are those of autograd through the loop."""

from __future__ import annotations

import torch


def linear_attention_sequence(q, k, v, g, scale, state):
    """q, k [T, H, K], v [T, H, V], g [H], state [H, K, V], all float64 -> (o [T, H, V], state)."""
    decay = torch.exp(g)[:, None, None]
    out = []
    for t in range(q.size(0)):
        state = decay * state + k[t][:, :, None] * v[t][:, None, :]
        out.append(scale * (q[t][:, :, None] * state).sum(dim=1))
    o = torch.stack(out) if out else v.new_zeros(0, *v.shape[1:])
    return o, state


def sequences_of(B, T, cu_seqlens=None, left_padded=False):
    """(row, first token, length) of every sequence."""
    if cu_seqlens is None:
        return [(b, 0, T) for b in range(B)]
    lens = [b - a for a, b in zip(cu_seqlens, cu_seqlens[1:])]
    if left_padded:
        return [(n, T - length, length) for n, length in enumerate(lens)]
    return [(0, first, length) for first, length in zip(cu_seqlens, lens)]


def linear_attention_ref(q, k, v, g=None, scale=None, initial_state=None, cu_seqlens=None, left_padded=False):
    """(o, final_state) in float64; ``cu_seqlens`` is a list.  Tokens of no sequence read as zeros.  Differentiable."""
    q, k, v = q.double(), k.double(), v.double()
    B, T, HK, K = q.shape
    H, V = v.size(2), v.size(3)
    q, k = q.repeat_interleave(H // HK, dim=2), k.repeat_interleave(H // HK, dim=2)
    g = torch.zeros(H, dtype=torch.float64) if g is None else g.double()
    scale = K**-0.5 if scale is None else scale
    pieces, states = [[] for _ in range(B)], []
    at = [0] * B
    for n, (b, first, length) in enumerate(sequences_of(B, T, cu_seqlens, left_padded)):
        state = v.new_zeros(H, K, V) if initial_state is None else initial_state[n].double()
        pick = slice(first, first + length)
        o, state = linear_attention_sequence(q[b, pick], k[b, pick], v[b, pick], g, scale, state)
        pieces[b] += [v.new_zeros(first - at[b], H, V), o]
        at[b] = first + length
        states.append(state)
    rows = [torch.cat(p + [v.new_zeros(T - end, H, V)]) for p, end in zip(pieces, at)]
    return torch.stack(rows), torch.stack(states)


def layer_norm_ref(x, weight=None, bias=None, eps=1e-5):
    x = x.double()
    centred = x - x.mean(dim=-1, keepdim=True)
    y = centred / torch.sqrt(centred.square().mean(dim=-1, keepdim=True) + eps)
    y = y if weight is None else y * weight.double()
    return y if bias is None else y + bias.double()
