"""Linear attention with a decay for each head, token by token in 64 bits, and the moves of cache pages on lists.

The definitions the kernels are tested against, written as the recurrence itself (no chunks).  ``bound`` runs the same
recurrence on absolute values: the sum of the magnitudes of all terms of an output, which is what rounding errors are
relative to.
"""
from __future__ import annotations

import torch


def linear_attention(q, k, v, log_decay, *, scale=None, mask=None, seq_idx=None, initial=None):
    """(o [B,T,H,Dv], final state [B,H,Dk,Dv]) in float64; differentiable by autograd."""
    B, T, H, Dk = q.shape
    Dv = v.shape[-1]
    scale = Dk ** -0.5 if scale is None else scale
    k = k.repeat_interleave(H // k.shape[2], 2)
    v = v.repeat_interleave(H // v.shape[2], 2)
    valid = torch.ones(B, T, dtype=torch.bool) if mask is None else (mask != 0)
    q, k, v = (torch.where(valid[..., None, None], x, torch.zeros((), dtype=x.dtype)).double() for x in (q, k, v))
    a = torch.exp(log_decay.double()).view(1, H, 1, 1)
    S = torch.zeros(B, H, Dk, Dv, dtype=torch.float64) if initial is None else initial.double()
    out = []
    for t in range(T):
        if seq_idx is not None and t > 0:
            same = (seq_idx[:, t] == seq_idx[:, t - 1]).view(B, 1, 1, 1)
            S = torch.where(same, S, torch.zeros((), dtype=torch.float64))
        new = a * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        S = torch.where(valid[:, t].view(B, 1, 1, 1), new, S)
        o = (q[:, t, :, :, None] * S).sum(-2) * scale
        out.append(torch.where(valid[:, t].view(B, 1, 1), o, torch.zeros((), dtype=torch.float64)))
    o = torch.stack(out, 1) if T else torch.zeros(B, 0, H, Dv, dtype=torch.float64)
    return o, S


def grads(q, k, v, log_decay, dout, *, scale=None, mask=None, seq_idx=None, initial=None, dfinal=None):
    """(dq, dk, dv, dinitial) in float64 (dinitial None without an initial state).  Values of masked tokens, dout's
    too, are not looked at."""
    if mask is not None:
        keep = (mask != 0)[..., None, None]
        q, k, v, dout = (torch.where(keep, x, torch.zeros((), dtype=x.dtype)) for x in (q, k, v, dout))
    leaves = [x.double().requires_grad_() for x in (q, k, v)]
    s0 = None if initial is None else initial.double().requires_grad_()
    o, S = linear_attention(*leaves, log_decay, scale=scale, mask=mask, seq_idx=seq_idx, initial=s0)
    total = (o * dout.double()).sum()
    if dfinal is not None:
        total = total + (S * dfinal.double()).sum()
    g = torch.autograd.grad(total, leaves + ([s0] if s0 is not None else []), allow_unused=True)
    g = [torch.zeros_like(x) if y is None else y for x, y in zip(leaves + ([s0] if s0 is not None else []), g)]
    return g[0], g[1], g[2], g[3] if s0 is not None else None


def move_pages(tensors, source, cleared=()):
    """New tensors: page i is old page source[i]; then the cleared ones are zero."""
    out = []
    for t in tensors:
        x = t[torch.as_tensor(source, dtype=torch.long)].clone()
        for i in cleared:
            x[i] = 0
        out.append(x)
    return out


def compact_plan(live):
    """(source, new_index, count) of compaction, from a list of truth values."""
    n = sum(map(bool, live))
    source, new = list(range(len(live))), [i if x else -1 for i, x in enumerate(live)]
    tails = [i for i in range(n, len(live)) if live[i]]
    for hole, tail in zip([i for i in range(n) if not live[i]], tails):
        source[hole], new[tail] = tail, hole
    return source, new, n
