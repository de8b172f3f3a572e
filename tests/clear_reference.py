"""Plain 64-bit forms of the operators in the clear, one token at a time, on the CPU.

Differentiable through torch's autograd, so the gradients' references are those of the recurrences
themselves.  Sequences come as a list of index ranges into the leading token axis.
"""
import math

import torch


def spans(lengths):
    at, out = 0, []
    for n in lengths:
        out.append((at, at + n))
        at += n
    return out


def scan(x, write, log_decay, B, C, D, initial, ranges):
    """(y, last states) of packed tokens; tokens outside of the ranges give zeros."""
    H, (G, N) = x.shape[1], B.shape[1:]
    rep = H // G
    ys, states = [torch.zeros(x.shape[1:], dtype=torch.float64)] * x.shape[0], []
    for i, (a, b) in enumerate(ranges):
        h = torch.zeros(H, x.shape[2], N, dtype=torch.float64) if initial is None else initial[i]
        for t in range(a, b):
            Bt, Ct = B[t].repeat_interleave(rep, 0), C[t].repeat_interleave(rep, 0)
            h = torch.exp(log_decay[t])[:, None, None] * h + (write[t][:, None] * x[t])[..., None] * Bt[:, None]
            y = (h * Ct[:, None]).sum(-1)
            ys[t] = y if D is None else y + D[:, None] * x[t]
        states.append(h)
    return torch.stack(ys) if ys else torch.zeros(x.shape, dtype=torch.float64), torch.stack(states)


def conv(x, weight, bias, initial, ranges, silu=True):
    K = weight.shape[1]
    ys, last = [torch.zeros(x.shape[1], dtype=torch.float64)] * x.shape[0], []
    for i, (a, b) in enumerate(ranges):
        first = torch.zeros(K - 1, x.shape[1], dtype=torch.float64) if initial is None else initial[i]
        wide = torch.cat([first, x[a:b]])
        for t in range(b - a):
            v = (wide[t: t + K] * weight.t()).sum(0)
            v = v if bias is None else v + bias
            ys[a + t] = v * torch.sigmoid(v) if silu else v
        last.append(wide[b - a:])
    return torch.stack(ys) if ys else torch.zeros(x.shape, dtype=torch.float64), torch.stack(last)


def logprob(logits, targets):
    """(log probability, entropy) of rows; rows without an allowed token: -inf and 0."""
    lps, ents = [], []
    for row, t in zip(logits, targets.tolist()):
        kept = row[row > -math.inf]
        if kept.numel() == 0:
            lps.append(row.new_tensor(0.0 if t < 0 else -math.inf))
            ents.append(row.new_tensor(0.0))
            continue
        lse = torch.logsumexp(kept, 0)
        lps.append(row[t] - lse if t >= 0 else row.new_tensor(0.0))
        ents.append(-(torch.exp(kept - lse) * (kept - lse)).sum())
    return torch.stack(lps), torch.stack(ents)


def rel(got, want):
    """2-norm of the difference over that of the reference (or of the difference alone)."""
    got, want = got.detach().double().cpu(), want.detach().double()
    assert got.shape == want.shape, (got.shape, want.shape)
    assert bool(torch.isfinite(got).all())
    d, n = float((got - want).norm()), float(want.norm())
    return d / n if n else d


# Bounds on rel(), from the formats:
#   a result rounded once to bfloat16 (8 bits) is at most 2^-8 off in each value;
#   inside, operands split into two bfloat16 pieces leave at most 2^-16 each: with two such
#   operands on the way and a factor of 4 for terms that cancel, 2^-13;
#   32-bit results of bfloat16 inputs carry that 2^-13 (gates' gradients) or, from
#   three pieces, the sums' own rounding;
#   32-bit sums of up to 2^10 products are off by 2^-24 sqrt(2^10) of their terms'
#   norm, with a factor of 8 for terms that cancel: 2^-16.
BF16, GATES, F32 = 2.0 ** -8 + 2.0 ** -13, 2.0 ** -13, 2.0 ** -16


def bound(t):
    return BF16 if t.dtype == torch.bfloat16 else F32
