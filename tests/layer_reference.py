"""Plain 64-bit forms of the operators around the mixer, on the CPU, differentiable through autograd."""
import math

import torch


def norm(x, weight, gate, groups, eps):
    v = x if gate is None else x * gate * torch.sigmoid(gate)
    parts = v.reshape(*v.shape[:-1], groups, -1)
    parts = parts / torch.sqrt((parts * parts).mean(-1, keepdim=True) + eps)
    return parts.reshape(v.shape) * weight


def add_norm(hidden, update, weight, scale, eps):
    h = hidden + (update if scale is None else update * scale)
    return h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * weight, h


def quantize(x):
    """(values, scale) of rows: the two quotients are rounded to 32 bits by definition, so they are taken there."""
    x = x.float()
    scale = x.abs().amax(-1) / 127.0
    ratio = torch.where(scale[..., None] > 0, x / scale[..., None], torch.zeros(()))
    values = torch.round(ratio).clamp(-127, 127)
    finite = torch.isfinite(x).all(-1)
    values = torch.where(finite[..., None], values, torch.zeros(()))
    return values.to(torch.int8), torch.where(finite, scale, torch.full((), math.nan))


def int8_linear(x, weight, weight_scale, bias):
    values, scale = quantize(x)
    y = (values.double() @ weight.double().t()) * scale.double()[..., None] * weight_scale.double()
    return y if bias is None else y + bias.double()


def beam(logits, scores, width, finished, end):
    """(score, parent, token) of [requests, beams, vocab], candidate by candidate."""
    out = []
    R, B, V = logits.shape
    for r in range(R):
        totals = torch.full((B, V), -math.inf, dtype=torch.float64)
        for b in range(B):
            s = float(scores[r, b])
            if finished is not None and bool(finished[r, b]):
                totals[b, end] = s
            elif s == -math.inf:
                pass
            else:
                row = logits[r, b].double()
                if bool(torch.isnan(row).any()) or bool((row == math.inf).any()) or not s < math.inf:
                    totals[b] = math.nan
                elif bool((row > -math.inf).any()):
                    m = row.max()
                    totals[b] = (row - m) - torch.log(torch.exp(row - m).sum()) + s
        order = sorted(range(B * V), key=lambda i: (not math.isnan(totals.view(-1)[i]), -totals.view(-1)[i]
                                                    if not math.isnan(totals.view(-1)[i]) else 0.0, i)) \
            if B * V <= 4096 else torch.sort(totals.view(-1), descending=True, stable=True).indices.tolist()
        order = order[:width]
        out.append(([float(totals.view(-1)[i]) for i in order], [i // V for i in order], [i % V for i in order]))
    return (torch.tensor([o[0] for o in out], dtype=torch.float64), torch.tensor([o[1] for o in out]),
            torch.tensor([o[2] for o in out]))


def moved(state, parent, slots):
    """The rows of `state` after they follow their beams."""
    new, old = state.clone(), state
    R, B = parent.shape
    for r in range(R):
        for j in range(B):
            p = int(parent[r, j])
            at = r * B + j if slots is None else int(slots[r, j])
            if not 0 <= p < B or not 0 <= at < state.shape[0]:
                continue
            source = r * B + p if slots is None else int(slots[r, p])
            if 0 <= source < state.shape[0]:
                new[at] = old[source]
    return new
