"""The scan and its gradients in 64 bits for many long sequences at once: the recurrences written out, both ways,
a token of every sequence at a time.  What clear_reference.scan and autograd give, at sizes that those cannot hold."""
import ctypes

import torch

from fhemamba_amd import _lib, clear


def scan(d, lengths, grads=None, device="cuda"):
    """(y, last states), with grads = (dy, dstate) also the gradients by name.  d: packed tensors by the names
    x, write, log_decay, B, C, D and initial."""
    S, n = len(lengths), max(lengths)
    starts = [sum(lengths[:i]) for i in range(S)]

    def pad(t):
        t = t.to(device)
        out = torch.zeros((S, n, *t.shape[1:]), dtype=torch.float64, device=device)
        for i, (a, m) in enumerate(zip(starts, lengths)):
            out[i, :m] = t[a:a + m]
        return out

    def back(t):
        return torch.cat([t[i, :m] for i, m in enumerate(lengths)])

    x, w, g = (pad(d[k]) for k in ("x", "write", "log_decay"))  # a token that is not there keeps the state
    H, (G, N) = x.shape[2], d["B"].shape[1:]
    P, rep = x.shape[3], H // G
    B, C = (pad(d[k]).repeat_interleave(rep, 2) for k in ("B", "C"))
    D = d["D"].double().to(device)
    h = d["initial"].double().to(device) if d.get("initial") is not None else x.new_zeros(S, H, P, N)
    y, kept = torch.empty_like(x), [h]
    for t in range(n):
        h = torch.exp(g[:, t])[..., None, None] * h + (w[:, t, :, None] * x[:, t])[..., None] * B[:, t, :, None]
        y[:, t] = (h * C[:, t, :, None]).sum(-1) + D[:, None] * x[:, t]
        if grads is not None:
            kept.append(h)
    if grads is None:
        return back(y), h
    dy = pad(grads[0])
    A = torch.zeros_like(h) if grads[1] is None else grads[1].double().to(device)
    dx, dw, dg, dB, dC = (torch.zeros_like(t) for t in (x, w, g, B, C))
    for t in reversed(range(n)):
        A = A + dy[:, t, :, :, None] * C[:, t, :, None]
        dC[:, t] = (dy[:, t, :, :, None] * kept.pop()).sum(2)
        v = (A * B[:, t, :, None]).sum(-1)
        dx[:, t] = w[:, t, :, None] * v + D[:, None] * dy[:, t]
        dw[:, t] = (x[:, t] * v).sum(-1)
        dB[:, t] = w[:, t, :, None] * (x[:, t, :, :, None] * A).sum(2)
        A = torch.exp(g[:, t])[..., None, None] * A
        dg[:, t] = (kept[-1] * A).sum((-1, -2))
    got = {"x": back(dx), "write": back(dw), "log_decay": back(dg),
           "B": back(dB.unflatten(2, (G, rep)).sum(3)), "C": back(dC.unflatten(2, (G, rep)).sum(3)),
           "D": (dy * x).sum((0, 1, 3))}
    if d.get("initial") is not None:
        got["initial"] = A
    return back(y), h, got


def rel(got, want):
    """2-norm of the difference over that of the reference."""
    got, want = got.detach().double(), want.to(got.device)
    assert got.shape == want.shape, (got.shape, want.shape)
    assert bool(torch.isfinite(got).all())
    return float((got - want).norm() / want.norm())


def segment_lengths(lengths, packed, shape, dtype):
    """The lengths of segments that the scan may cut these sequences into, as the size of its workspace tells
    (a segment's state and decays each), or none where the sequences stay whole.  No GPU is needed."""
    H, P, N, G = shape
    S = len(lengths)
    tokens = sum(lengths) if packed else lengths[0]
    at = (4096, 0, 64, 64)
    args = clear._SCAN.pack(clear._DTYPES[dtype], S, H, P, N, G, tokens, 4096 if packed else 0, *at * 5, 0, 0)
    size = ctypes.c_size_t()
    _lib.call("fhe_ssm_scan_workspace", args, 0, ctypes.byref(size))

    def up(n):
        return (n + 255) // 256 * 256

    found = []
    for length in range(64, tokens, 64):
        items = tokens // length + S + 2 if packed else S * -(-tokens // length)
        table = up(16 * items) + up(4 * (S + 1)) if packed else 0
        if size.value == table + up(items * H * 4) + up(items * H * P * N * 4):
            found.append(length)
    whole = up(16 * (1 + S + 2)) + up(4 * (S + 1)) if packed else 0
    assert found or size.value == whole, "the workspace is laid out in another way"
    return found
