"""Workloads of the operators around the Mamba-2 mixer in the clear: embedding lookup, norms fused with the
gate and the residual, projections in 8-bit integers, the selection of a beam search and its states.

Each case is a plain dict: `op` names the operator, `dtype` the type of the activations, the rest its
shape.  Where `own` is false, run() computes the operator from elementary torch operations in 32 bits,
rounded once; where it is true it calls fhemamba_amd.clear.

  norm      n = v / sqrt(mean(v^2) + eps) * w  with v = x silu(z), over each of some groups of channels
  add_norm  h' = h + s u  and  n = h' / sqrt(mean(h'^2) + eps) * w: the residual and the next layer's norm
  int8      y = (q W^T) a b + bias: rows of x rounded to 8-bit q with a scale a each, 8-bit weights W with
            a scale b for each output channel; a = max|x| / 127 and x / a are 32-bit numbers, q the nearest
            integer (even among equals)
  embed     scale * weight[id], zeros where the id is below 0, and the weight's gradient
  beam      the best of (a beam's score + log softmax of its logits), a finished beam going on with the end
            token alone at its own score; then every layer's states follow their beams, in place

The sizes are those of the 130M decode (768 channels, 1536 inside a layer, 3352 projected, 24 heads of 64,
128 states, 1792 convolved channels, 50280 tokens) and of the test chains, from one token to a batch of
long prompts.
"""
import math
import os
import sys

import torch

own = False

MODEL, INNER, PROJECTED, VOCAB = 768, 1536, 3352, 50280
STATES = {"heads": 24, "head_dim": 64, "states": 128, "channels": 1792, "taps": 4}
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5


def listed():
    return [
        # One decoded token of one request: the residual and the next layer's norm.  Latency.
        {"name": "add_norm_one", "op": "add_norm", "rows": 1, "channels": MODEL, "hidden": "fp32", "dtype": "bf16",
         "scaled": False, "train": False},
        # The same in a training step over four texts of 2048 tokens, with a residual scale: every gradient.
        {"name": "add_norm_train", "op": "add_norm", "rows": 8192, "channels": MODEL, "hidden": "fp32", "dtype": "bf16",
         "scaled": True, "train": True},
        # The gate and its norm over a batch of long prompts; the gate is a slice of the projection's output.
        {"name": "gated_norm_prompts", "op": "norm", "rows": 30011, "channels": INNER, "groups": 1, "gated": True,
         "sliced": True, "dtype": "bf16", "out": "bf16", "train": False},
        # A training step of a gated norm in 32 bits at odd sizes: two groups of 333 channels.
        {"name": "gated_norm_train_odd_fp32", "op": "norm", "rows": 1777, "channels": 666, "groups": 2, "gated": True,
         "sliced": False, "dtype": "fp32", "out": "fp32", "train": True},
        # The head for one decoded token: all of its weights are read for one row.
        {"name": "int8_head_one", "op": "int8", "rows": 1, "inputs": MODEL, "outputs": VOCAB, "bias": False,
         "dtype": "bf16"},
        # A layer's output projection for one token of each of 250 requests, in 32 bits, with a bias.
        {"name": "int8_step_fp32", "op": "int8", "rows": 250, "inputs": INNER, "outputs": MODEL, "bias": True,
         "dtype": "fp32"},
        # A layer's input projection over a batch of long prompts: the largest product.
        {"name": "int8_prompts", "op": "int8", "rows": 30011, "inputs": MODEL, "outputs": PROJECTED, "bias": False,
         "dtype": "bf16"},
        # The embeddings of a batch of prompts, some of its rows padding.
        {"name": "embed_prompts", "op": "embed", "tokens": 30011, "vocab": VOCAB, "channels": MODEL, "dtype": "fp32",
         "scale": 1.0, "padded": True, "train": False},
        # A training step's lookup and the embedding's gradient, tokens as frequent as in text.
        {"name": "embed_train", "op": "embed", "tokens": 8192, "vocab": VOCAB, "channels": MODEL, "dtype": "fp32",
         "scale": 1.0, "padded": False, "train": True},
        # The same in 16 bits with scaled embeddings at an odd width.
        {"name": "embed_train_odd", "op": "embed", "tokens": 3001, "vocab": 9973, "channels": 333, "dtype": "bf16",
         "scale": 18.25, "padded": True, "train": True},
        # One step of a search with four beams for one request; the states of all 24 layers follow.
        {"name": "beam_one", "op": "beam", "requests": 1, "beams": 4, "vocab": VOCAB, "dtype": "fp32", "masked": False,
         "ended": False, "first": False, "layers": 24, **STATES},
        # A batch of searches with eight beams in 16 bits, some beams finished, part of the vocabulary masked off;
        # two layers' states.
        {"name": "beam_many", "op": "beam", "requests": 32, "beams": 8, "vocab": VOCAB, "dtype": "bf16", "masked": True,
         "ended": True, "first": False, "layers": 2, **STATES},
    ]


def _log(rng, lo, hi):
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["add_norm", "norm", "norm", "int8", "int8", "int8", "embed", "embed", "beam", "beam"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op in ("add_norm", "norm"):
        train = rng.random() < 0.5
        channels = rng.choice([MODEL, INNER, MODEL, INNER, 64, 96, 333, 640, 1001, 2048, 4096])
        rows = _log(rng, 1, int((6.2e6 if train else 4.6e7) / channels / (2 if dtype == "fp32" else 1)))
        if op == "add_norm":
            hidden = rng.choice(["fp32", "fp32", dtype])
            return {"op": op, "rows": rows, "channels": channels, "hidden": hidden, "dtype": dtype,
                    "scaled": rng.random() < 0.5, "train": train}
        gated = rng.random() < 0.7
        groups = rng.choice([1, 1, 1, 2, 3])
        return {"op": op, "rows": rows, "channels": channels - channels % groups, "groups": groups, "gated": gated,
                "sliced": not train and rng.random() < 0.5, "dtype": dtype,
                "out": rng.choice(["bf16", dtype]), "train": train}
    if op == "int8":
        inputs, outputs = rng.choice([(MODEL, PROJECTED), (INNER, MODEL), (MODEL, VOCAB), (96, 392), (1001, 643),
                                      (2048, 2048), (64, 17), (333, 1280)])
        most = min(30000, int(1.0e8 / outputs / (2 if dtype == "fp32" else 1)), int(7.7e10 / inputs / outputs))
        return {"op": op, "rows": _log(rng, 1, most), "inputs": inputs, "outputs": outputs, "bias": rng.random() < 0.5,
                "dtype": dtype}
    if op == "embed":
        channels = rng.choice([MODEL, MODEL, 64, 96, 333, 1001, 2048])
        vocab = VOCAB if rng.random() < 0.5 else _log(rng, 93, VOCAB)
        train = rng.random() < 0.6
        if channels == 2048 and train:
            vocab = min(vocab, 18000)
        return {"op": op, "tokens": _log(rng, 1, int((8192 if train else 30000) * min(1.0, MODEL / channels))),
                "vocab": vocab, "channels": channels, "dtype": dtype, "scale": rng.choice([1.0, 1.0, 27.5]),
                "padded": rng.random() < 0.5, "train": train}
    vocab = VOCAB if rng.random() < 0.5 else _log(rng, 93, VOCAB)
    beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
    c = {"op": op, "requests": _log(rng, 1, 240 // beams), "beams": beams, "vocab": vocab, "dtype": dtype,
         "masked": rng.random() < 0.4, "ended": rng.random() < 0.4, "first": rng.random() < 0.2, "layers": 2}
    if rng.random() < 0.5:
        return {**c, **STATES}
    return {**c, "heads": rng.randint(1, 12), "head_dim": rng.choice([16, 33, 48, 64]),
            "states": rng.choice([16, 33, 40, 128]), "channels": rng.choice([96, 640, 1001]),
            "taps": rng.choice([2, 4])}


# ----------------------------------------------------------------- inputs
def _normal(gen, shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _uniform(gen, shape):
    return torch.rand(shape, generator=gen, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    c, dt = case, DTYPES[case["dtype"]]
    s = {"case": c}
    if c["op"] == "add_norm":
        R, Cn, ht = c["rows"], c["channels"], DTYPES[c["hidden"]]
        size = torch.exp(_normal(gen, (R, 1)))                     # rows of different sizes
        s["hidden"] = (2.0 * size * _normal(gen, (R, Cn))).to(ht)
        s["update"] = (size * _normal(gen, (R, Cn))).to(dt)
        s["weight"] = 1.0 + 0.2 * _normal(gen, (Cn,))
        s["scale"] = 0.5 + 0.1 * _normal(gen, (Cn,)) if c["scaled"] else None
        if c["train"]:
            s["dn"], s["dh"] = _normal(gen, (R, Cn), dt), _normal(gen, (R, Cn), ht)
            s["leaves"] = [s[k] for k in ("hidden", "update", "weight") + (("scale",) if c["scaled"] else ())]
    elif c["op"] == "norm":
        R, Cn = c["rows"], c["channels"]
        s["x"] = (torch.exp(_normal(gen, (R, 1))) * _normal(gen, (R, Cn))).to(dt)
        wide = 1816 if c["sliced"] else 0
        s["gate"] = _normal(gen, (R, Cn + wide), dt)[:, :Cn] if c["gated"] else None
        s["weight"] = 1.0 + 0.2 * _normal(gen, (Cn,))
        if c["train"]:
            s["dn"] = _normal(gen, (R, Cn), DTYPES[c["out"]])
            s["leaves"] = [s[k] for k in ("x", "weight") + (("gate",) if c["gated"] else ())]
    elif c["op"] == "int8":
        R, K, N = c["rows"], c["inputs"], c["outputs"]
        s["x"] = (torch.exp(_normal(gen, (R, 1))) * _normal(gen, (R, K))).to(dt)
        real = _normal(gen, (N, K)) / math.sqrt(K)
        s["weight_scale"] = real.abs().amax(1) / 127.0
        s["weight"] = torch.round(real / s["weight_scale"][:, None]).clamp(-127, 127).to(torch.int8)
        s["bias"] = 0.1 * _normal(gen, (N,)) if c["bias"] else None
    elif c["op"] == "embed":
        T, V, Cn = c["tokens"], c["vocab"], c["channels"]
        # frequencies of words: the n-th about 1 / (n + 3), in an order of their own
        rank = torch.exp(_uniform(gen, (T,)).double() * math.log((V + 3) / 3.0)) * 3.0 - 3.0
        s["ids"] = torch.randperm(V, generator=gen, device="cuda")[rank.long().clamp(0, V - 1)]
        if c["padded"]:
            s["ids"][_uniform(gen, (T,)) < 0.1] = -1
        s["weight"] = (0.02 * _normal(gen, (V, Cn))).to(dt)
        if c["train"]:
            s["dy"] = _normal(gen, (T, Cn), dt)
            s["leaves"] = [s["weight"]]
    else:
        R, B, V = c["requests"], c["beams"], c["vocab"]
        s["logits"] = (3.0 * _normal(gen, (R, B, V))).to(dt)
        if c["masked"]:
            s["logits"].masked_fill_(_uniform(gen, (R, B, V)) < 0.3, -math.inf)
        s["scores"] = -5.0 - 3.0 * _uniform(gen, (R, B))
        if c["first"]:
            s["scores"][:, 1:] = -math.inf
        s["finished"] = _uniform(gen, (R, B)) < 0.2 if c["ended"] else None
        cache = R * B + 5
        s["slots"] = torch.randperm(cache, generator=gen, device="cuda")[: R * B].reshape(R, B).to(torch.int32)
        s["cache"] = []
        for _ in range(c["layers"]):
            s["cache"].append(0.3 * _normal(gen, (cache, c["heads"], c["head_dim"], c["states"])))
            s["cache"].append(_normal(gen, (cache, c["taps"] - 1, c["channels"]), dt))
    for t in s.get("leaves", ()):
        t.requires_grad_(True)
    return s


# ----------------------------------------------------------------- plain forms
def _plain_norm(v, weight, groups):
    v = v.unflatten(-1, (groups, -1))
    n = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    return n.flatten(-2) * weight


def _plain_int8(s):
    """The quotient's rounding to an integer is next to a border for values half between two: in 64 bits, then 32."""
    x = s["x"].float()
    a = (x.abs().amax(-1, keepdim=True).double() / 127.0).float()
    q = torch.where(a > 0, (x.double() / a.double()).float(), torch.zeros((), device="cuda"))
    q = torch.round(q).clamp(-127.0, 127.0)
    y = (q @ s["weight"].float().t()) * (a * s["weight_scale"])
    return y if s["bias"] is None else y + s["bias"]


def _plain_beam(s):
    """In 64 bits: the order of near scores."""
    c = s["case"]
    R, B, V = c["requests"], c["beams"], c["vocab"]
    l = s["logits"].double()
    m = l.amax(-1, keepdim=True)
    total = l - m - torch.log(torch.exp(l - m).sum(-1, keepdim=True)) + s["scores"].double()[..., None]
    if s["finished"] is not None:
        end = torch.arange(V, device="cuda") == V - 1
        stays = torch.where(end, s["scores"].double()[..., None], torch.full((), -math.inf, device="cuda").double())
        total = torch.where(s["finished"][..., None], stays, total)
    best, at = torch.sort(total.reshape(R, B * V), dim=-1, descending=True, stable=True)
    best, at = best[:, :B], at[:, :B]
    parent = torch.div(at, V, rounding_mode="floor")
    source, target = s["slots"].long().gather(1, parent).reshape(-1), s["slots"].long().reshape(-1)
    for t in s["cache"]:
        t[target] = t[source]
    return best.float(), parent.to(torch.int32), (at % V).to(torch.int32), s["cache"]


def _run_plain(s):
    c, dt = s["case"], DTYPES[s["case"]["dtype"]]
    if c["op"] == "add_norm":
        u = s["update"].float() if s["scale"] is None else s["update"].float() * s["scale"]
        h = s["hidden"].float() + u
        n, h = _plain_norm(h, s["weight"], 1).to(dt), h.to(DTYPES[c["hidden"]])
        if not c["train"]:
            return n, h
        return n.detach(), h.detach(), *torch.autograd.grad([n, h], s["leaves"], [s["dn"], s["dh"]])
    if c["op"] == "norm":
        v = s["x"].float()
        if c["gated"]:
            z = s["gate"].float()
            v = v * (z / (1.0 + torch.exp(-z)))
        n = _plain_norm(v, s["weight"], c["groups"]).to(DTYPES[c["out"]])
        if not c["train"]:
            return n
        return n.detach(), *torch.autograd.grad(n, s["leaves"], s["dn"])
    if c["op"] == "int8":
        return _plain_int8(s).to(dt)
    if c["op"] == "embed":
        real = s["ids"] >= 0
        ids = s["ids"].clamp(min=0)
        y = s["weight"].detach()[ids].float() * c["scale"]
        y = torch.where(real[:, None], y, torch.zeros((), device="cuda")).to(dt)
        if not c["train"]:
            return y
        d = torch.where(real[:, None], s["dy"].float() * c["scale"], torch.zeros((), device="cuda"))
        return y, torch.zeros(s["weight"].shape, device="cuda").index_add_(0, ids, d).to(dt)
    return _plain_beam(s)


def _run_own(s):
    from fhemamba_amd import clear

    c, dt = s["case"], DTYPES[s["case"]["dtype"]]
    if c["op"] == "add_norm":
        n, h = clear.add_norm(s["hidden"], s["update"], s["weight"], scale=s["scale"], eps=EPS)
        if not c["train"]:
            return n, h
        return n.detach(), h.detach(), *torch.autograd.grad([n, h], s["leaves"], [s["dn"], s["dh"]])
    if c["op"] == "norm":
        n = clear.rms_norm(s["x"], s["weight"], gate=s["gate"], groups=c["groups"], eps=EPS, dtype=DTYPES[c["out"]])
        if not c["train"]:
            return n
        return n.detach(), *torch.autograd.grad(n, s["leaves"], s["dn"])
    if c["op"] == "int8":
        return clear.int8_linear(s["x"], s["weight"], s["weight_scale"], s["bias"])
    if c["op"] == "embed":
        y = clear.embed(s["weight"], s["ids"], scale=c["scale"])
        if not c["train"]:
            return y
        return y.detach(), *torch.autograd.grad(y, s["leaves"], s["dy"])
    got = clear.beam_select(s["logits"], s["scores"], c["beams"], finished=s["finished"],
                            end=None if s["finished"] is None else c["vocab"] - 1)
    clear.reorder_states(s["cache"], got.parent, slots=s["slots"])
    return got.score, got.parent, got.token, s["cache"]


def run(state):
    if not own:
        return _run_plain(state)
    path = os.path.join(os.getcwd(), "fhe-mamba_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    return _run_own(state)


# ----------------------------------------------------------------- work
def work(case):
    c, e = case, 2 if case["dtype"] == "bf16" else 4
    if c["op"] == "add_norm":
        n, h = c["rows"] * c["channels"], 2 if c["hidden"] == "bf16" else 4
        weights = 4 * c["channels"] * (2 if c["scaled"] else 1)
        w = {"bytes": n * (2 * h + 2 * e) + weights, "flops": 6 * n}
        if c["train"]:  # dn and dh in, dhidden and dupdate out, and h' again
            w = {"bytes": w["bytes"] + n * (2 * e + 3 * h) + weights, "flops": 18 * n}
        return w
    if c["op"] == "norm":
        n, o, g = c["rows"] * c["channels"], 2 if c["out"] == "bf16" else 4, 2 if c["gated"] else 1
        w = {"bytes": n * (g * e + o) + 4 * c["channels"], "flops": n * (4 + 5 * (g - 1))}
        if c["train"]:
            w = {"bytes": w["bytes"] + n * (2 * g * e + o) + 4 * c["channels"], "flops": n * (14 + 20 * (g - 1))}
        return w
    if c["op"] == "int8":
        R, K, N = c["rows"], c["inputs"], c["outputs"]
        return {"bytes": R * K * e + N * K + R * N * e + 4 * N * (2 if c["bias"] else 1), "flops": 2 * R * K * N}
    if c["op"] == "embed":
        T, Cn = c["tokens"], c["channels"]
        w = {"bytes": T * (8 + Cn * e) + min(T, c["vocab"]) * Cn * e, "flops": T * Cn}
        if c["train"]:
            w = {"bytes": w["bytes"] + T * (8 + Cn * e) + c["vocab"] * Cn * e, "flops": 3 * T * Cn}
        return w
    n, B = c["requests"] * c["beams"], c["beams"]
    state = c["layers"] * (4 * c["heads"] * c["head_dim"] * c["states"] + e * (c["taps"] - 1) * c["channels"])
    moved = n * (B - 1) / B                                         # a beam in B goes on where it lies
    return {"bytes": int(n * (c["vocab"] * e + 16) + 2 * moved * state), "flops": 4 * n * c["vocab"]}


# ----------------------------------------------------------------- 64 bits
def _exact_add_norm(s):
    c = s["case"]
    h, u, w = (s[k].detach().double() for k in ("hidden", "update", "weight"))
    scale = torch.ones_like(w) if s["scale"] is None else s["scale"].detach().double()
    h = h + scale * u
    r = 1.0 / torch.sqrt(h.square().mean(-1, keepdim=True) + EPS)
    n = h * r * w
    if not c["train"]:
        return n, h
    dn, unit = s["dn"].double(), h * r
    g = dn * w
    d = s["dh"].double() + r * (g - unit * (g * unit).mean(-1, keepdim=True))
    return (n, h, d, d * scale, (dn * unit).sum(0), *([(d * u).sum(0)] if c["scaled"] else []))


def _exact_norm(s):
    c = s["case"]
    G = c["groups"]
    x, w = s["x"].detach().double(), s["weight"].detach().double()
    z = s["gate"].detach().double() if c["gated"] else None
    sig = None if z is None else torch.sigmoid(z)
    v = x if z is None else x * z * sig

    def mean(t):
        return t.unflatten(-1, (G, -1)).mean(-1).repeat_interleave(c["channels"] // G, dim=-1)

    r = 1.0 / torch.sqrt(mean(v * v) + EPS)
    n = v * r * w
    if not c["train"]:
        return n
    dn, unit = s["dn"].double(), v * r
    g = dn * w
    d = r * (g - unit * mean(g * unit))
    dw = (dn * unit).sum(0)
    if z is None:
        return n, d, dw
    return n, d * z * sig, dw, d * x * sig * (1.0 + z * (1.0 - sig))


def _exact_int8(s):
    x = s["x"].double()
    scale = (x.abs().max(dim=-1).values / 127.0).float().double()[:, None]
    ratio = (x / torch.where(scale > 0, scale, 1.0)).float().double()   # as the definition has it, of 32 bits
    q = torch.clamp(torch.round(ratio), -127.0, 127.0)
    y = torch.matmul(q * scale, (s["weight"].double() * s["weight_scale"].double()[:, None]).T)
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_embed(s):
    c = s["case"]
    w = s["weight"].detach().double()
    y = torch.zeros(c["tokens"], c["channels"], dtype=torch.float64, device="cuda")
    real = (s["ids"] >= 0).nonzero()[:, 0]
    y[real] = w[s["ids"][real]] * c["scale"]
    if not c["train"]:
        return y
    d = torch.zeros_like(w)
    order = torch.sort(s["ids"][real], stable=True)
    sums = torch.cumsum(s["dy"].double()[real][order.indices], 0)
    last = torch.cat([order.values[1:] != order.values[:-1], torch.ones(1, dtype=torch.bool, device="cuda")]) \
        if real.numel() else torch.zeros(0, dtype=torch.bool, device="cuda")
    ends = sums[last]
    if real.numel():
        d[order.values[last]] = c["scale"] * (ends - torch.cat([torch.zeros_like(ends[:1]), ends[:-1]]))
    return y, d


def _exact_beam(s):
    """The scores; which they are has no value in 64 bits beside the whole numbers themselves."""
    c = s["case"]
    scores = torch.log_softmax(s["logits"].double(), -1) + s["scores"].double()[..., None]
    if s["finished"] is not None:
        scores[s["finished"]] = -math.inf
        scores[..., c["vocab"] - 1] = torch.where(s["finished"], s["scores"].double(), scores[..., c["vocab"] - 1])
    best = torch.topk(scores.flatten(1), c["beams"], dim=-1).values
    return best, None, None, [None] * len(s["cache"])


def exact(case, seed):
    s = prepare(case, seed)
    return {"add_norm": _exact_add_norm, "norm": _exact_norm, "int8": _exact_int8, "embed": _exact_embed,
            "beam": _exact_beam}[case["op"]](s)
