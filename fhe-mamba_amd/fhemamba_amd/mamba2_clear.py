"""A chain payload's Mamba-2 model in the clear on the GPU.

A client that holds the prompt runs the model on it here, the whole prompt in one call, and whoever
fits the polynomials or tunes the weights to them runs and differentiates the same model.  The states
that it leaves start the plain decode (mamba2_payload.decode_tokens); the encrypted decode starts from
empty ones.  The layer is mamba2_payload.layer_step with exact functions
(src/fhemamba/reference.py:182-339): RMSNorm, in_proj, causal convolution and SiLU, the selective scan,
the gate and its norm, out_proj, the residual; the norms and projections are torch's, the rest
clear.py's kernels.

    python -m fhemamba_amd.mamba2_clear PAYLOAD RESULT [--prompt-tokens K] [--dtype float32|bfloat16]
        [--top N] [--states FILE]

runs a payload's test embeddings: the first K (default: all but one) in one call, the others token by
token from the states that it leaves, checks every final hidden vector against the payload's exact
reference, and writes a fhemamba-m2-clear-result-v1 report.  With a client head in the payload the
report has the log probability of the greedy token, the entropy and the N likeliest tokens of each
step.  --states writes the carried states (ssm_<layer> [heads][head_dim][states], fifo_<layer>
[taps - 1][channels]) as a .npz file.  Exit code 1: a result is further than the tolerance.
"""
from __future__ import annotations

import argparse
import json
import sys
import time
from dataclasses import dataclass
from typing import Optional

import numpy as np
import torch

from . import clear
from .mamba2_payload import ChainPayload, LayerPayload, LayerState, read_chain_payload

# Relative 2-norm error of a final hidden vector: float32 sums over a layer's thousands of terms, or
# bfloat16 activations, each rounding 2^-8, through the layers' residuals.
TOLERANCE = {torch.float32: 1e-4, torch.bfloat16: 5e-2}


@dataclass
class State:
    """One layer's carried state: ssm [rows, heads, head_dim, states] float32 and the convolution's last
    inputs [rows, taps - 1, channels], oldest first; a row a sequence (or a request's slot)."""
    ssm: torch.Tensor
    conv: torch.Tensor


class Layer:
    """A payload layer's weights on the GPU; projections in the model's type, the others float32."""

    PROJECTIONS = ("in_proj_w", "out_proj_w")
    OTHERS = ("conv_w", "conv_b", "dt_bias", "a_log", "d_skip", "block_norm_w", "gated_norm_w")

    def __init__(self, lay: LayerPayload, dtype: torch.dtype, device):
        self.shape = lay
        self.weights = {k: torch.as_tensor(lay.t(k), dtype=dtype, device=device) for k in self.PROJECTIONS}
        self.weights.update({k: torch.as_tensor(lay.t(k), dtype=torch.float32, device=device) for k in self.OTHERS})

    def __call__(self, hidden: torch.Tensor, state: Optional[State], mixer) -> tuple:
        """hidden [.., d_model] float32 -> (hidden, state); `mixer` runs the convolution and the scan."""
        w, s = self.weights, self.shape
        dtype = w["in_proj_w"].dtype
        normed = hidden * torch.rsqrt(hidden.square().mean(-1, keepdim=True) + s.eps_block) * w["block_norm_w"]
        proj = normed.to(dtype) @ w["in_proj_w"].t()
        z, inputs, dt = torch.split(proj, [s.d_inner, s.conv_dim, s.num_heads], dim=-1)
        write = torch.nn.functional.softplus(dt.float() + w["dt_bias"])
        y, state = mixer(self, inputs, write, write * -torch.exp(w["a_log"]), state)
        gated = y.flatten(-2).float() * torch.nn.functional.silu(z.float())
        gated = gated * torch.rsqrt(gated.square().mean(-1, keepdim=True) + s.eps_gated) * w["gated_norm_w"]
        return hidden + (gated.to(dtype) @ w["out_proj_w"].t()).float(), state

    def split(self, conv: torch.Tensor) -> tuple:
        """x, B and C as views of the convolution's output."""
        s = self.shape
        x, B, C = torch.split(conv, [s.d_inner, s.state_size, s.state_size], dim=-1)
        return x.unflatten(-1, (s.num_heads, s.head_dim)), B.unsqueeze(-2), C.unsqueeze(-2)


class ClearMamba2:
    """The layers and the final norm of a chain payload, and its client head if it has one."""

    def __init__(self, chain: ChainPayload, dtype: torch.dtype = torch.float32, device="cuda"):
        if dtype not in TOLERANCE:
            raise ValueError(f"dtype must be float32 or bfloat16, not {dtype}")
        self.dtype, self.device = dtype, torch.device(device)
        self.layers = [Layer(lay, dtype, device) for lay in chain.layers]
        self.norm_eps = chain.final_norm_eps
        self.norm_w = torch.as_tensor(chain.final_norm_w, dtype=torch.float32, device=device)
        self.embedding = self.head = self.head_bias = None
        ar = chain.autoregressive
        if ar is not None:
            self.embedding = torch.as_tensor(ar.embedding_w, dtype=torch.float32, device=device)
            tied = ar.lm_head_w is None
            self.head = self.embedding.to(dtype) if tied else torch.as_tensor(ar.lm_head_w, dtype=dtype, device=device)
            if ar.lm_head_b is not None:
                self.head_bias = torch.as_tensor(ar.lm_head_b, dtype=torch.float32, device=device)

    def parameters(self) -> list:
        """The layers' and the final norm's weights (the head and the embeddings stay as they are)."""
        return [v for lay in self.layers for v in lay.weights.values()] + [self.norm_w]

    def zero_states(self, rows: int) -> list:
        """States of `rows` sequences or slots, as step() updates them in place."""
        out = []
        for lay in self.layers:
            s = lay.shape
            out.append(State(torch.zeros(rows, s.num_heads, s.head_dim, s.state_size, device=self.device),
                             torch.zeros(rows, s.conv_kernel - 1, s.conv_dim, dtype=self.dtype, device=self.device)))
        return out

    def _final(self, hidden):
        return hidden * torch.rsqrt(hidden.square().mean(-1, keepdim=True) + self.norm_eps) * self.norm_w

    def forward(self, embeddings, states=None, *, cu_seqlens=None) -> tuple:
        """Whole sequences [sequences, tokens, d_model] float32, or packed [tokens, d_model] with cu_seqlens,
        from `states` (default zeros): (final normed hidden, the states behind the last tokens)."""
        def mixer(lay, inputs, write, log_decay, state):
            conv, last = clear.causal_conv(inputs, lay.weights["conv_w"], lay.weights["conv_b"],
                                           initial_state=None if state is None else state.conv,
                                           cu_seqlens=cu_seqlens, return_state=True)
            y, ssm = clear.ssm_scan(*self._scan_inputs(lay, conv, write, log_decay), lay.weights["d_skip"],
                                    initial_state=None if state is None else state.ssm, cu_seqlens=cu_seqlens,
                                    return_state=True)
            return y, State(ssm, last)

        hidden, out = embeddings, []
        for i, lay in enumerate(self.layers):
            hidden, state = lay(hidden, None if states is None else states[i], mixer)
            out.append(state)
        return self._final(hidden), out

    @staticmethod
    def _scan_inputs(lay, conv, write, log_decay):
        x, B, C = lay.split(conv)
        return x, write, log_decay, B, C

    @torch.no_grad()
    def step(self, embeddings, states, *, slots=None):
        """One token of each request [requests, d_model]: the final normed hidden; `states` move on in place.
        slots as in clear.ssm_step."""
        def mixer(lay, inputs, write, log_decay, state):
            conv = clear.causal_conv_step(state.conv, inputs, lay.weights["conv_w"], lay.weights["conv_b"], slots=slots)
            y = clear.ssm_step(state.ssm, *self._scan_inputs(lay, conv, write, log_decay), lay.weights["d_skip"],
                               slots=slots)
            return y, state

        hidden = embeddings
        for lay, state in zip(self.layers, states):
            hidden, _ = lay(hidden, state, mixer)
        return self._final(hidden)

    def logits(self, hidden):
        if self.head is None:
            raise ValueError("the payload has no client head")
        out = hidden.to(self.dtype) @ self.head.t()
        return out if self.head_bias is None else (out.float() + self.head_bias).to(self.dtype)

    def score(self, hidden, targets, top: int = 0) -> clear.TokenLogprobs:
        """Log probabilities of target tokens, entropies and likeliest tokens at each hidden vector."""
        return clear.token_logprobs(self.logits(hidden), targets, top=top)

    def loss(self, ids, *, cu_seqlens=None):
        """Mean negative log probability of each token's successor; ids [sequences, tokens], or packed, where
        tokens outside of every sequence take no part."""
        hidden, _ = self.forward(self.embedding[ids], cu_seqlens=cu_seqlens)
        targets = torch.cat([ids[..., 1:], torch.full_like(ids[..., :1], -1)], dim=-1)
        if cu_seqlens is not None:  # neither a sequence's last token nor one outside of all has a successor
            begins, ends = cu_seqlens[:-1].long(), cu_seqlens[1:].long()
            at = torch.arange(ids.shape[0], device=ids.device)
            own = torch.searchsorted(ends, at, right=True).clamp(max=ends.shape[0] - 1)  # the first that ends behind it
            targets = torch.where((at >= begins[own]) & (at + 1 < ends[own]), targets, -1)
        scored = self.score(hidden, targets).logprob
        return -scored.sum() / (targets >= 0).sum().clamp(min=1)


def layer_states(states, row: int = 0) -> list:
    """One row of the states as mamba2_payload.LayerState, the start of a plain decode."""
    return [LayerState(s.ssm[row].double().cpu().numpy(), list(s.conv[row].double().cpu().numpy())) for s in states]


def run(chain: ChainPayload, *, prompt_tokens: Optional[int] = None, dtype=torch.float32, top: int = 5,
        states_file: Optional[str] = None) -> dict:
    model = ClearMamba2(chain, dtype)
    tokens = torch.as_tensor(chain.input_embeddings, dtype=torch.float32, device=model.device)
    n = tokens.shape[0]
    k = max(n - 1, 1) if prompt_tokens is None else prompt_tokens
    if not 1 <= k <= n:
        raise ValueError(f"prompt tokens must be 1 to {n}")
    with torch.no_grad():
        torch.cuda.synchronize()
        begin = time.monotonic()
        hidden, states = model.forward(tokens[None, :k])
        torch.cuda.synchronize()
        prompt_s = time.monotonic() - begin
        finals, begin = [hidden[0]], time.monotonic()
        for t in range(k, n):
            finals.append(model.step(tokens[t: t + 1], states))
        torch.cuda.synchronize()
        step_s = time.monotonic() - begin
        final = torch.cat(finals)
        want = np.asarray(chain.expected_final, dtype=np.float64)[:n]
        errors = np.linalg.norm(final.double().cpu().numpy() - want, axis=-1) / np.linalg.norm(want, axis=-1)
        report = {"format": "fhemamba-m2-clear-result-v1", "dtype": str(dtype).replace("torch.", ""),
                  "layers": len(model.layers), "prompt_tokens": k, "step_tokens": n - k, "seconds_prompt": prompt_s,
                  "seconds_per_step": step_s / (n - k) if n > k else None,
                  "relative_errors": [float(e) for e in errors], "tolerance": TOLERANCE[dtype],
                  "passed": bool(np.all(errors <= TOLERANCE[dtype]))}
        if model.head is not None:
            greedy = model.logits(final).argmax(-1)
            scored = model.score(final, greedy, min(top, model.head.shape[0], clear.MAX_TOP))
            report["head"] = {"greedy": greedy.tolist(), "logprob": scored.logprob.tolist(),
                              "entropy": scored.entropy.tolist()}
            if scored.top_index is not None:
                report["head"].update(top_index=scored.top_index.tolist(), top_logprob=scored.top_logprob.tolist())
        if states_file:
            arrays = {}
            for i, s in enumerate(layer_states(states)):
                arrays[f"ssm_{i:02d}"], arrays[f"fifo_{i:02d}"] = s.ssm, np.stack(s.fifo)
            np.savez(states_file, **arrays)
    return report


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(prog="fhemamba_amd.mamba2_clear",
                                 description="A chain payload in the clear on the GPU.")
    ap.add_argument("payload")
    ap.add_argument("result")
    ap.add_argument("--prompt-tokens", type=int, default=None)
    ap.add_argument("--dtype", choices=("float32", "bfloat16"), default="float32")
    ap.add_argument("--top", type=int, default=5)
    ap.add_argument("--states", default=None)
    args = ap.parse_args(argv)
    report = run(read_chain_payload(args.payload), prompt_tokens=args.prompt_tokens,
                 dtype=getattr(torch, args.dtype), top=args.top, states_file=args.states)
    with open(args.result, "w") as f:
        json.dump(report, f, indent=1)
    print(json.dumps({k: v for k, v in report.items() if k != "head"}))
    return 0 if report["passed"] else 1


if __name__ == "__main__":
    sys.exit(main())
