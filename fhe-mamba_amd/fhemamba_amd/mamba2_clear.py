"""A chain payload's Mamba-2 model in the clear on the GPU.

A client that holds the prompt runs the model on it here, the whole prompt in one call, and whoever
fits the polynomials or tunes the weights to them runs and differentiates the same model.  The states
that it leaves start the plain decode (mamba2_payload.decode_tokens); the encrypted decode starts from
empty ones.  The layer is mamba2_payload.layer_step with exact functions
(src/fhemamba/reference.py:182-339): RMSNorm, in_proj, causal convolution and SiLU, the selective scan,
the gate and its norm, out_proj, the residual; the projections are torch's unless they are asked for in
8-bit integers, the rest clear.py's kernels.

    python -m fhemamba_amd.mamba2_clear PAYLOAD RESULT [--prompt-tokens K] [--dtype float32|bfloat16]
        [--int8] [--top N] [--beams K] [--states FILE]

runs a payload's test embeddings: the first K (default: all but one) in one call, the others token by
token from the states that it leaves, checks every final hidden vector against the payload's exact
reference, and writes a fhemamba-m2-clear-result-v1 report.  With a client head in the payload the
report has the log probability of the greedy token, the entropy and the N likeliest tokens of each
step, and with --beams the K best continuations of the payload's prompt by a beam search.  --states
writes the carried states (ssm_<layer> [heads][head_dim][states], fifo_<layer> [taps - 1][channels]) as a
.npz file.  Exit code 1: a result is further than the tolerance.
"""
from __future__ import annotations

import argparse
import json
import sys
import time
from dataclasses import dataclass
from typing import NamedTuple, Optional

import numpy as np
import torch

from . import clear
from .mamba2_payload import ChainPayload, LayerPayload, LayerState, read_chain_payload

# Relative 2-norm error of a final hidden vector: float32 sums over a layer's thousands of terms, or
# bfloat16 activations, each rounding 2^-8, through the layers' residuals.
TOLERANCE = {torch.float32: 1e-4, torch.bfloat16: 5e-2}
# The same with projections in 8 bits: an operand's error is max / (127 sqrt(12)), 0.7% of rows whose largest
# is three times their size, both operands' 1%; two products a layer, 7% over 24 layers, and what the gates
# and exponentials make of it.
INT8_TOLERANCE = 2e-1


@dataclass
class State:
    """One layer's carried state: ssm [rows, heads, head_dim, states] float32 and the convolution's last
    inputs [rows, taps - 1, channels], oldest first; a row a sequence (or a request's slot)."""
    ssm: torch.Tensor
    conv: torch.Tensor


def _project(x: torch.Tensor, weight, bias=None) -> torch.Tensor:
    """x times a table's transpose, in x's type; the table in x's type or 8-bit rows."""
    if isinstance(weight, clear.Int8Rows):
        return clear.int8_linear(x, weight.values, weight.scale, bias)
    out = x @ weight.t()
    return out if bias is None else (out.float() + bias).to(x.dtype)


def _next_norm(hidden, update, weight, eps: float, dtype: torch.dtype) -> tuple:
    """(the norm of hidden + update in dtype, the sum); no update yet: None."""
    if hidden.dtype == torch.float64:  # a caller's own: the kernels' streams are of 32 bits or 16
        hidden = hidden if update is None else hidden + update
        return (hidden * torch.rsqrt(hidden.square().mean(-1, keepdim=True) + eps) * weight).to(dtype), hidden
    if update is None:
        return clear.rms_norm(hidden, weight, eps=eps, dtype=dtype), hidden
    return clear.add_norm(hidden, update, weight, eps=eps)


def _table(values, dtype: torch.dtype, device, int8: bool):
    if int8:
        return clear.quantize_rows(torch.as_tensor(values, dtype=torch.float32, device=device))
    return torch.as_tensor(values, dtype=dtype, device=device)


class Layer:
    """A payload layer's weights on the GPU; projections in the model's type or 8 bits, the others float32."""

    PROJECTIONS = ("in_proj_w", "out_proj_w")
    OTHERS = ("conv_w", "conv_b", "dt_bias", "a_log", "d_skip", "block_norm_w", "gated_norm_w")

    def __init__(self, lay: LayerPayload, dtype: torch.dtype, device, int8: bool = False):
        self.shape = lay
        self.weights = {k: _table(lay.t(k), dtype, device, int8) for k in self.PROJECTIONS}
        self.weights.update({k: torch.as_tensor(lay.t(k), dtype=torch.float32, device=device) for k in self.OTHERS})

    def __call__(self, normed: torch.Tensor, state: Optional[State], mixer) -> tuple:
        """normed [.., d_model], the layer's input behind its norm -> (what the layer adds to the residual, state);
        `mixer` runs the convolution and the scan."""
        w, s = self.weights, self.shape
        proj = _project(normed, w["in_proj_w"])
        z, inputs, dt = torch.split(proj, [s.d_inner, s.conv_dim, s.num_heads], dim=-1)
        write = torch.nn.functional.softplus(dt.float() + w["dt_bias"])
        y, state = mixer(self, inputs, write, write * -torch.exp(w["a_log"]), state)
        gated = clear.rms_norm(y.flatten(-2), w["gated_norm_w"], gate=z, eps=s.eps_gated)
        return _project(gated, w["out_proj_w"]), state

    def split(self, conv: torch.Tensor) -> tuple:
        """x, B and C as views of the convolution's output."""
        s = self.shape
        x, B, C = torch.split(conv, [s.d_inner, s.state_size, s.state_size], dim=-1)
        return x.unflatten(-1, (s.num_heads, s.head_dim)), B.unsqueeze(-2), C.unsqueeze(-2)


class BeamResult(NamedTuple):
    """tokens [requests, beams, steps] int64 and score [requests, beams] float32, best first."""
    tokens: torch.Tensor
    score: torch.Tensor


class ClearMamba2:
    """The layers and the final norm of a chain payload, and its client head if it has one.

    int8: the projections and the head in 8-bit integers with a scale for each output and token, for serving."""

    def __init__(self, chain: ChainPayload, dtype: torch.dtype = torch.float32, device="cuda", int8: bool = False):
        if dtype not in TOLERANCE:
            raise ValueError(f"dtype must be float32 or bfloat16, not {dtype}")
        self.dtype, self.device, self.int8 = dtype, torch.device(device), int8
        self.layers = [Layer(lay, dtype, device, int8) for lay in chain.layers]
        self.norm_eps = chain.final_norm_eps
        self.norm_w = torch.as_tensor(chain.final_norm_w, dtype=torch.float32, device=device)
        self.embedding = self.head = self.head_bias = None
        ar = chain.autoregressive
        if ar is not None:
            self.embedding = torch.as_tensor(ar.embedding_w, dtype=torch.float32, device=device)
            if ar.lm_head_w is None and not int8:
                self.head = self.embedding.to(dtype)
            else:
                self.head = _table(ar.embedding_w if ar.lm_head_w is None else ar.lm_head_w, dtype, device, int8)
            if ar.lm_head_b is not None:
                self.head_bias = torch.as_tensor(ar.lm_head_b, dtype=torch.float32, device=device)

    def parameters(self) -> list:
        """The layers' and the final norm's weights (the head and the embeddings stay as they are)."""
        if self.int8:
            raise ValueError("a model in 8-bit integers is not trained")
        return [v for lay in self.layers for v in lay.weights.values()] + [self.norm_w]

    def zero_states(self, rows: int) -> list:
        """States of `rows` sequences or slots, as step() updates them in place."""
        out = []
        for lay in self.layers:
            s = lay.shape
            out.append(State(torch.zeros(rows, s.num_heads, s.head_dim, s.state_size, device=self.device),
                             torch.zeros(rows, s.conv_kernel - 1, s.conv_dim, dtype=self.dtype, device=self.device)))
        return out

    def _run(self, hidden, states, mixer) -> tuple:
        """Residual stream [.., d_model] -> (final normed hidden, states), both of 32 bits; a stream of 64 stays one."""
        hidden = hidden if hidden.dtype == torch.float64 else hidden.float()
        update, out = None, []
        for i, lay in enumerate(self.layers):
            normed, hidden = _next_norm(hidden, update, lay.weights["block_norm_w"], lay.shape.eps_block, self.dtype)
            update, state = lay(normed, None if states is None else states[i], mixer)
            out.append(state)
        if update is not None:
            update = update.float()
        return _next_norm(hidden, update, self.norm_w, self.norm_eps, hidden.dtype)[0], out

    def forward(self, embeddings, states=None, *, cu_seqlens=None) -> tuple:
        """Whole sequences [sequences, tokens, d_model] float32, or packed [tokens, d_model] with cu_seqlens,
        from `states` (default zeros): (final normed hidden, the states behind the last tokens).  Embeddings of
        float64 make a residual stream, its norms and the result of 64 bits; what a layer adds is of 32 or 16."""
        def mixer(lay, inputs, write, log_decay, state):
            conv, last = clear.causal_conv(inputs, lay.weights["conv_w"], lay.weights["conv_b"],
                                           initial_state=None if state is None else state.conv,
                                           cu_seqlens=cu_seqlens, return_state=True)
            y, ssm = clear.ssm_scan(*self._scan_inputs(lay, conv, write, log_decay), lay.weights["d_skip"],
                                    initial_state=None if state is None else state.ssm, cu_seqlens=cu_seqlens,
                                    return_state=True)
            return y, State(ssm, last)

        return self._run(embeddings, states, mixer)

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

        return self._run(embeddings, states, mixer)[0]

    def logits(self, hidden):
        if self.head is None:
            raise ValueError("the payload has no client head")
        return _project(hidden.to(self.dtype), self.head, self.head_bias)

    def score(self, hidden, targets, top: int = 0) -> clear.TokenLogprobs:
        """Log probabilities of target tokens, entropies and likeliest tokens at each hidden vector."""
        return clear.token_logprobs(self.logits(hidden), targets, top=top)

    def _rows(self, ids):
        """Rows of the embeddings' table: ids below 0 count from its end.  Those that then are below 0 still become very
        large numbers: no row, rather than padding."""
        if ids.dtype != torch.int64:
            raise ValueError(f"ids must be of type torch.int64, not {ids.dtype}")
        return torch.where(ids < 0, (ids + self.embedding.shape[0]) & (2 ** 63 - 1), ids)

    def embed(self, ids):
        """Embeddings of token ids; those below 0 count from the table's end.  One outside of it gives NaN."""
        return clear.embed(self.embedding, self._rows(ids))

    def _check(self, rows):
        """Starts to look for rows that the table does not have; a call of what is returned waits for the answer, not
        for work begun in between, and raises ValueError.  A capture waits for nothing: no check in there."""
        if rows.numel() == 0 or torch.cuda.is_current_stream_capturing():
            return lambda: None
        largest = torch.empty((), dtype=torch.int64, pin_memory=True)
        largest.copy_(rows.max(), non_blocking=True)
        answered = torch.cuda.current_stream(rows.device).record_event()

        def wait():
            answered.synchronize()
            if largest >= self.embedding.shape[0]:
                raise ValueError(f"ids outside of the table of {self.embedding.shape[0]} embeddings")
        return wait

    @torch.no_grad()
    def beam_search(self, ids, steps: int, *, beams: int = 4, end: Optional[int] = None, cu_seqlens=None) -> BeamResult:
        """The `beams` (at most 32) continuations of `steps` tokens of each prompt that a beam search finds.

        ids [requests, tokens], or packed [tokens] with cu_seqlens, each prompt one token or more.  A beam that
        has taken the token `end` goes on with it at no cost.  The score is the sum of the tokens' log
        probabilities.  Prompts without a token and ids outside of the table raise ValueError, for which the call
        waits for the GPU before the search (not in a capture)."""
        if self.head is None:
            raise ValueError("the payload has no client head")
        if steps < 1 or ids.shape[-1] < 1:
            raise ValueError("steps must be 1 or more, and so must a prompt's tokens")
        rows = self._rows(ids)
        checked = self._check(rows)
        if cu_seqlens is not None and not torch.cuda.is_current_stream_capturing():
            clear._offsets(cu_seqlens, ids)
            ends = cu_seqlens.tolist()
            if ends[0] < 0 or ends[-1] > ids.shape[0] or any(a >= b for a, b in zip(ends, ends[1:])):
                raise ValueError(f"cu_seqlens must give each prompt one token or more of the {ids.shape[0]}")
        checked()
        hidden, states = self.forward(clear.embed(self.embedding, rows), cu_seqlens=cu_seqlens)
        last = hidden[:, -1] if cu_seqlens is None else hidden[cu_seqlens[1:].long() - 1]
        requests = last.shape[0]
        score, parent, token = clear.beam_select(self.logits(last).unsqueeze(1), last.new_zeros(requests, 1), beams)
        states = [State(s.ssm.repeat_interleave(beams, 0), s.conv.repeat_interleave(beams, 0)) for s in states]
        held = [t for s in states for t in (s.ssm, s.conv)]
        tokens = token.long().unsqueeze(-1)
        finished = None if end is None else token == end
        for _ in range(steps - 1):
            hidden = self.step(clear.embed(self.embedding, tokens[..., -1].reshape(-1)), states)
            score, parent, token = clear.beam_select(self.logits(hidden).unflatten(0, (requests, beams)), score,
                                                     finished=finished, end=end)
            clear.reorder_states(held, parent)
            parent, token = parent.long(), token.long()
            tokens = torch.cat([tokens.gather(1, parent.unsqueeze(-1).expand(tokens.shape)), token.unsqueeze(-1)], -1)
            if end is not None:
                finished = token == end  # a finished beam's only token is `end`
        return BeamResult(tokens, score)

    def loss(self, ids, *, cu_seqlens=None):
        """Mean negative log probability of each token's successor; ids [sequences, tokens], or packed, where
        tokens outside of every sequence take no part.  Ids outside of the table raise ValueError, for which the
        call waits until the GPU has seen them (in a capture: NaN)."""
        rows = self._rows(ids)
        checked = self._check(rows)
        hidden, _ = self.forward(clear.embed(self.embedding, rows), cu_seqlens=cu_seqlens)
        targets = torch.cat([ids[..., 1:], torch.full_like(ids[..., :1], -1)], dim=-1)
        if cu_seqlens is not None:  # neither a sequence's last token nor one outside of all has a successor
            begins, ends = cu_seqlens[:-1].long(), cu_seqlens[1:].long()
            at = torch.arange(ids.shape[0], device=ids.device)
            own = torch.searchsorted(ends, at, right=True).clamp(max=ends.shape[0] - 1)  # the first that ends behind it
            targets = torch.where((at >= begins[own]) & (at + 1 < ends[own]), targets, -1)
        scored = self.score(hidden, targets).logprob
        checked()
        return -scored.sum() / (targets >= 0).sum().clamp(min=1)


def layer_states(states, row: int = 0) -> list:
    """One row of the states as mamba2_payload.LayerState, the start of a plain decode."""
    return [LayerState(s.ssm[row].double().cpu().numpy(), list(s.conv[row].double().cpu().numpy())) for s in states]


def run(chain: ChainPayload, *, prompt_tokens: Optional[int] = None, dtype=torch.float32, top: int = 5,
        states_file: Optional[str] = None, int8: bool = False, beams: int = 0) -> dict:
    model = ClearMamba2(chain, dtype, int8=int8)
    if beams and chain.autoregressive is None:
        raise ValueError("a beam search needs the payload's client head and prompt")
    tolerance = INT8_TOLERANCE if int8 else TOLERANCE[dtype]
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
                  "relative_errors": [float(e) for e in errors], "tolerance": tolerance,
                  "passed": bool(np.all(errors <= tolerance))}
        if int8:
            report["int8"] = True
        if model.head is not None:
            greedy = model.logits(final).argmax(-1)
            scored = model.score(final, greedy, min(top, chain.autoregressive.vocab, clear.MAX_TOP))
            report["head"] = {"greedy": greedy.tolist(), "logprob": scored.logprob.tolist(),
                              "entropy": scored.entropy.tolist()}
            if scored.top_index is not None:
                report["head"].update(top_index=scored.top_index.tolist(), top_logprob=scored.top_logprob.tolist())
        if beams:
            ar = chain.autoregressive
            found = model.beam_search(torch.as_tensor([ar.prompt_ids], device=model.device), ar.generate_tokens,
                                      beams=beams)
            report["beams"] = {"tokens": found.tokens[0].tolist(), "score": found.score[0].tolist()}
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
    ap.add_argument("--int8", action="store_true", help="projections and head in 8-bit integers")
    ap.add_argument("--top", type=int, default=5)
    ap.add_argument("--beams", type=int, default=0, help="continuations of the payload's prompt by a beam search")
    ap.add_argument("--states", default=None)
    args = ap.parse_args(argv)
    report = run(read_chain_payload(args.payload), prompt_tokens=args.prompt_tokens,
                 dtype=getattr(torch, args.dtype), top=args.top, states_file=args.states, int8=args.int8,
                 beams=args.beams)
    with open(args.result, "w") as f:
        json.dump(report, f, indent=1)
    print(json.dumps({k: v for k, v in report.items() if k != "head"}))
    return 0 if report["passed"] else 1


if __name__ == "__main__":
    sys.exit(main())
