"""Mamba-2 in the clear on the GPU: the operators that a layer and its head are made of.

The encrypted decode evaluates one token at a time under polynomials.  What the client runs on its
own prompt, and whoever fits those polynomials or tunes the model to them, is the same model in
the clear (the reference does it in PyTorch on the host, src/fhemamba/reference.py:182-339):

  ssm_scan        the selective scan over whole sequences, with its gradients
  ssm_step        one token of each request on a cache of states
  causal_conv     the causal convolution before it, with its gradients
  causal_conv_step
  token_logprobs  log probabilities of given tokens, entropy and likeliest tokens, with gradients

They take torch tensors on the GPU, run libfhecore's kernels on torch's current stream and return
without waiting; inputs made on another stream need the usual synchronisation.  Activations are
float32 or bfloat16 (float16 products of the scan leave its range), gates, states and weights
float32.  Rows are read where they lie: any strides, as long as the last axis is contiguous (else it
is copied); 16-byte aligned rows are read fastest.

Sequences are [sequence, token, ...], or packed as [token, ...] with cu_seqlens, int32 offsets on the
GPU: tokens cu_seqlens[i] .. cu_seqlens[i + 1] are sequence i, which may be empty; tokens outside of
every sequence give zeros.  Nothing crosses from one sequence into another.  A number that is not
finite makes what depends on it not finite, and may do the same to other tokens of the 64 around it
in its own sequence.  The gradients' sums have a fixed order: equal inputs give equal bits.
"""
from __future__ import annotations

import ctypes
import struct
from typing import NamedTuple, Optional

import torch

from . import _lib

MAX_STATES, MAX_TAPS, MAX_TOP = 128, 8, 32
_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
# include/fhecore.h's structures: a strided tensor is an address and three strides
_STRIDED = "Q3q"
_SCAN = struct.Struct("=6IqQ" + 5 * _STRIDED + "2Q")
_SCAN_GRADS = struct.Struct("=" + _STRIDED + "8Q")
_STEP = struct.Struct("=7I4xQ" + 5 * _STRIDED + "2Q")
_CONV = struct.Struct("=4IqQ" + _STRIDED + "3Qi4x")
_CONV_GRADS = struct.Struct("=" + _STRIDED + "5Q")
_CONV_STEP = struct.Struct("=5I4xQ" + _STRIDED + "3Qi4x")
_LOGPROB = struct.Struct("=2I3q2Q")
_LOGPROB_OUT = struct.Struct("=6Q")


class _Device:
    """Makes a tensor's device current where it is not, for one call."""

    def __init__(self, t: torch.Tensor):
        self.index = t.device.index
        self.other = None

    def __enter__(self):
        if self.index != torch.cuda.current_device():
            self.other = torch.cuda.device(self.index)
            self.other.__enter__()
        return torch.cuda.current_stream().cuda_stream

    def __exit__(self, *exc):
        if self.other is not None:
            self.other.__exit__(*exc)


def _need(ok, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _gpu(name: str, t, dtypes, shape, like: torch.Tensor) -> None:
    _need(isinstance(t, torch.Tensor), f"{name} must be a tensor")
    _need(t.device == like.device, f"{name} is on {t.device}, not {like.device}")
    _need(t.dtype in dtypes, f"{name} must be of type {' or '.join(str(d) for d in dtypes)}, not {t.dtype}")
    _need(tuple(t.shape) == tuple(shape), f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def _first(name: str, t, dims) -> None:
    _need(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a tensor on the GPU")
    _need(t.dtype in _DTYPES, f"{name} must be float32 or bfloat16, not {t.dtype}")
    _need(t.dim() in dims, f"{name} must have {' or '.join(str(d) for d in dims)} axes, not {t.dim()}")


_F32 = (torch.float32,)


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """The tensor itself where its last axis is contiguous."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _strides(t: torch.Tensor, packed: bool, inner: int) -> tuple:
    """(address, sequence, token and head strides); `inner` axes follow the token."""
    s = t.stride()
    at = 0 if packed else 1
    return t.data_ptr(), 0 if packed else s[0], s[at], s[at + 1] if inner else 0


def _workspace(entry: str, device, *args) -> tuple:
    size = ctypes.c_size_t()
    _lib.call(entry, *args, ctypes.byref(size))
    return torch.empty(size.value, dtype=torch.uint8, device=device), size.value


def _offsets(cu_seqlens, like: torch.Tensor) -> None:
    _need(isinstance(cu_seqlens, torch.Tensor) and cu_seqlens.dim() == 1 and cu_seqlens.numel() >= 2,
          "cu_seqlens must be a vector of one offset more than there are sequences")
    _gpu("cu_seqlens", cu_seqlens, (torch.int32,), cu_seqlens.shape, like)
    _need(cu_seqlens.is_contiguous(), "cu_seqlens must be contiguous")


# ----------------------------------------------------------------- selective scan
class _ScanArgs:
    """Checked arguments of a scan and their packed form.  Holds what the packed form points to."""

    def __init__(self, x, write, log_decay, B, C, D, initial_state, cu_seqlens):
        packed = cu_seqlens is not None
        _first("x", x, (3,) if packed else (4,))
        lead, (H, P) = x.shape[:-2], x.shape[-2:]
        _need(isinstance(B, torch.Tensor) and B.dim() == x.dim(), f"B must have {x.dim()} axes")
        G, N = B.shape[-2:]
        _need(H >= 1 and P >= 1 and G >= 1 and N >= 1 and H % G == 0,
              f"{H} heads do not divide into {G} groups")
        _need(N <= MAX_STATES, f"{N} states: at most {MAX_STATES}")
        _gpu("B", B, (x.dtype,), (*lead, G, N), x)
        _gpu("C", C, (x.dtype,), (*lead, G, N), x)
        _gpu("write", write, _F32, (*lead, H), x)
        _gpu("log_decay", log_decay, _F32, (*lead, H), x)
        if packed:
            _offsets(cu_seqlens, x)
        self.seqs = cu_seqlens.numel() - 1 if packed else lead[0]
        self.tokens = lead[-1]
        _need(self.seqs >= 1, "no sequences")
        self.state_shape = (self.seqs, H, P, N)
        if D is not None:
            _gpu("D", D, _F32, (H,), x)
            D = D.contiguous()
        if initial_state is not None:
            _gpu("initial_state", initial_state, _F32, self.state_shape, x)
            initial_state = initial_state.contiguous()
        x, B, C = _rows(x), _rows(B), _rows(C)
        self.held = x, write, log_decay, B, C, D, initial_state, cu_seqlens
        self.packed = _SCAN.pack(
            _DTYPES[x.dtype], self.seqs, H, P, N, G, self.tokens, _ptr(cu_seqlens),
            *_strides(x, packed, 1), *_strides(B, packed, 1), *_strides(C, packed, 1),
            *_strides(write, packed, 1), *_strides(log_decay, packed, 1), _ptr(D), _ptr(initial_state))


def _scan_forward(args: _ScanArgs, return_state: bool):
    x = args.held[0]
    with _Device(x) as stream:
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        state = torch.empty(args.state_shape, dtype=torch.float32, device=x.device) if return_state else None
        space, size = _workspace("fhe_ssm_scan_workspace", x.device, args.packed, 0)
        _lib.call("fhe_ssm_scan", args.packed, _ptr(y), _ptr(state), _ptr(space), size, stream)
    return y, state


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, return_state, cu_seqlens, x, write, log_decay, B, C, D, initial_state):
        args = _ScanArgs(x, write, log_decay, B, C, D, initial_state, cu_seqlens)
        ctx.save_for_backward(x, write, log_decay, B, C, D, initial_state, cu_seqlens)
        ctx.set_materialize_grads(False)
        return _scan_forward(args, return_state)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dstate):
        x, write, log_decay, B, C, D, initial_state, cu_seqlens = ctx.saved_tensors
        args = _ScanArgs(x, write, log_decay, B, C, D, initial_state, cu_seqlens)
        dy = torch.zeros_like(x) if dy is None else _rows(dy)
        dstate = None if dstate is None else dstate.contiguous()

        def new(like, wanted=True):
            return torch.empty(like.shape, dtype=like.dtype, device=x.device) if wanted else None

        with _Device(x) as stream:
            dx, dw, dg, dB, dC = (new(t) for t in (x, write, log_decay, B, C))
            dD = None if D is None else new(D, ctx.needs_input_grad[7])
            dh = None if initial_state is None else new(initial_state, ctx.needs_input_grad[8])
            grads = _SCAN_GRADS.pack(
                *_strides(dy, cu_seqlens is not None, 1), _ptr(dstate), _ptr(dx), _ptr(dw), _ptr(dg), _ptr(dB),
                _ptr(dC), _ptr(dD), _ptr(dh))
            space, size = _workspace("fhe_ssm_scan_workspace", x.device, args.packed, 1)
            _lib.call("fhe_ssm_scan_backward", args.packed, grads, _ptr(space), size, stream)
        return None, None, dx, dw, dg, dB, dC, dD, dh


def ssm_scan(x, write, log_decay, B, C, D=None, *, initial_state=None, cu_seqlens=None,
             return_state: bool = False):
    """h_t = exp(log_decay_t) h_{t-1} + (write_t x_t) B_t^T,  y_t = h_t C_t + D x_t  for every head.

    x [.., heads, head_dim], B and C [.., groups, states] of its type (a group serves heads / groups
    heads; at most 128 states), write and log_decay [.., heads] and D [heads] float32.  In Mamba-2
    write is dt and log_decay is dt A; -inf forgets the state.  initial_state [sequences, heads,
    head_dim, states] float32 (default zeros).  Returns y, or (y, the last states) with return_state.
    Differentiable in every tensor but cu_seqlens.  Products are of 16-bit pieces with 32-bit sums for
    bfloat16 (the state and the gradients keep at least 16 bits on the way), of 32 bits for float32."""
    tensors = (x, write, log_decay, B, C, D, initial_state)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors):
        y, state = _Scan.apply(return_state, cu_seqlens, *tensors)
    else:
        y, state = _scan_forward(_ScanArgs(*tensors, cu_seqlens), return_state)
    return (y, state) if return_state else y


def _no_grad(name: str, tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{name} has no gradient: call it under torch.no_grad()")


def _slots(slots, requests: int, cache: int, like: torch.Tensor) -> None:
    if slots is None:
        _need(requests <= cache, f"{requests} requests and {cache} rows of the state")
        return
    _gpu("slots", slots, (torch.int32,), (requests,), like)
    _need(slots.is_contiguous(), "slots must be contiguous")


def ssm_step(state, x, write, log_decay, B, C, D=None, *, slots=None):
    """One token of each request: ssm_scan's recurrence on state[slots], updated in place.

    state [cache, heads, head_dim, states] float32 and contiguous, x [requests, heads, head_dim], the
    others alike.  slots [requests] int32 names each request's row (default its own number), no row
    twice; a slot outside of the cache is padding: its y is zero and no state changes.  Returns y."""
    _first("x", x, (3,))
    R, H, P = x.shape
    _need(isinstance(B, torch.Tensor) and B.dim() == 3, "B must have 3 axes")
    G, N = B.shape[-2:]
    _need(R >= 1, "no requests")
    _need(H >= 1 and P >= 1 and G >= 1 and N >= 1 and H % G == 0, f"{H} heads do not divide into {G} groups")
    _need(N <= MAX_STATES, f"{N} states: at most {MAX_STATES}")
    _gpu("B", B, (x.dtype,), (R, G, N), x)
    _gpu("C", C, (x.dtype,), (R, G, N), x)
    _gpu("write", write, _F32, (R, H), x)
    _gpu("log_decay", log_decay, _F32, (R, H), x)
    _need(isinstance(state, torch.Tensor) and state.dim() == 4 and state.shape[0] >= 1, "state must have 4 axes")
    _gpu("state", state, _F32, (state.shape[0], H, P, N), x)
    _need(state.is_contiguous(), "state must be contiguous: it is updated in place")
    if D is not None:
        _gpu("D", D, _F32, (H,), x)
        D = D.contiguous()
    _slots(slots, R, state.shape[0], x)
    _no_grad("ssm_step", (state, x, write, log_decay, B, C, D))
    x, B, C = _rows(x), _rows(B), _rows(C)
    with _Device(x) as stream:
        y = torch.empty((R, H, P), dtype=x.dtype, device=x.device)
        args = _STEP.pack(_DTYPES[x.dtype], R, state.shape[0], H, P, N, G, _ptr(slots), *_strides(x, True, 1),
                          *_strides(B, True, 1), *_strides(C, True, 1), *_strides(write, True, 1),
                          *_strides(log_decay, True, 1), _ptr(D), state.data_ptr())
        _lib.call("fhe_ssm_step", args, y.data_ptr(), stream)
    return y


# ----------------------------------------------------------------- causal convolution
class _ConvArgs:
    def __init__(self, x, weight, bias, initial_state, cu_seqlens, silu):
        packed = cu_seqlens is not None
        _first("x", x, (2,) if packed else (3,))
        Cn = x.shape[-1]
        _need(isinstance(weight, torch.Tensor) and weight.dim() == 2, "weight must be [channels, taps]")
        K = weight.shape[1]
        _need(Cn >= 1 and 2 <= K <= MAX_TAPS, f"{K} taps: 2 to {MAX_TAPS}")
        _gpu("weight", weight, _F32, (Cn, K), x)
        weight = weight.contiguous()
        if bias is not None:
            _gpu("bias", bias, _F32, (Cn,), x)
            bias = bias.contiguous()
        if packed:
            _offsets(cu_seqlens, x)
        self.seqs = cu_seqlens.numel() - 1 if packed else x.shape[0]
        _need(self.seqs >= 1, "no sequences")
        self.state_shape = (self.seqs, K - 1, Cn)
        if initial_state is not None:
            _gpu("initial_state", initial_state, (x.dtype,), self.state_shape, x)
            initial_state = initial_state.contiguous()
        x = _rows(x)
        self.held = x, weight, bias, initial_state, cu_seqlens
        self.packed = _CONV.pack(_DTYPES[x.dtype], self.seqs, Cn, K, x.shape[-2], _ptr(cu_seqlens),
                                 *_strides(x, packed, 0), _ptr(weight), _ptr(bias), _ptr(initial_state), int(silu))


def _conv_forward(args: _ConvArgs, return_state: bool):
    x = args.held[0]
    with _Device(x) as stream:
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        state = torch.empty(args.state_shape, dtype=x.dtype, device=x.device) if return_state else None
        _lib.call("fhe_causal_conv", args.packed, _ptr(y), _ptr(state), stream)
    return y, state


class _Conv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, return_state, cu_seqlens, silu, x, weight, bias, initial_state):
        args = _ConvArgs(x, weight, bias, initial_state, cu_seqlens, silu)
        ctx.save_for_backward(x, weight, bias, initial_state, cu_seqlens)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return _conv_forward(args, return_state)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dstate):
        x, weight, bias, initial_state, cu_seqlens = ctx.saved_tensors
        args = _ConvArgs(x, weight, bias, initial_state, cu_seqlens, ctx.silu)
        dy = torch.zeros_like(x) if dy is None else _rows(dy)
        dstate = None if dstate is None else dstate.contiguous()
        with _Device(x) as stream:
            dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            dw = torch.empty(weight.shape, dtype=torch.float32, device=x.device)
            db = None if bias is None else torch.empty(bias.shape, dtype=torch.float32, device=x.device)
            dh = None if initial_state is None else torch.empty(args.state_shape, dtype=x.dtype, device=x.device)
            grads = _CONV_GRADS.pack(*_strides(dy, cu_seqlens is not None, 0), _ptr(dstate), _ptr(dx), _ptr(dw),
                                     _ptr(db), _ptr(dh))
            space, size = _workspace("fhe_causal_conv_workspace", x.device, args.packed)
            _lib.call("fhe_causal_conv_backward", args.packed, grads, _ptr(space), size, stream)
        return None, None, None, dx, dw, db, dh


def causal_conv(x, weight, bias=None, *, initial_state=None, cu_seqlens=None, silu: bool = True,
                return_state: bool = False):
    """y_t = silu(bias + sum_k weight_k x_{t - taps + 1 + k}) for every channel.

    x [.., channels], weight [channels, taps] (2 to 8) and bias [channels] float32.  initial_state
    [sequences, taps - 1, channels] of x's type holds the inputs before each sequence's first, oldest
    first (default zeros).  silu=False leaves the sums as they are.  Returns y, or (y, each sequence's
    last taps - 1 inputs) with return_state.  Differentiable in every tensor but cu_seqlens."""
    tensors = (x, weight, bias, initial_state)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors):
        y, state = _Conv.apply(return_state, cu_seqlens, silu, *tensors)
    else:
        y, state = _conv_forward(_ConvArgs(*tensors, cu_seqlens, silu), return_state)
    return (y, state) if return_state else y


def causal_conv_step(state, x, weight, bias=None, *, silu: bool = True, slots=None):
    """One token of each request: causal_conv on state[slots] [cache, taps - 1, channels], which moves
    on by x [requests, channels] in place.  slots as in ssm_step.  Returns y [requests, channels]."""
    _first("x", x, (2,))
    R, Cn = x.shape
    _need(R >= 1, "no requests")
    _need(isinstance(weight, torch.Tensor) and weight.dim() == 2, "weight must be [channels, taps]")
    K = weight.shape[1]
    _need(Cn >= 1 and 2 <= K <= MAX_TAPS, f"{K} taps: 2 to {MAX_TAPS}")
    _gpu("weight", weight, _F32, (Cn, K), x)
    weight = weight.contiguous()
    if bias is not None:
        _gpu("bias", bias, _F32, (Cn,), x)
        bias = bias.contiguous()
    _need(isinstance(state, torch.Tensor) and state.dim() == 3 and state.shape[0] >= 1, "state must have 3 axes")
    _gpu("state", state, (x.dtype,), (state.shape[0], K - 1, Cn), x)
    _need(state.is_contiguous(), "state must be contiguous: it is updated in place")
    _slots(slots, R, state.shape[0], x)
    _no_grad("causal_conv_step", (state, x, weight, bias))
    x = _rows(x)
    with _Device(x) as stream:
        y = torch.empty((R, Cn), dtype=x.dtype, device=x.device)
        args = _CONV_STEP.pack(_DTYPES[x.dtype], R, state.shape[0], Cn, K, _ptr(slots), *_strides(x, True, 0),
                               _ptr(weight), _ptr(bias), state.data_ptr(), int(silu))
        _lib.call("fhe_causal_conv_step", args, y.data_ptr(), stream)
    return y


# ----------------------------------------------------------------- log probabilities
class TokenLogprobs(NamedTuple):
    """logprob and entropy [..] float32; top_logprob [.., top] float32 and top_index [.., top] int32,
    or None where none were asked for."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprob: Optional[torch.Tensor]
    top_index: Optional[torch.Tensor]


def _logprob_args(logits, targets, top: int) -> bytes:
    return _LOGPROB.pack(_DTYPES[logits.dtype], top, logits.shape[0], logits.shape[1], logits.stride(0),
                         logits.data_ptr(), _ptr(targets))


def _logprob_forward(logits, targets, top: int):
    rows = logits.shape[0]
    with _Device(logits) as stream:
        stats = torch.empty((4, rows), dtype=torch.float32, device=logits.device)
        best = index = None
        if top:
            best = torch.empty((rows, top), dtype=torch.float32, device=logits.device)
            index = torch.empty((rows, top), dtype=torch.int32, device=logits.device)
        args = _logprob_args(logits, targets, top)
        at = stats.data_ptr()
        out = _LOGPROB_OUT.pack(at, at + 4 * rows, at + 8 * rows, at + 12 * rows, _ptr(best), _ptr(index))
        space, size = _workspace("fhe_token_logprobs_workspace", logits.device, args)
        _lib.call("fhe_token_logprobs", args, out, _ptr(space), size, stream)
    return stats, best, index


class _Logprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top):
        stats, best, index = _logprob_forward(logits, targets, top)
        ctx.save_for_backward(logits, targets, stats[1:])
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(best, index)
        return stats[0], stats[1], best, index

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dlogprob, dentropy, *_):
        logits, targets, stats = ctx.saved_tensors
        at, rows = stats.data_ptr(), logits.shape[0]  # entropy, peak, log sum
        dlogprob, dentropy = (None if d is None else d.contiguous() for d in (dlogprob, dentropy))
        with _Device(logits) as stream:
            grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
            _lib.call("fhe_token_logprobs_backward", _logprob_args(logits, targets, 0), at + 4 * rows,
                      at + 8 * rows, at, _ptr(dlogprob), _ptr(dentropy), _ptr(grad), stream)
        return grad, None, None


def token_logprobs(logits, targets, *, top: int = 0) -> TokenLogprobs:
    """Log softmax of logits [.., vocab] at targets [..] (int64), the entropy of each row's
    distribution, and its `top` (at most 32) likeliest tokens, the lower index first among equals.

    A target below 0 is left out: log probability 0 and no gradient from it; one of vocab or more
    gives NaN.  A logit of -inf is a token that is not allowed; a row of nothing else has log
    probability -inf, entropy 0 and gradient 0.  logprob and entropy are differentiable in logits."""
    _need(isinstance(logits, torch.Tensor) and logits.is_cuda, "logits must be a tensor on the GPU")
    _need(logits.dtype in _DTYPES, f"logits must be float32 or bfloat16, not {logits.dtype}")
    _need(logits.dim() >= 1 and logits.shape[-1] >= 1, "logits must have a vocabulary axis")
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    _gpu("targets", targets, (torch.int64,), lead, logits)
    _need(0 <= top <= min(MAX_TOP, vocab), f"top must be 0 to {min(MAX_TOP, vocab)}")
    flat = _rows(logits.reshape(-1, vocab))
    if flat.shape[0] == 0:
        empty = logits.sum(-1).float()
        return TokenLogprobs(empty, empty, *((empty.new_empty((*lead, top)),
                                              torch.empty((*lead, top), dtype=torch.int32, device=logits.device))
                                             if top else (None, None)))
    if flat.shape[0] > 1 and flat.stride(0) < vocab:  # one row for all
        flat = flat.contiguous()
    targets = targets.reshape(-1).contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        logprob, entropy, best, index = _Logprobs.apply(flat, targets, top)
    else:
        stats, best, index = _logprob_forward(flat, targets, top)
        logprob, entropy = stats[0], stats[1]
    return TokenLogprobs(logprob.reshape(lead), entropy.reshape(lead),
                         None if best is None else best.reshape(*lead, top),
                         None if index is None else index.reshape(*lead, top))
