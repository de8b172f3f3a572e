"""Mamba-2 in the clear on the GPU: the operators that a layer and its head are made of.

The encrypted decode evaluates one token at a time under polynomials.  What the client runs on its
own prompt, and whoever fits those polynomials or tunes the model to them, is the same model in
the clear (the reference does it in PyTorch on the host, src/fhemamba/reference.py:182-339):

  ssm_scan        the selective scan over whole sequences, with its gradients
  ssm_step        one token of each request on a cache of states
  causal_conv     the causal convolution before it, with its gradients
  causal_conv_step
  token_logprobs  log probabilities of given tokens, entropy and likeliest tokens, with gradients
  embed           embeddings of tokens, with the table's gradient
  rms_norm        the norm with or without a gate before it, with gradients
  add_norm        the residual and the next layer's norm, with gradients
  quantize_rows   rows as 8-bit integers and a scale
  int8_linear     projections in 8-bit integers, for serving
  beam_select     the best continuations of a search's beams
  reorder_states  their states follow them

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
Gradients are of reverse mode and first order.
"""
from __future__ import annotations

import ctypes
import struct
from itertools import chain, repeat
from operator import attrgetter
from typing import NamedTuple, Optional

import torch

from . import _lib

MAX_STATES, MAX_TAPS, MAX_TOP, MAX_ROW = 128, 8, 32, 32768
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
_ROWS = struct.Struct("=Qq")  # an address and the elements between rows
_NORM = struct.Struct("=3If2qQqQqQ")
_NORM_GRADS = struct.Struct("=Qq3Q")
_ADD_NORM = struct.Struct("=2If4x2qQqQq2Q")
_ADD_NORM_GRADS = struct.Struct("=QqQq5Q")
_QUANTIZE = struct.Struct("=I4x2qQq")
_INT8 = struct.Struct("=I4x3qQq3Q")
_EMBED = struct.Struct("=If3qQqQ")
_BEAM = struct.Struct("=4I3q3Q")
_BEAM_OUT = struct.Struct("=3Q")

_F32 = (torch.float32,)
# of a tensor that a kernel wrote in place: a backward pass that saved it raises, as after torch's own
_changed = torch.autograd.graph.increment_version
_forward_ad = torch.autograd.forward_ad
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_device_of, _size_of, _is_contiguous = torch.Tensor.get_device, torch.Tensor.size, torch.Tensor.is_contiguous
_requires_grad = attrgetter("requires_grad")


def _run(entry, like: torch.Tensor, *args) -> None:
    """An entry point on the tensor's device and torch's current stream there."""
    index = like.get_device()
    if index == _current_device():
        code = entry(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            code = entry(*args, _raw_stream(index))
    if code:
        _lib.check(code)


# The checks pass in a comparison each; what they say is put together when they fail.
def _gpu(name: str, t, dtypes, shape, like: torch.Tensor) -> None:
    if isinstance(t, torch.Tensor) and t.dtype in dtypes and t.shape == shape and t.device == like.device:
        return
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, not {like.device}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be of type {' or '.join(str(d) for d in dtypes)}, not {t.dtype}")
    raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def _first(name: str, t, dims: int) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a tensor on the GPU")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name} must be float32 or bfloat16, not {t.dtype}")
    if t.dim() != dims:
        raise ValueError(f"{name} must have {dims} axes, not {t.dim()}")


def _axes(name: str, t, dims: int, what: str) -> None:
    if not isinstance(t, torch.Tensor) or t.dim() != dims:
        raise ValueError(f"{name} must {what}")


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """The tensor itself where its last axis is contiguous."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _strides(t: torch.Tensor, packed: bool) -> tuple:
    """(address, sequence, token and head strides) of [sequence, token, head, ..]."""
    s = t.stride()
    return (t.data_ptr(), 0, s[0], s[1]) if packed else (t.data_ptr(), s[0], s[1], s[2])


def _strides2(t: torch.Tensor, packed: bool) -> tuple:
    """The same of [sequence, token, channel]."""
    s = t.stride()
    return (t.data_ptr(), 0, s[0], 0) if packed else (t.data_ptr(), s[0], s[1], 0)


def _workspace(entry, like: torch.Tensor, *args, more: int = 0) -> tuple:
    """(bytes that the entry point asks for and `more` behind them, or None for none; how many it asks for)."""
    size = ctypes.c_size_t()
    code = entry(*args, ctypes.byref(size))
    if code:
        _lib.check(code)
    size = size.value
    return like.new_empty(size + more, dtype=torch.uint8) if size + more else None, size


def _offsets(cu_seqlens, like: torch.Tensor) -> None:
    if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2:
        raise ValueError("cu_seqlens must be a vector of one offset more than there are sequences")
    _gpu("cu_seqlens", cu_seqlens, (torch.int32,), cu_seqlens.shape, like)
    if not cu_seqlens.is_contiguous():
        raise ValueError("cu_seqlens must be contiguous")


def _wants_grad(*tensors) -> bool:
    if getattr(_forward_ad, "_current_level", 0) >= 0:  # within a level of forward-mode derivatives
        for t in tensors:
            if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError("forward-mode derivatives are not available: a tensor has a tangent")
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


# ----------------------------------------------------------------- selective scan
def _heads(H: int, P: int, G: int, N: int) -> None:
    if min(H, P, G, N) < 1 or H % G:
        raise ValueError(f"{H} heads do not divide into {G} groups")
    if N > MAX_STATES:
        raise ValueError(f"{N} states: at most {MAX_STATES}")


def _check_scan(x, write, log_decay, B, C, D, initial_state, cu_seqlens) -> None:
    packed = cu_seqlens is not None
    dims = 3 if packed else 4
    _first("x", x, dims)
    _axes("B", B, dims, f"have {dims} axes")
    lead, (H, P), (G, N) = x.shape[:-2], x.shape[-2:], B.shape[-2:]
    _heads(H, P, G, N)
    _gpu("B", B, (x.dtype,), (*lead, G, N), x)
    _gpu("C", C, (x.dtype,), B.shape, x)
    _gpu("write", write, _F32, (*lead, H), x)
    _gpu("log_decay", log_decay, _F32, (*lead, H), x)
    if packed:
        _offsets(cu_seqlens, x)
    if lead[0] < 1 and not packed:
        raise ValueError("no sequences")
    if D is not None:
        _gpu("D", D, _F32, (H,), x)
    if initial_state is not None:
        seqs = cu_seqlens.numel() - 1 if packed else lead[0]
        _gpu("initial_state", initial_state, _F32, (seqs, H, P, N), x)


def _pack_scan(x, write, log_decay, B, C, D, initial_state, cu_seqlens) -> tuple:
    """(the packed arguments, the state's shape, the tensors that they point to)."""
    packed = cu_seqlens is not None
    x, B, C = _rows(x), _rows(B), _rows(C)
    D = None if D is None else D.contiguous()
    initial_state = None if initial_state is None else initial_state.contiguous()
    (tokens, H, P), (G, N) = x.shape[-3:], B.shape[-2:]
    seqs = cu_seqlens.numel() - 1 if packed else x.shape[0]
    args = _SCAN.pack(
        _DTYPES[x.dtype], seqs, H, P, N, G, tokens, _ptr(cu_seqlens), *_strides(x, packed), *_strides(B, packed),
        *_strides(C, packed), *_strides(write, packed), *_strides(log_decay, packed), _ptr(D), _ptr(initial_state))
    return args, (seqs, H, P, N), (x, B, C, D, initial_state)


def _scan_forward(tensors, return_state: bool):
    x = tensors[0]
    args, state_shape, held = _pack_scan(*tensors)
    y = x.new_empty(x.shape)
    state = x.new_empty(state_shape, dtype=torch.float32) if return_state else None
    space, size = _workspace(_lib.lib.fhe_ssm_scan_workspace, x, args, 0)
    _run(_lib.lib.fhe_ssm_scan, x, args, _ptr(y), _ptr(state), _ptr(space), size)
    return y, state


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, return_state, *tensors):
        ctx.save_for_backward(*tensors)
        ctx.set_materialize_grads(False)
        return _scan_forward(tensors, return_state)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dstate):
        tensors = ctx.saved_tensors
        x, write, log_decay, B, C, D, initial_state, cu_seqlens = tensors
        args, _, held = _pack_scan(*tensors)
        dy = torch.zeros_like(x) if dy is None else _rows(dy)
        dstate = None if dstate is None else dstate.contiguous()

        def new(like, wanted=True):
            if like is None or not wanted:
                return None
            return like.new_empty(like.shape)

        dx, dw, dg, dB, dC = new(x), new(write), new(log_decay), new(B), new(C)
        dD, dh = new(D, ctx.needs_input_grad[6]), new(initial_state, ctx.needs_input_grad[7])
        grads = _SCAN_GRADS.pack(*_strides(dy, cu_seqlens is not None), _ptr(dstate), _ptr(dx), _ptr(dw), _ptr(dg),
                                 _ptr(dB), _ptr(dC), _ptr(dD), _ptr(dh))
        space, size = _workspace(_lib.lib.fhe_ssm_scan_workspace, x, args, 1)
        _run(_lib.lib.fhe_ssm_scan_backward, x, args, grads, _ptr(space), size)
        return None, dx, dw, dg, dB, dC, dD, dh, None


def ssm_scan(x, write, log_decay, B, C, D=None, *, initial_state=None, cu_seqlens=None,
             return_state: bool = False):
    """h_t = exp(log_decay_t) h_{t-1} + (write_t x_t) B_t^T,  y_t = h_t C_t + D x_t  for every head.

    x [.., heads, head_dim], B and C [.., groups, states] of its type (a group serves heads / groups
    heads; at most 128 states), write and log_decay [.., heads] and D [heads] float32.  In Mamba-2
    write is dt and log_decay is dt A; -inf forgets the state.  initial_state [sequences, heads,
    head_dim, states] float32 (default zeros).  Returns y, or (y, the last states) with return_state.
    Differentiable in every tensor but cu_seqlens.  Products are of 16-bit pieces with 32-bit sums for
    bfloat16 (the state and the gradients keep at least 16 bits on the way), of 32 bits for float32."""
    tensors = (x, write, log_decay, B, C, D, initial_state, cu_seqlens)
    _check_scan(*tensors)
    if _wants_grad(*tensors):
        y, state = _Scan.apply(return_state, *tensors)
    else:
        y, state = _scan_forward(tensors, return_state)
    return (y, state) if return_state else y


def _slots(slots, requests: int, state: torch.Tensor, like: torch.Tensor) -> None:
    if requests < 1:
        raise ValueError("no requests")
    if not state.is_contiguous():
        raise ValueError("state must be contiguous: it is updated in place")
    if slots is None:
        if requests > state.shape[0]:
            raise ValueError(f"{requests} requests and {state.shape[0]} rows of the state")
        return
    _gpu("slots", slots, (torch.int32,), (requests,), like)
    if not slots.is_contiguous():
        raise ValueError("slots must be contiguous")


def ssm_step(state, x, write, log_decay, B, C, D=None, *, slots=None):
    """One token of each request: ssm_scan's recurrence on state[slots], updated in place.

    state [cache, heads, head_dim, states] float32 and contiguous, x [requests, heads, head_dim], the
    others alike.  slots [requests] int32 names each request's row (default its own number), no row
    twice; a slot outside of the cache is padding: its y is zero and no state changes.  Returns y.
    A backward pass that needs the state as it was before raises, as after torch's in-place operations."""
    _first("x", x, 3)
    _axes("B", B, 3, "have 3 axes")
    _axes("state", state, 4, "have 4 axes")
    (R, H, P), (G, N) = x.shape, B.shape[-2:]
    _heads(H, P, G, N)
    _gpu("B", B, (x.dtype,), (R, G, N), x)
    _gpu("C", C, (x.dtype,), B.shape, x)
    _gpu("write", write, _F32, (R, H), x)
    _gpu("log_decay", log_decay, _F32, (R, H), x)
    _gpu("state", state, _F32, (state.shape[0], H, P, N), x)
    if D is not None:
        _gpu("D", D, _F32, (H,), x)
        D = D.contiguous()
    _slots(slots, R, state, x)
    if _wants_grad(state, x, write, log_decay, B, C, D):
        raise ValueError("ssm_step has no gradient: call it under torch.no_grad()")
    x, B, C = _rows(x), _rows(B), _rows(C)
    y = x.new_empty((R, H, P))
    args = _STEP.pack(_DTYPES[x.dtype], R, state.shape[0], H, P, N, G, _ptr(slots), *_strides(x, True),
                      *_strides(B, True), *_strides(C, True), *_strides(write, True), *_strides(log_decay, True),
                      _ptr(D), state.data_ptr())
    _run(_lib.lib.fhe_ssm_step, x, args, y.data_ptr())
    _changed(state)
    return y


# ----------------------------------------------------------------- causal convolution
def _check_weight(weight, bias, x: torch.Tensor) -> int:
    _axes("weight", weight, 2, "be [channels, taps]")
    channels, taps = x.shape[-1], weight.shape[1]
    if channels < 1 or not 2 <= taps <= MAX_TAPS:
        raise ValueError(f"{taps} taps: 2 to {MAX_TAPS}")
    _gpu("weight", weight, _F32, (channels, taps), x)
    if bias is not None:
        _gpu("bias", bias, _F32, (channels,), x)
    return taps


def _check_conv(x, weight, bias, initial_state, cu_seqlens) -> None:
    packed = cu_seqlens is not None
    _first("x", x, 2 if packed else 3)
    taps = _check_weight(weight, bias, x)
    if packed:
        _offsets(cu_seqlens, x)
    seqs = cu_seqlens.numel() - 1 if packed else x.shape[0]
    if seqs < 1:
        raise ValueError("no sequences")
    if initial_state is not None:
        _gpu("initial_state", initial_state, (x.dtype,), (seqs, taps - 1, x.shape[-1]), x)


def _pack_conv(x, weight, bias, initial_state, cu_seqlens, silu) -> tuple:
    """(the packed arguments, the state's shape, the tensors that they point to)."""
    packed = cu_seqlens is not None
    x, weight = _rows(x), weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    initial_state = None if initial_state is None else initial_state.contiguous()
    seqs = cu_seqlens.numel() - 1 if packed else x.shape[0]
    channels, taps = weight.shape
    args = _CONV.pack(_DTYPES[x.dtype], seqs, channels, taps, x.shape[-2], _ptr(cu_seqlens), *_strides2(x, packed),
                      _ptr(weight), _ptr(bias), _ptr(initial_state), int(silu))
    return args, (seqs, taps - 1, channels), (x, weight, bias, initial_state)


def _conv_forward(tensors, silu: bool, return_state: bool):
    x = tensors[0]
    args, state_shape, held = _pack_conv(*tensors, silu)
    y = x.new_empty(x.shape)
    state = x.new_empty(state_shape) if return_state else None
    _run(_lib.lib.fhe_causal_conv, x, args, _ptr(y), _ptr(state))
    return y, state


class _Conv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, return_state, silu, *tensors):
        ctx.save_for_backward(*tensors)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return _conv_forward(tensors, silu, return_state)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dstate):
        tensors = ctx.saved_tensors
        x, weight, bias, initial_state, cu_seqlens = tensors
        args, state_shape, held = _pack_conv(*tensors, ctx.silu)
        dy = torch.zeros_like(x) if dy is None else _rows(dy)
        dstate = None if dstate is None else dstate.contiguous()
        dx = x.new_empty(x.shape)
        dw = weight.new_empty(weight.shape)
        db = None if bias is None else bias.new_empty(bias.shape)
        dh = None if initial_state is None else x.new_empty(state_shape)
        grads = _CONV_GRADS.pack(*_strides2(dy, cu_seqlens is not None), _ptr(dstate), _ptr(dx), _ptr(dw), _ptr(db),
                                 _ptr(dh))
        space, size = _workspace(_lib.lib.fhe_causal_conv_workspace, x, args)
        _run(_lib.lib.fhe_causal_conv_backward, x, args, grads, _ptr(space), size)
        return None, None, dx, dw, db, dh, None


def causal_conv(x, weight, bias=None, *, initial_state=None, cu_seqlens=None, silu: bool = True,
                return_state: bool = False):
    """y_t = silu(bias + sum_k weight_k x_{t - taps + 1 + k}) for every channel.

    x [.., channels], weight [channels, taps] (2 to 8) and bias [channels] float32.  initial_state
    [sequences, taps - 1, channels] of x's type holds the inputs before each sequence's first, oldest
    first (default zeros).  silu=False leaves the sums as they are.  Returns y, or (y, each sequence's
    last taps - 1 inputs) with return_state.  Differentiable in every tensor but cu_seqlens."""
    tensors = (x, weight, bias, initial_state, cu_seqlens)
    _check_conv(*tensors)
    if _wants_grad(*tensors):
        y, state = _Conv.apply(return_state, silu, *tensors)
    else:
        y, state = _conv_forward(tensors, silu, return_state)
    return (y, state) if return_state else y


def causal_conv_step(state, x, weight, bias=None, *, silu: bool = True, slots=None):
    """One token of each request: causal_conv on state[slots] [cache, taps - 1, channels], which moves
    on by x [requests, channels] in place.  slots as in ssm_step.  Returns y [requests, channels]."""
    _first("x", x, 2)
    _axes("state", state, 3, "have 3 axes")
    taps = _check_weight(weight, bias, x)
    R, channels = x.shape
    _gpu("state", state, (x.dtype,), (state.shape[0], taps - 1, channels), x)
    _slots(slots, R, state, x)
    if _wants_grad(state, x, weight, bias):
        raise ValueError("causal_conv_step has no gradient: call it under torch.no_grad()")
    x, weight = _rows(x), weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    y = x.new_empty((R, channels))
    args = _CONV_STEP.pack(_DTYPES[x.dtype], R, state.shape[0], channels, taps, _ptr(slots), *_strides2(x, True),
                           _ptr(weight), _ptr(bias), state.data_ptr(), int(silu))
    _run(_lib.lib.fhe_causal_conv_step, x, args, y.data_ptr())
    _changed(state)
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


def _logprob_forward(logits, targets, top: int, keep: bool):
    """(log probability, entropy, best, index, each a tensor of its own, and with `keep` the peaks and the logs
    of the sums for the backward pass)."""
    rows = logits.shape[0]
    logprob = logits.new_empty(rows, dtype=torch.float32)
    entropy = logits.new_empty(rows, dtype=torch.float32)
    best = index = stats = None
    if top:
        best = logits.new_empty((rows, top), dtype=torch.float32)
        index = logits.new_empty((rows, top), dtype=torch.int32)
    args = _logprob_args(logits, targets, top)
    space, size = _workspace(_lib.lib.fhe_token_logprobs_workspace, logits, args, more=0 if keep else 8 * rows)
    if keep:
        stats = logits.new_empty((2, rows), dtype=torch.float32)
    at = stats.data_ptr() if keep else space.data_ptr() + size  # a workspace is whole words
    out = _LOGPROB_OUT.pack(logprob.data_ptr(), entropy.data_ptr(), at, at + 4 * rows, _ptr(best), _ptr(index))
    _run(_lib.lib.fhe_token_logprobs, logits, args, out, space.data_ptr(), size)
    return logprob, entropy, best, index, stats


class _Logprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top):
        logprob, entropy, best, index, stats = _logprob_forward(logits, targets, top, True)
        ctx.save_for_backward(logits, targets, entropy, stats)
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(best, index)
        return logprob, entropy, best, index

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dlogprob, dentropy, *_):
        logits, targets, entropy, stats = ctx.saved_tensors
        peak, rows = stats.data_ptr(), logits.shape[0]
        dlogprob, dentropy = (None if d is None else d.contiguous() for d in (dlogprob, dentropy))
        grad = logits.new_empty(logits.shape)
        _run(_lib.lib.fhe_token_logprobs_backward, logits, _logprob_args(logits, targets, 0), peak, peak + 4 * rows,
             entropy.data_ptr(), _ptr(dlogprob), _ptr(dentropy), _ptr(grad))
        return grad, None, None


def token_logprobs(logits, targets, *, top: int = 0) -> TokenLogprobs:
    """Log softmax of logits [.., vocab] at targets [..] (int64), the entropy of each row's
    distribution, and its `top` (at most 32) likeliest tokens, the lower index first among equals.

    A target below 0 is left out: log probability 0 and no gradient from it; one of vocab or more
    gives NaN.  A logit of -inf is a token that is not allowed; a row of nothing else has log
    probability -inf, entropy 0 and gradient 0.  A NaN makes its row NaN.  logprob and entropy are
    differentiable in logits; the backward pass needs the entropy as it was."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise ValueError("logits must be a tensor on the GPU")
    if logits.dtype not in _DTYPES:
        raise ValueError(f"logits must be float32 or bfloat16, not {logits.dtype}")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("logits must have a vocabulary axis")
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    _gpu("targets", targets, (torch.int64,), lead, logits)
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"top must be 0 to {min(MAX_TOP, vocab)}")
    flat = logits.dim() == 2
    rows = _rows(logits if flat else logits.reshape(-1, vocab))
    if rows.shape[0] == 0:
        empty = logits.sum(-1).float()
        best = index = None
        if top:
            best = empty.new_empty((*lead, top))
            index = torch.empty((*lead, top), dtype=torch.int32, device=logits.device)
        return TokenLogprobs(empty, empty.clone(), best, index)
    if rows.shape[0] > 1 and rows.stride(0) < vocab:  # one row for all
        rows = rows.contiguous()
    targets = (targets if flat else targets.reshape(-1)).contiguous()
    if _wants_grad(logits):
        logprob, entropy, best, index = _Logprobs.apply(rows, targets, top)
    else:
        logprob, entropy, best, index, _ = _logprob_forward(rows, targets, top, False)
    if flat:
        return TokenLogprobs(logprob, entropy, best, index)
    return TokenLogprobs(logprob.reshape(lead), entropy.reshape(lead),
                         None if best is None else best.reshape(*lead, top),
                         None if index is None else index.reshape(*lead, top))


# ----------------------------------------------------------------- rows of channels
def _leading(name: str, t) -> None:
    """A float tensor [.., channels] on the GPU."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a tensor on the GPU")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name} must be float32 or bfloat16, not {t.dtype}")
    if t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError(f"{name} must have an axis of channels")


def _flat(t: torch.Tensor) -> torch.Tensor:
    """[rows, channels] with contiguous rows."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return _rows(t)


def _row(t: Optional[torch.Tensor]) -> tuple:
    return (0, 0) if t is None else (t.data_ptr(), t.stride(0))


def _like(t: torch.Tensor) -> torch.Tensor:
    """A new contiguous tensor of t's shape and type."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _eps(eps) -> float:
    if not 0.0 <= eps < 3.4e38:
        raise ValueError("eps must be 0 or more and finite")
    return eps


def _narrower(name: str, dtype, like: torch.Tensor):
    if dtype is None:
        return like.dtype
    if dtype not in (like.dtype, torch.bfloat16):
        raise ValueError(f"{name} must be {like.dtype} or torch.bfloat16, not {dtype}")
    return dtype


def _first_order(backward):
    """A backward pass whose results cannot be differentiated again.  Where no graph of it is asked for, they are not
    looked at, which is 5 us of a call."""
    marked = torch.autograd.function.once_differentiable(backward)
    return lambda ctx, *grads: marked(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)


# ----------------------------------------------------------------- norms
def _pack_norm(x, weight, gate, groups, eps, dtype) -> tuple:
    """(the packed arguments, the tensors that they point to)."""
    x, weight = _flat(x), weight.contiguous()
    rows, channels = x.shape
    at = row = 0
    if gate is not None:
        gate = _flat(gate)
        at, row = gate.data_ptr(), gate.stride(0)
    args = _NORM.pack(_DTYPES[x.dtype], _DTYPES[dtype], groups, eps, rows, channels, x.data_ptr(), x.stride(0), at, row,
                      weight.data_ptr())
    return args, (x, weight, gate)


def _norm_forward(x, weight, gate, groups, eps, dtype):
    args, held = _pack_norm(x, weight, gate, groups, eps, dtype)
    y = _like(x) if dtype == x.dtype else x.new_empty(x.shape, dtype=dtype)
    _run(_lib.lib.fhe_rms_norm, x, args, y.data_ptr())
    return y


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, gate, groups, eps, dtype):
        ctx.save_for_backward(x, weight, gate)
        ctx.options = groups, eps, dtype
        return _norm_forward(x, weight, gate, groups, eps, dtype)

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        x, weight, gate = ctx.saved_tensors
        args, held = _pack_norm(x, weight, gate, *ctx.options)
        dy = _flat(dy)
        dx, dw, dgate = _like(x), _like(weight), None if gate is None else _like(gate)
        grads = _NORM_GRADS.pack(*_row(dy), dx.data_ptr(), _ptr(dgate), dw.data_ptr())
        space, size = _workspace(_lib.lib.fhe_rms_norm_workspace, x, args)
        _run(_lib.lib.fhe_rms_norm_backward, x, args, grads, space.data_ptr(), size)
        return dx, dw, dgate, None, None, None


def rms_norm(x, weight, *, gate=None, groups: int = 1, eps: float = 1e-5, dtype=None):
    """v / sqrt(mean(v^2) + eps) * weight with v = x silu(gate), or x without a gate.

    x [.., channels] and gate alike, weight [channels] float32.  The mean is over each of `groups`
    equal parts of the channels, of at most 32768 each.  The result is of x's type or, with dtype,
    bfloat16.  Differentiable in x, weight and gate.  Squares are summed in 32 bits: a row whose
    squares come to 2^128 or more gives zeros, squares below 2^-126 lose bits, and a row with a value that is
    not finite has NaN in it; the gradient's products with v are summed in 32 bits too."""
    _leading("x", x)
    channels = x.shape[-1]
    if groups < 1 or channels % groups or channels // groups > MAX_ROW or groups > 65535:
        raise ValueError(f"{channels} channels do not divide into {groups} groups of at most {MAX_ROW}")
    _gpu("weight", weight, _F32, (channels,), x)
    if gate is not None:
        _gpu("gate", gate, (x.dtype,), x.shape, x)
    dtype, eps = _narrower("dtype", dtype, x), _eps(eps)
    if _wants_grad(x, weight, gate):
        return _Norm.apply(x, weight, gate, groups, eps, dtype)
    return _norm_forward(x, weight, gate, groups, eps, dtype)


class AddNorm(NamedTuple):
    """normed [.., channels] of the update's type and hidden, the sum, of the first hidden's."""
    normed: torch.Tensor
    hidden: torch.Tensor


def _pack_add_norm(hidden, update, weight, scale, eps, dtypes, shape) -> tuple:
    """(the packed arguments, the tensors that they point to)."""
    weight = weight.contiguous()
    if hidden is not None:
        hidden, update = _flat(hidden), _flat(update)
    if scale is not None:
        scale = scale.contiguous()
    channels = shape[-1]
    args = _ADD_NORM.pack(_DTYPES[dtypes[0]], _DTYPES[dtypes[1]], eps, shape.numel() // channels, channels,
                          *_row(hidden), *_row(update), _ptr(scale), weight.data_ptr())
    return args, (hidden, update, weight, scale)


def _add_norm_forward(hidden, update, weight, scale, eps):
    args, held = _pack_add_norm(hidden, update, weight, scale, eps, (hidden.dtype, update.dtype), hidden.shape)
    total, y = _like(hidden), _like(update)
    _run(_lib.lib.fhe_add_norm, hidden, args, total.data_ptr(), y.data_ptr())
    return y, total


class _AddNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, update, weight, scale, eps):
        y, total = _add_norm_forward(hidden, update, weight, scale, eps)
        ctx.options = eps, (hidden.dtype, update.dtype), hidden.shape
        ctx.whole = hidden.dtype == torch.float32 and scale is None  # the sum says all that the gradient needs
        if ctx.whole:
            ctx.save_for_backward(weight, total)
        else:
            ctx.save_for_backward(weight, hidden, update, scale)
        ctx.set_materialize_grads(False)
        return y, total

    @staticmethod
    @_first_order
    def backward(ctx, dy, dtotal):
        eps, dtypes, shape = ctx.options
        total = hidden = update = scale = None
        if ctx.whole:
            weight, total = ctx.saved_tensors
        else:
            weight, hidden, update, scale = ctx.saved_tensors
        args, held = _pack_add_norm(hidden, update, weight, scale, eps, dtypes, shape)
        dy, dtotal = None if dy is None else _flat(dy), None if dtotal is None else _flat(dtotal)
        dh, du = weight.new_empty(shape, dtype=dtypes[0]), weight.new_empty(shape, dtype=dtypes[1])
        dw, ds = _like(weight), None if scale is None else _like(scale)
        grads = _ADD_NORM_GRADS.pack(*_row(dy), *_row(dtotal), _ptr(total), dh.data_ptr(), du.data_ptr(), _ptr(ds),
                                     dw.data_ptr())
        space, size = _workspace(_lib.lib.fhe_add_norm_workspace, weight, args)
        _run(_lib.lib.fhe_add_norm_backward, weight, args, grads, space.data_ptr(), size)
        return dh, du, dw, ds, None


def add_norm(hidden, update, weight, *, scale=None, eps: float = 1e-5) -> AddNorm:
    """The residual and the next norm: h = hidden + scale update, and h / sqrt(mean(h^2) + eps) * weight.

    hidden [.., channels] (at most 32768) and update alike, of hidden's type or bfloat16; scale (default
    ones) and weight [channels] float32.  The norm is of the unrounded sum, and has the update's type.
    Differentiable in all four; the backward pass needs the sum (32-bit hidden without a scale) or hidden
    and update as they were.  Large and not finite values as in rms_norm."""
    _leading("hidden", hidden)
    channels = hidden.shape[-1]
    if channels > MAX_ROW:
        raise ValueError(f"{channels} channels: at most {MAX_ROW}")
    _gpu("update", update, (hidden.dtype, torch.bfloat16), hidden.shape, hidden)
    _gpu("weight", weight, _F32, (channels,), hidden)
    if scale is not None:
        _gpu("scale", scale, _F32, (channels,), hidden)
    eps = _eps(eps)
    if _wants_grad(hidden, update, weight, scale):
        return AddNorm(*_AddNorm.apply(hidden, update, weight, scale, eps))
    return AddNorm(*_add_norm_forward(hidden, update, weight, scale, eps))


# ----------------------------------------------------------------- 8-bit products
class Int8Rows(NamedTuple):
    """values [.., channels] int8 and scale [..] float32: a row is its values times its scale."""
    values: torch.Tensor
    scale: torch.Tensor


def quantize_rows(x) -> Int8Rows:
    """Each row of x [.., channels] (at most 32768) as 8-bit integers: scale = max|x| / 127, values = the
    integer nearest to x / scale, even among equals, both quotients rounded to float32 first.

    A row of zeros has scale 0; one with a value that is not finite has scale NaN and values 0."""
    _leading("x", x)
    channels = x.shape[-1]
    if channels > MAX_ROW:
        raise ValueError(f"{channels} channels: at most {MAX_ROW}")
    if _wants_grad(x):
        raise ValueError("quantize_rows has no gradient: call it under torch.no_grad()")
    rows = _flat(x)
    values = x.new_empty(x.shape, dtype=torch.int8)
    scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
    args = _QUANTIZE.pack(_DTYPES[x.dtype], rows.shape[0], channels, *_row(rows))
    _run(_lib.lib.fhe_quantize_rows, x, args, values.data_ptr(), scale.data_ptr())
    return Int8Rows(values, scale)


def int8_linear(x, weight, weight_scale, bias=None):
    """x [.., inputs] times weight [outputs, inputs] int8 and weight_scale [outputs] float32 (as
    quantize_rows gives them), plus bias [outputs] float32: [.., outputs] of x's type.

    x's rows are rounded as quantize_rows does (at most 32768 inputs; a result of fewer than 2^34 elements);
    the sums of products are exact, and scaled in 32 bits.  A row with a value that is not finite gives NaN.
    For serving: no gradient."""
    _leading("x", x)
    _axes("weight", weight, 2, "be [outputs, inputs]")
    inputs, outputs = x.shape[-1], weight.shape[0]
    if inputs > MAX_ROW:
        raise ValueError(f"{inputs} inputs: at most {MAX_ROW}")
    if outputs < 1:
        raise ValueError("no outputs")
    _gpu("weight", weight, (torch.int8,), (outputs, inputs), x)
    _gpu("weight_scale", weight_scale, _F32, (outputs,), x)
    if bias is not None:
        _gpu("bias", bias, _F32, (outputs,), x)
        bias = bias.contiguous()
    if _wants_grad(x, weight_scale, bias):
        raise ValueError("int8_linear has no gradient: call it under torch.no_grad()")
    rows, weight, weight_scale = _flat(x), weight.contiguous(), weight_scale.contiguous()
    y = x.new_empty((*x.shape[:-1], outputs))
    args = _INT8.pack(_DTYPES[x.dtype], rows.shape[0], inputs, outputs, *_row(rows), weight.data_ptr(),
                      weight_scale.data_ptr(), _ptr(bias))
    space, size = _workspace(_lib.lib.fhe_int8_linear_workspace, x, args)  # none for the fewest rows
    _run(_lib.lib.fhe_int8_linear, x, args, y.data_ptr(), _ptr(space), size)
    return y


# ----------------------------------------------------------------- embeddings
def _pack_embed(weight: Optional[torch.Tensor], ids, scale: float, dtype, vocab: int, channels: int) -> bytes:
    return _EMBED.pack(_DTYPES[dtype], scale, ids.numel(), vocab, channels, *_row(weight), ids.data_ptr())


def _embed_forward(weight, ids, scale: float):
    rows, ids = _rows(weight), ids.contiguous()
    y = weight.new_empty((*ids.shape, weight.shape[1]))
    _run(_lib.lib.fhe_embed, weight, _pack_embed(rows, ids, scale, weight.dtype, *weight.shape), y.data_ptr())
    return y


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale):
        ctx.save_for_backward(ids)
        ctx.options = scale, weight.dtype, *weight.shape
        return _embed_forward(weight, ids, scale)

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        (ids,) = ctx.saved_tensors
        ids, dy = ids.contiguous(), _flat(dy)
        args = _pack_embed(None, ids, *ctx.options)
        dw = dy.new_empty(ctx.options[2:])
        space, size = _workspace(_lib.lib.fhe_embed_workspace, dy, args)  # none for few tokens
        _run(_lib.lib.fhe_embed_backward, dy, args, _ROWS.pack(*_row(dy)), dw.data_ptr(), _ptr(space), size)
        return dw, None, None


def embed(weight, ids, *, scale: float = 1.0):
    """scale * weight[ids]: weight [vocab, channels], ids [..] int64 -> [.., channels] of weight's type.

    An id below 0 is padding: zeros, and no gradient from it; one of vocab or more gives NaN.
    Differentiable in weight: the gradient is dense, each row the sum in 32 bits of its tokens', in an
    order that the ids fix."""
    _first("weight", weight, 2)
    if min(weight.shape) < 1:
        raise ValueError("weight must have a vocabulary and channels")
    if not isinstance(ids, torch.Tensor):
        raise ValueError("ids must be a tensor")
    _gpu("ids", ids, (torch.int64,), ids.shape, weight)
    if not abs(scale) < 3.4e38:
        raise ValueError("scale must be finite")
    if _wants_grad(weight):
        return _Embed.apply(weight, ids, scale)
    return _embed_forward(weight, ids, scale)


# ----------------------------------------------------------------- beam search
class BeamChoice(NamedTuple):
    """score float32, parent and token int32, each [requests, width], best first."""
    score: torch.Tensor
    parent: torch.Tensor
    token: torch.Tensor


def beam_select(logits, scores, width: Optional[int] = None, *, finished=None, end: Optional[int] = None) -> BeamChoice:
    """The `width` (default: as many as there are beams; at most 32) best continuations of each request.

    logits [requests, beams, vocab] (at most 32 beams) and scores [requests, beams] float32: a candidate is
    a beam and a token, its score the beam's plus the token's log probability; the lower beam, then the
    lower token first among equals.  Scores are 64-bit numbers, of two beams good to about 2^-40, until they
    are rounded for the result.  A beam of score -inf has none.  finished [requests, beams] bool: such
    a beam has the one candidate `end`, at its own score.  Where fewer candidates are allowed, others
    follow with score -inf.  A NaN or +inf among a live beam's logits, or for a score, makes the beam's
    candidates NaN, which come first.  No gradient (token_logprobs at the chosen tokens has one).  Where the
    width is not the number of beams, reorder_states has to be told how many beams there were."""
    _first("logits", logits, 3)
    requests, beams, vocab = logits.shape
    if min(requests, beams, vocab) < 1 or beams > MAX_TOP or requests > 65535:
        raise ValueError(f"logits must be [requests, beams, vocab] with 1 to 65535 requests and 1 to {MAX_TOP} beams")
    _gpu("scores", scores, _F32, (requests, beams), logits)
    width = beams if width is None else width
    if not 1 <= width <= min(MAX_TOP, beams * vocab):
        raise ValueError(f"width must be 1 to {min(MAX_TOP, beams * vocab)}")
    if finished is not None:
        _gpu("finished", finished, (torch.bool,), (requests, beams), logits)
        if end is None or not 0 <= end < vocab:
            raise ValueError("end must be a token where beams may be finished")
        finished = finished.contiguous()
    if _wants_grad(logits, scores):
        raise ValueError("beam_select has no gradient: call it under torch.no_grad()")
    rows, scores = _flat(logits), scores.contiguous()
    if rows.shape[0] > 1 and rows.stride(0) < vocab:  # one row for all
        rows = rows.contiguous()
    args = _BEAM.pack(_DTYPES[logits.dtype], requests, beams, width, vocab, rows.stride(0), -1 if end is None else end,
                      rows.data_ptr(), scores.data_ptr(), _ptr(finished))
    score = scores.new_empty((requests, width))
    parent, token = (scores.new_empty((requests, width), dtype=torch.int32) for _ in range(2))
    out = _BEAM_OUT.pack(score.data_ptr(), parent.data_ptr(), token.data_ptr())
    space, size = _workspace(_lib.lib.fhe_beam_select_workspace, logits, args)
    _run(_lib.lib.fhe_beam_select, logits, args, out, space.data_ptr(), size)
    return BeamChoice(score, parent, token)


def reorder_states(states, parent, *, slots=None, beams: Optional[int] = None) -> None:
    """The states follow their beams, in place: row slots[r, j] takes what row slots[r, parent[r, j]] held.

    states: a tensor [cache, ..] or a sequence of them with as many rows, of any type, contiguous, none of
    which shares memory with another.  parent [requests, width] int32 as beam_select gives it; `beams` (at
    most 32) is how many beams each request had before, to be given where that is not the width.  slots
    [requests, the larger of width and beams] (default: rows in order, as many for each request), no row
    twice: the first `width` of them are written, the others stay as they were.  A parent that is no beam
    leaves the row as it is; a slot outside of the cache is padding.  A backward pass that needs a state as
    it was before raises."""
    states = (states,) if isinstance(states, torch.Tensor) else tuple(states)
    if not states:
        raise ValueError("no states")
    _axes("parent", parent, 2, "be [requests, beams]")
    requests, width = parent.shape
    beams = width if beams is None else beams
    first = states[0]
    # there may be two for each layer: checked in as few Python steps as can be
    if not all(map(isinstance, states, repeat(torch.Tensor))) or not first.is_cuda:
        raise ValueError("states must be tensors on the GPU")
    if len(set(map(_device_of, states))) > 1:
        raise ValueError("states must be tensors on one GPU")
    if not (1 <= requests <= 65535 and 1 <= width <= MAX_TOP and 1 <= beams <= MAX_TOP):
        raise ValueError(f"parent must be [requests, beams] with 1 to 65535 requests and 1 to {MAX_TOP} beams")
    _gpu("parent", parent, (torch.int32,), (requests, width), first)
    if width < beams:  # rows without a parent stay
        parent = torch.nn.functional.pad(parent, (0, beams - width), value=-1)
    elif width > beams:  # and those whose parent is none of the beams that were
        parent = parent.masked_fill(parent >= beams, -1)
        beams = width
    try:
        rows = set(map(_size_of, states, repeat(0)))
    except IndexError:  # a tensor without axes
        rows = ()
    if len(rows) != 1 or (cache := rows.pop()) < 1:
        raise ValueError("states must have the same number of rows, one or more")
    if slots is not None:
        _gpu("slots", slots, (torch.int32,), (requests, beams), first)
        slots = slots.contiguous()
    elif requests * beams > cache:
        raise ValueError(f"{requests * beams} beams and {cache} rows of the states")
    if not all(map(_is_contiguous, states)):
        raise ValueError("states must be contiguous: they are updated in place")
    if getattr(_forward_ad, "_current_level", 0) >= 0 or any(map(_requires_grad, states)):
        if _wants_grad(*states):
            raise ValueError("reorder_states has no gradient: call it under torch.no_grad()")
    packed = struct.pack(f"={2 * len(states)}q",
                         *chain.from_iterable((t.data_ptr(), t.nbytes // cache) for t in states))
    parent = parent.contiguous()
    _run(_lib.lib.fhe_reorder_states, first, packed, len(states), requests, beams, cache, parent.data_ptr(),
         _ptr(slots))
    _changed(states)
