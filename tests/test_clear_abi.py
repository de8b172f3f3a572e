"""Refusals of the operators' C entry points, which come before any GPU call, and the packed
structures' layouts.  No GPU is needed."""
import ctypes

import pytest

pytest.importorskip("torch")

from fhemamba_amd import _lib, clear  # noqa: E402


def scan(**kw):
    v = dict(dtype=0, seqs=1, heads=2, head_dim=8, states=16, groups=1, tokens=10, offsets=0, data=4096,
             strides=(0, 16, 8), d=0, initial=0, gate=4096)
    v.update(kw)
    t = (v["data"], *v["strides"])
    g = (v["gate"], *v["strides"])
    head = (v[k] for k in ("dtype", "seqs", "heads", "head_dim", "states", "groups", "tokens", "offsets"))
    return clear._SCAN.pack(*head, *t, *t, *t, *g, *g, v["d"], v["initial"])


def test_structures_have_the_c_sizes():
    strided = 32
    assert clear._SCAN.size == 24 + 8 + 8 + 5 * strided + 16
    assert clear._SCAN_GRADS.size == strided + 64
    assert clear._STEP.size == 32 + 8 + 5 * strided + 16
    assert clear._CONV.size == 16 + 16 + strided + 24 + 8
    assert clear._CONV_GRADS.size == strided + 40
    assert clear._CONV_STEP.size == 24 + 8 + strided + 24 + 8
    assert clear._LOGPROB.size == 48 and clear._LOGPROB_OUT.size == 48


@pytest.mark.parametrize("kw,match", [
    ({"dtype": 2}, "dtype"), ({"seqs": 0}, "seqs"), ({"heads": 3, "groups": 2}, "groups"), ({"groups": 0}, "groups"),
    ({"head_dim": 0}, "head_dim"), ({"states": 129}, "states"), ({"tokens": -1}, "tokens"),
    ({"tokens": 2 ** 31}, "tokens"),
    ({"data": 0}, "null"), ({"data": 4097, "dtype": 1}, "aligned"), ({"strides": (0, -1, 8)}, "negative"),
    ({"d": 2}, "aligned"), ({"initial": 3}, "aligned"), ({"gate": 0}, "null"),
])
def test_scan_arguments(kw, match):
    size = ctypes.c_size_t()
    with pytest.raises(ValueError, match=match):
        _lib.call("fhe_ssm_scan_workspace", scan(**kw), 0, ctypes.byref(size))


def test_scan_workspace_is_checked():
    size = ctypes.c_size_t()
    args = scan(tokens=100000)
    _lib.call("fhe_ssm_scan_workspace", args, 0, ctypes.byref(size))
    assert size.value > 0
    with pytest.raises(ValueError, match="too small"):
        _lib.call("fhe_ssm_scan", args, 4096, 0, 4096, size.value - 1, 0)
    with pytest.raises(ValueError, match="256-byte"):
        _lib.call("fhe_ssm_scan", args, 4096, 0, 4097, size.value, 0)
    with pytest.raises(ValueError, match="null workspace"):
        _lib.call("fhe_ssm_scan", args, 4096, 0, 0, size.value, 0)
    with pytest.raises(ValueError, match="null output"):
        _lib.call("fhe_ssm_scan", args, 0, 0, 4096, size.value, 0)
    with pytest.raises(ValueError, match="null argument"):
        _lib.call("fhe_ssm_scan", None, 4096, 0, 4096, size.value, 0)


@pytest.mark.parametrize("kw,match", [
    ({"requests": 0}, "requests"), ({"cache": 0}, "cache"), ({"requests": 9}, "more requests"),
    ({"groups": 3}, "groups"), ({"states": 200}, "states"), ({"state": 0}, "null state"), ({"data": 0}, "null input"),
])
def test_step_arguments(kw, match):
    v = dict(dtype=0, requests=2, cache=8, heads=2, head_dim=8, states=16, groups=1, data=4096, state=4096)
    v.update(kw)
    t = (v["data"], 0, 16, 8)
    head = (v[k] for k in ("dtype", "requests", "cache", "heads", "head_dim", "states", "groups"))
    args = clear._STEP.pack(*head, 0, *t, *t, *t, *t, *t, 0, v["state"])
    with pytest.raises(ValueError, match=match):
        _lib.call("fhe_ssm_step", args, 4096, 0)


@pytest.mark.parametrize("kw,match", [({"taps": 1}, "taps"), ({"taps": 9}, "taps"), ({"channels": 0}, "channels"),
                                      ({"weight": 0}, "weight"), ({"dtype": 5}, "dtype"), ({"data": 0}, "null input")])
def test_convolution_arguments(kw, match):
    v = dict(dtype=1, seqs=1, channels=8, taps=4, tokens=10, data=4096, weight=4096)
    v.update(kw)
    head = (v[k] for k in ("dtype", "seqs", "channels", "taps", "tokens"))
    args = clear._CONV.pack(*head, 0, v["data"], 0, 8, 0, v["weight"], 0, 0, 1)
    with pytest.raises(ValueError, match=match):
        _lib.call("fhe_causal_conv", args, 4096, 0, 0)


@pytest.mark.parametrize("kw,match", [({"rows": 0}, "rows"), ({"vocab": 0}, "vocab"), ({"row_stride": 5}, "row_stride"),
                                      ({"top": 33}, "top"), ({"top": 11}, "top"), ({"logits": 0}, "null"),
                                      ({"logits": 4097}, "aligned"), ({"targets": 4}, "aligned"),
                                      ({"rows": 2 ** 22, "vocab": 2 ** 24, "row_stride": 2 ** 24}, "too many")])
def test_logprob_arguments(kw, match):
    v = dict(dtype=1, top=0, rows=2, vocab=10, row_stride=10, logits=4096, targets=4096)
    v.update(kw)
    args = clear._LOGPROB.pack(*(v[k] for k in ("dtype", "top", "rows", "vocab", "row_stride", "logits", "targets")))
    size = ctypes.c_size_t()
    with pytest.raises(ValueError, match=match):
        _lib.call("fhe_token_logprobs_workspace", args, ctypes.byref(size))


def test_tensors_off_the_gpu_are_refused():
    import torch

    z = torch.zeros
    with pytest.raises(ValueError, match="on the GPU"):
        clear.ssm_scan(z(2, 5, 2, 8), z(2, 5, 2), z(2, 5, 2), z(2, 5, 1, 4), z(2, 5, 1, 4))
    with pytest.raises(ValueError, match="on the GPU"):
        clear.ssm_step(z(2, 2, 8, 4), z(2, 2, 8), z(2, 2), z(2, 2), z(2, 1, 4), z(2, 1, 4))
    with pytest.raises(ValueError, match="on the GPU"):
        clear.causal_conv(z(2, 5, 8), z(8, 4))
    with pytest.raises(ValueError, match="on the GPU"):
        clear.causal_conv_step(z(2, 3, 8), z(2, 8), z(8, 4))
    with pytest.raises(ValueError, match="on the GPU"):
        clear.token_logprobs(z(2, 8), z(2, dtype=torch.int64))
