"""Refusals of the C entry points round the mixer, which come before any GPU call, and the packed
structures' layouts.  No GPU is needed."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")

from fhemamba_amd import _lib, clear  # noqa: E402


def size_of(name, args):
    size = ctypes.c_size_t()
    _lib.call(name, args, ctypes.byref(size))
    return size.value


def test_structures_have_the_c_sizes():
    assert clear._ROWS.size == 16
    assert clear._NORM.size == 16 + 16 + 32 + 8 and clear._NORM_GRADS.size == 16 + 24
    assert clear._ADD_NORM.size == 16 + 16 + 32 + 16 and clear._ADD_NORM_GRADS.size == 32 + 40
    assert clear._QUANTIZE.size == 8 + 16 + 16 and clear._INT8.size == 8 + 24 + 16 + 24
    assert clear._EMBED.size == 8 + 24 + 16 + 8
    assert clear._BEAM.size == 16 + 24 + 24 and clear._BEAM_OUT.size == 24


def norm(**kw):
    v = dict(dtype=0, out=0, groups=1, eps=1e-5, rows=3, channels=8, x=4096, x_row=8, gate=0, gate_row=0, weight=4096)
    v.update(kw)
    return clear._NORM.pack(*v.values())


@pytest.mark.parametrize("kw,match", [
    ({"dtype": 2}, "dtype"), ({"out": 3}, "dtype"), ({"dtype": 1, "out": 0}, "out_dtype"), ({"groups": 0}, "groups"),
    ({"groups": 3}, "groups"), ({"eps": -1.0}, "eps"), ({"eps": math.nan}, "eps"), ({"eps": math.inf}, "eps"),
    ({"rows": -1}, "rows"), ({"rows": 2 ** 31}, "rows"), ({"channels": 0}, "channels"),
    ({"channels": 32769}, "32768"), ({"channels": 2 ** 20 + 2, "groups": 2 ** 10 + 2}, "channels"), ({"x": 0}, "null"),
    ({"x": 4097, "dtype": 1, "out": 1}, "aligned"), ({"x_row": -8}, "negative"), ({"gate": 4098}, "aligned"),
    ({"weight": 0}, "null weight"), ({"weight": 2}, "aligned"),
])
def test_norm_arguments(kw, match):
    with pytest.raises(ValueError, match=match):
        size_of("fhe_rms_norm_workspace", norm(**kw))
    with pytest.raises(ValueError, match=match):
        _lib.call("fhe_rms_norm", norm(**kw), 4096, 0)


def test_norm_outputs_and_workspace():
    args = norm(rows=5000, channels=70, x_row=70)
    size = size_of("fhe_rms_norm_workspace", args)
    assert size >= 70 * 4
    grads = clear._NORM_GRADS.pack(4096, 70, 4096, 0, 4096)
    for y, match in ((0, "null output"), (4098, "aligned")):
        with pytest.raises(ValueError, match=match):
            _lib.call("fhe_rms_norm", args, y, 0)
    for space, given, match in ((4096, size - 1, "too small"), (4097, size, "256-byte"), (0, size, "null workspace")):
        with pytest.raises(ValueError, match=match):
            _lib.call("fhe_rms_norm_backward", args, grads, space, given, 0)
    for bad in ((0, 70, 4096, 0, 4096), (4096, 70, 0, 0, 4096), (4096, 70, 4096, 0, 0), (4096, -1, 4096, 0, 4096)):
        with pytest.raises(ValueError):
            _lib.call("fhe_rms_norm_backward", args, clear._NORM_GRADS.pack(*bad), 4096, size, 0)
    gated = norm(gate=4096, gate_row=8)
    with pytest.raises(ValueError, match="null output"):  # a gate without its gradient
        _lib.call("fhe_rms_norm_backward", gated, clear._NORM_GRADS.pack(4096, 8, 4096, 0, 4096), 4096, 1 << 20, 0)
    with pytest.raises(ValueError, match="null argument"):
        _lib.call("fhe_rms_norm", None, 4096, 0)


def add_norm(**kw):
    v = dict(dtype=0, out=1, eps=1e-5, rows=3, channels=8, hidden=4096, hidden_row=8, update=4096, update_row=8, scale=0,
             weight=4096)
    v.update(kw)
    return clear._ADD_NORM.pack(*v.values())


@pytest.mark.parametrize("kw,match", [
    ({"dtype": 1, "out": 0}, "out_dtype"), ({"eps": -1.0}, "eps"), ({"rows": 2 ** 31}, "rows"),
    ({"channels": 32769}, "channels"), ({"hidden": 0}, "null"), ({"update": 0}, "null"), ({"update": 4097}, "aligned"),
    ({"update_row": -1}, "negative"), ({"weight": 0}, "null weight"), ({"scale": 6}, "aligned"),
])
def test_add_norm_arguments(kw, match):
    with pytest.raises(ValueError, match=match):
        _lib.call("fhe_add_norm", add_norm(**kw), 4096, 4096, 0)
    grads = clear._ADD_NORM_GRADS.pack(4096, 8, 4096, 8, 0, 4096, 4096, 0, 4096)
    with pytest.raises(ValueError, match=match):
        _lib.call("fhe_add_norm_backward", add_norm(**kw), grads, 4096, 1 << 20, 0)


def test_add_norm_outputs():
    args = add_norm()
    for out in ((0, 4096), (4096, 0), (4098, 4096), (4096, 4097)):
        with pytest.raises(ValueError):
            _lib.call("fhe_add_norm", args, *out, 0)
    size = size_of("fhe_add_norm_workspace", args)
    assert size_of("fhe_add_norm_workspace", add_norm(scale=4096)) == 2 * size
    ok = [4096, 8, 4096, 8, 0, 4096, 4096, 0, 4096]
    for i, v in ((8, 0), (0, 4097), (1, -1), (2, 4098), (4, 4098), (5, 4098), (6, 4097), (7, 2), (8, 2)):
        bad = list(ok)
        bad[i] = v
        with pytest.raises(ValueError):
            _lib.call("fhe_add_norm_backward", args, clear._ADD_NORM_GRADS.pack(*bad), 4096, size, 0)
    with pytest.raises(ValueError, match="too small"):
        _lib.call("fhe_add_norm_backward", args, clear._ADD_NORM_GRADS.pack(*ok), 4096, size - 1, 0)
    ok[7] = 4096
    with pytest.raises(ValueError, match="a scale that is not there"):
        _lib.call("fhe_add_norm_backward", args, clear._ADD_NORM_GRADS.pack(*ok), 4096, size, 0)


@pytest.mark.parametrize("kw,match", [({"dtype": 7}, "dtype"), ({"rows": -1}, "rows"), ({"channels": 0}, "channels"),
                                      ({"channels": 32769}, "channels"), ({"x": 0}, "null"), ({"x": 4098}, "aligned"),
                                      ({"x_row": -1}, "negative")])
def test_quantize_arguments(kw, match):
    v = dict(dtype=0, rows=2, channels=8, x=4096, x_row=8)
    v.update(kw)
    with pytest.raises(ValueError, match=match):
        _lib.call("fhe_quantize_rows", clear._QUANTIZE.pack(*v.values()), 4096, 4096, 0)


def int8(**kw):
    v = dict(dtype=1, rows=2, inputs=8, outputs=5, x=4096, x_row=8, weight=4096, scale=4096, bias=0)
    v.update(kw)
    return clear._INT8.pack(*v.values())


@pytest.mark.parametrize("kw,match", [
    ({"dtype": 2}, "dtype"), ({"rows": 2 ** 31}, "rows"), ({"inputs": 0}, "inputs"), ({"inputs": 40000}, "inputs"),
    ({"outputs": 0}, "outputs"), ({"outputs": 2 ** 25}, "outputs"), ({"rows": 2 ** 24, "outputs": 2 ** 12}, "too many"),
    ({"x": 0}, "null"), ({"x": 4097}, "aligned"), ({"weight": 0}, "null weight"), ({"scale": 0}, "null weight"),
    ({"scale": 6}, "aligned"), ({"bias": 6}, "aligned"),
])
def test_int8_arguments(kw, match):
    with pytest.raises(ValueError, match=match):
        size_of("fhe_int8_linear_workspace", int8(**kw))


def test_int8_outputs_and_workspace():
    args = int8(rows=200)
    size = size_of("fhe_int8_linear_workspace", args)
    assert size >= 200 * 8 + 800
    for y, space, given, match in ((0, 4096, size, "null output"), (4097, 4096, size, "aligned"),
                                   (4096, 4096, size - 1, "too small"), (4096, 0, size, "null workspace")):
        with pytest.raises(ValueError, match=match):
            _lib.call("fhe_int8_linear", args, y, space, given, 0)
    with pytest.raises(ValueError, match="null output"):
        _lib.call("fhe_quantize_rows", clear._QUANTIZE.pack(0, 2, 8, 4096, 8), 0, 4096, 0)


def embed(**kw):
    v = dict(dtype=0, scale=1.0, tokens=4, vocab=10, channels=8, weight=4096, weight_row=8, ids=4096)
    v.update(kw)
    return clear._EMBED.pack(*v.values())


@pytest.mark.parametrize("kw,match", [
    ({"dtype": 2}, "dtype"), ({"tokens": -1}, "tokens"), ({"tokens": 2 ** 29}, "tokens"), ({"vocab": 0}, "vocab"),
    ({"vocab": 2 ** 25}, "vocab"), ({"channels": 0}, "channels"), ({"channels": 2 ** 21}, "channels"), ({"ids": 0}, "ids"),
    ({"ids": 4}, "aligned"),
])
def test_embed_arguments(kw, match):
    with pytest.raises(ValueError, match=match):
        size_of("fhe_embed_workspace", embed(**kw))
    with pytest.raises(ValueError, match=match):
        _lib.call("fhe_embed", embed(**kw), 4096, 0)


def test_embed_outputs_and_workspace():
    for kw, y, match in (({"weight": 0}, 4096, "null"), ({"weight_row": -1}, 4096, "negative"), ({}, 0, "null output"),
                         ({"dtype": 1}, 4097, "aligned")):
        with pytest.raises(ValueError, match=match):
            _lib.call("fhe_embed", embed(**kw), y, 0)
    args = embed(weight=0, tokens=4000)
    size = size_of("fhe_embed_workspace", args)
    assert size >= 4 * 11 + 8 * 4000 and size_of("fhe_embed_workspace", embed(weight=0)) == 0
    dy, none = clear._ROWS.pack(4096, 8), clear._ROWS.pack(0, 8)
    for d, dw, given, match in ((dy, 0, size, "null"), (None, 4096, size, "null"), (none, 4096, size, "null"),
                                (dy, 4098, size, "aligned"), (dy, 4096, size - 1, "too small")):
        with pytest.raises(ValueError, match=match):
            _lib.call("fhe_embed_backward", args, d, dw, 4096, given, 0)


def beam(**kw):
    v = dict(dtype=0, requests=2, beams=3, width=3, vocab=10, row_stride=10, end=-1, logits=4096, scores=4096, finished=0)
    v.update(kw)
    return clear._BEAM.pack(*v.values())


@pytest.mark.parametrize("kw,match", [
    ({"dtype": 2}, "dtype"), ({"requests": 0}, "requests"), ({"requests": 65536}, "requests"), ({"beams": 0}, "beams"),
    ({"beams": 33}, "beams"), ({"width": 0}, "width"), ({"width": 33}, "width"),
    ({"width": 7, "vocab": 2, "row_stride": 2}, "width"),
    ({"vocab": 0}, "vocab"), ({"row_stride": 9}, "row_stride"), ({"logits": 0}, "null"), ({"scores": 0}, "null"),
    ({"logits": 4098}, "aligned"), ({"scores": 4098}, "aligned"), ({"finished": 4096}, "end"),
    ({"finished": 4096, "end": 10}, "end"),
    ({"requests": 65535, "beams": 32, "vocab": 2 ** 24, "row_stride": 2 ** 24}, "too many"),
])
def test_beam_arguments(kw, match):
    with pytest.raises(ValueError, match=match):
        size_of("fhe_beam_select_workspace", beam(**kw))


def test_beam_outputs_and_workspace():
    size = size_of("fhe_beam_select_workspace", beam())
    for out, given, match in (((0, 4096, 4096), size, "null output"), ((4096, 4098, 4096), size, "aligned"),
                              ((4096, 4096, 4096), size - 1, "too small")):
        with pytest.raises(ValueError, match=match):
            _lib.call("fhe_beam_select", beam(), clear._BEAM_OUT.pack(*out), 4096, given, 0)


@pytest.mark.parametrize("kw,match", [
    ({"count": 0}, "count"), ({"requests": 0}, "requests"), ({"beams": 0}, "beams"), ({"beams": 33}, "beams"),
    ({"cache": 0}, "cache"), ({"cache": 5}, "more beams"), ({"parent": 0}, "null"), ({"parent": 4098}, "aligned"),
    ({"slots": 4098}, "aligned"), ({"data": 0}, "null state"), ({"row_bytes": -1}, "row_bytes"),
    ({"row_bytes": 2 ** 30 + 1}, "row_bytes"),
])
def test_reorder_arguments(kw, match):
    v = dict(data=4096, row_bytes=64, count=1, requests=2, beams=3, cache=6, parent=4096, slots=0)
    v.update(kw)
    states = clear._ROWS.pack(v["data"], v["row_bytes"])
    with pytest.raises(ValueError, match=match):
        _lib.call("fhe_reorder_states", states, *(v[k] for k in ("count", "requests", "beams", "cache", "parent", "slots")), 0)


def test_tensors_off_the_gpu_are_refused():
    z = torch.zeros
    ids = z(3, dtype=torch.int64)
    for call in (lambda: clear.rms_norm(z(2, 8), z(8)), lambda: clear.add_norm(z(2, 8), z(2, 8), z(8)),
                 lambda: clear.quantize_rows(z(2, 8)), lambda: clear.embed(z(4, 8), ids),
                 lambda: clear.int8_linear(z(2, 8), z(3, 8, dtype=torch.int8), z(3)),
                 lambda: clear.beam_select(z(1, 2, 8), z(1, 2)),
                 lambda: clear.reorder_states(z(2, 8), z(1, 2, dtype=torch.int32))):
        with pytest.raises(ValueError, match="on the GPU"):
            call()


@pytest.mark.parametrize("states", [[(4096, 64), (4096, 64)], [(8192, 16), (4096, 64), (4096 + 6 * 64 - 1, 4)],
                                    [(4096, 64), (4096 + 64, 8)]])
def test_states_that_share_memory_are_refused(states):
    """Rows of one that are rows of another would be moved twice, at once."""
    packed = b"".join(clear._ROWS.pack(*s) for s in states)
    with pytest.raises(ValueError, match="share memory"):
        _lib.call("fhe_reorder_states", packed, len(states), 2, 3, 6, 4096, 0, 0)
