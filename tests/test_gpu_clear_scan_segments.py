"""The scan where its segments are longer than a chunk and where long sequences stay whole, as large batches have
them, against the recurrences in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

import clear_batched as B  # noqa: E402
import clear_reference as R  # noqa: E402
import test_gpu_clear_scan as T  # noqa: E402

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


# sequences, packed, (heads, head_dim, states, groups), least and most tokens of a segment (0: whole)
LONG = [1, 0, 2666, 1333, 1333, 2670]
SHORT = [1300, 0, 1, 1257, 443]
PLANS = {
    "chunks": ([700] * 2, False, (3, 32, 32, 1), 64, 64),
    "two_segments": ([1024] * 16, False, (32, 64, 32, 1), 257, 960),
    "packed": (LONG, True, (36, 64, 32, 1), 257, 512),
    "packed_odd": (LONG, True, (64, 10, 7, 2), 257, 512),
    "one_item_a_gate_group": (SHORT, True, (48, 64, 32, 1), 192, 192),
    "two_items_a_gate_group": (SHORT, True, (64, 32, 32, 1), 128, 128),
    # a sequence or two in each item's length, as prompts of a serving batch
    "many_short": ([(37 * i) % 101 for i in range(240)], True, (8, 32, 32, 1), 64, 128),
    "whole": ([2048] * 32, False, (64, 8, 8, 1), 0, 0),
    "packed_whole": ([1300], True, (4096, 4, 4, 1), 0, 0),
    "whole_odd": ([777] * 60, False, (60, 10, 7, 3), 0, 0),
}


def plan_of(name, dtype):
    lengths, packed, shape, least, most = PLANS[name]
    found = B.segment_lengths(lengths, packed, shape, dtype)
    assert (not found) if not most else found and least <= min(found) and max(found) <= most, found
    return lengths, packed, shape


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("name", list(PLANS))
def test_values_and_gradients(name, dtype):
    """Slow decays that reach across chunks and segments, initial states, gradients of the last ones."""
    lengths, packed, (H, P, N, G) = plan_of(name, dtype)
    total, S = sum(lengths), len(lengths)
    print(f"[scan] {name} {dtype} {B.segment_lengths(lengths, packed, (H, P, N, G), dtype)[:1]}", flush=True)
    d = T.make(total, total, H, P, N, G, dtype, seqs=S, gate=0.02)
    gen = torch.Generator().manual_seed(1)
    grads = T.normal(gen, total, H, P, dtype=dtype), T.normal(gen, S, H, P, N)
    y, h, got = T.run(d, lengths, packed, grads)
    y0, h0, want = B.scan(d, lengths, grads)
    assert B.rel(y, y0) <= R.bound(y) and B.rel(h, h0) <= R.F32
    for k in got:
        gates = R.GATES if dtype == BF and k in ("write", "log_decay") else R.bound(got[k])
        assert B.rel(got[k], want[k]) <= gates, k


@pytest.mark.parametrize("name", ["two_segments", "whole"])
def test_gate_gradients_keep_to_their_size(name):
    """Gradients that come in a thousand times larger at the last 256 tokens: what that takes from the gates'
    gradients of the tokens before is in their own size, not in that of the last ones.  The bound is that of 32-bit
    sums of up to 2^10 products."""
    lengths, packed, (H, P, N, G) = plan_of(name, F32)
    total, S, n = sum(lengths), len(lengths), lengths[0]
    d = T.make(5, total, H, P, N, G, F32, seqs=S)
    gen = torch.Generator().manual_seed(1)
    dy = T.normal(gen, total, H, P).reshape(S, n, H, P)
    dy[:, -256:] *= 1e3
    grads = dy.reshape(total, H, P), None
    _, _, got = T.run(d, lengths, packed, grads)
    _, _, want = B.scan(d, lengths, grads)
    early = n - 320  # decays of exp(-1/4) a token leave little of the large ones there
    for k in ("write", "log_decay"):
        a, b = (v[k].reshape(S, n, H)[:, :early].contiguous() for v in (got, want))
        assert B.rel(a, b) <= R.F32, k


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("name", ["chunks", "two_segments", "whole"])
def test_how_far_a_nan_reaches(name, dtype):
    """A NaN of x, or of the gradient of y, reaches what does not depend on it for at most the 64 tokens around it."""
    lengths, packed, (H, P, N, G) = plan_of(name, dtype)
    total, S, n = sum(lengths), len(lengths), lengths[0]
    for late in (True, False):
        at = n - 170 if late else 170
        d = T.make(6, total, H, P, N, G, dtype)
        dy = T.normal(torch.Generator().manual_seed(1), total, H, P, dtype=dtype)
        (d["x"] if late else dy).reshape(S, n, H, P)[1, at, 2, 3] = math.nan
        y, _, got = T.run(d, lengths, packed, (dy, None))
        for k, v in [("y", y), ("x", got["x"]), ("write", got["write"]), ("log_decay", got["log_decay"])]:
            bad = ~torch.isfinite(v.reshape(S, n, H, -1)).all(-1)
            # x at a token: y from there on, the gates' gradients; dy at one: gradients up to there
            free = bad[1, : at - 64] if late else bad[1, at + 64:]
            assert not bool(free.any()), (k, late)
            bad[1, :, 2] = False
            assert not bool(bad.any()), (k, late)
        assert bool(torch.isnan(got["log_decay"]).any())


@pytest.mark.parametrize("dtype", [F32, BF])
def test_long_stretches_outside_of_every_sequence(dtype):
    """700 tokens before the first sequence and 900 behind the last, all NaN: zeros, and the sequences as without."""
    from fhemamba_amd import clear

    lengths, (H, P, N, G), before, behind = [2900, 0, 1, 3502], (36, 64, 32, 1), 700, 900
    inside = sum(lengths)
    total = before + inside + behind
    found = B.segment_lengths([before, *lengths, behind], True, (H, P, N, G), dtype)
    assert found and min(found) > 256  # segments of several windows
    d = T.make(9, inside, H, P, N, G, dtype, seqs=4, gate=0.02)
    gen = torch.Generator().manual_seed(1)
    grads = T.normal(gen, inside, H, P, dtype=dtype), T.normal(gen, 4, H, P, N)
    leaves = {}
    for k in T.NAMES:
        t = d[k]
        if k != "D":
            t = torch.full((total, *t.shape[1:]), math.nan, dtype=t.dtype)
            t[before:before + inside] = d[k]
        leaves[k] = t.cuda().requires_grad_(True)
    leaves["initial"] = d["initial"].cuda().requires_grad_(True)
    cu = before + torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32)
    y, h = clear.ssm_scan(*(leaves[k] for k in T.NAMES), initial_state=leaves["initial"], cu_seqlens=cu.cuda(),
                          return_state=True)
    dy = torch.full((total, H, P), math.nan, dtype=dtype)
    dy[before:before + inside] = grads[0]
    got = dict(zip(leaves, torch.autograd.grad([y, h], list(leaves.values()), [dy.cuda(), grads[1].cuda()])))
    y0, h0, want = B.scan(d, lengths, grads)
    assert B.rel(y[before:before + inside], y0) <= R.bound(y) and B.rel(h, h0) <= R.F32
    assert bool((y[:before] == 0).all()) and bool((y[before + inside:] == 0).all())
    for k in got:
        gates = R.GATES if dtype == BF and k in ("write", "log_decay") else R.bound(got[k])
        own = k in ("D", "initial")
        assert B.rel(got[k] if own else got[k][before:before + inside], want[k]) <= gates, k
        assert own or bool((got[k][:before] == 0).all()) and bool((got[k][before + inside:] == 0).all()), k
