"""The causal convolution, its gradients and its single-token form against 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

import clear_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def make(seed, tokens, channels, taps, dtype, seqs):
    gen = torch.Generator().manual_seed(seed)

    def n(*shape, dtype=F32):
        return torch.randn(shape, generator=gen).to(dtype)

    return {"x": n(tokens, channels, dtype=dtype), "weight": n(channels, taps), "bias": n(channels),
            "initial": n(seqs, taps - 1, channels, dtype=dtype), "dy": n(tokens, channels, dtype=dtype),
            "dstate": n(seqs, taps - 1, channels, dtype=dtype)}


LENGTHS = [[1], [2], [16], [17, 17], [33], [100], [1, 0, 3, 50, 2, 0, 31]]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("channels,taps", [(1, 2), (24, 4), (33, 3), (64, 8), (7, 5), (40, 2)])
def test_convolution_and_gradients(channels, taps, lengths, dtype):
    from fhemamba_amd import clear

    S, total = len(lengths), sum(lengths)
    d = make(total + channels * taps, total, channels, taps, dtype, S)
    packed = len(set(lengths)) > 1
    print(f"[conv] {channels} x {taps} {lengths} {dtype}", flush=True)
    names = ("x", "weight", "bias", "initial")
    leaves = {k: d[k].cuda() for k in names}
    shape = d["x"].shape if packed else (S, lengths[0], channels)
    leaves = {k: (v.reshape(shape) if k == "x" else v).requires_grad_(True) for k, v in leaves.items()}
    ends = torch.tensor(lengths).cumsum(0).tolist()
    cu = torch.tensor([0, *ends], dtype=torch.int32, device="cuda") if packed else None
    y, last = clear.causal_conv(leaves["x"], leaves["weight"], leaves["bias"], initial_state=leaves["initial"],
                                cu_seqlens=cu, return_state=True)
    got = torch.autograd.grad([y, last], list(leaves.values()), [d["dy"].cuda().reshape(shape), d["dstate"].cuda()])
    ref = {k: d[k].double().requires_grad_(True) for k in names}
    y0, last0 = R.conv(ref["x"], ref["weight"], ref["bias"], ref["initial"], R.spans(lengths))
    loss = (y0 * d["dy"].double()).sum() + (last0 * d["dstate"].double()).sum()
    want = torch.autograd.grad(loss, list(ref.values()))
    assert R.rel(y.reshape(d["x"].shape), y0) <= R.bound(y)
    assert torch.equal(last.cpu().double(), last0.detach())
    for k, a, b in zip(names, got, want):
        assert a.dtype == d[k].dtype
        assert R.rel(a.reshape(d[k].shape), b) <= R.bound(a), k


@pytest.mark.parametrize("dtype", [F32, BF])
def test_sums_without_activation_bias_or_state(dtype):
    from fhemamba_amd import clear

    d = make(3, 90, 48, 4, dtype, 2)
    wide = torch.zeros(2, 45, 70, dtype=dtype, device="cuda")
    wide[..., 5:53] = d["x"].cuda().reshape(2, 45, 48)
    x = wide[..., 5:53].requires_grad_(True)  # rows that are not 16-byte aligned
    y, last = clear.causal_conv(x, d["weight"].cuda(), silu=False, return_state=True)
    (g,) = torch.autograd.grad(y, x, d["dy"].cuda().reshape(2, 45, 48))
    ref = d["x"].double().requires_grad_(True)
    y0, last0 = R.conv(ref, d["weight"].double(), None, None, [(0, 45), (45, 90)], silu=False)
    (want,) = torch.autograd.grad((y0 * d["dy"].double()).sum(), ref)
    assert R.rel(y.reshape(90, 48), y0) <= R.bound(y) and torch.equal(last.cpu().double(), last0.detach())
    assert R.rel(g.reshape(90, 48), want) <= R.bound(g)


@pytest.mark.parametrize("taps", [2, 3, 4, 7])
def test_a_nan_reaches_its_own_taps_only(taps):
    """Values that are not finite at one token, in another sequence and outside of all of them."""
    from fhemamba_amd import clear

    d = make(4, 80, 16, taps, F32, 2)
    d["x"][:4] = math.nan
    d["x"][70:] = math.inf
    d["x"][20, 3] = math.nan
    cu = torch.tensor([4, 36, 70], dtype=torch.int32, device="cuda")
    x = d["x"].cuda().requires_grad_(True)
    y = clear.causal_conv(x, d["weight"].cuda(), d["bias"].cuda(), cu_seqlens=cu)
    (g,) = torch.autograd.grad(y, x, d["dy"].cuda())
    bad = torch.zeros(80, 16, dtype=torch.bool)
    bad[20:20 + taps, 3] = True
    assert torch.equal(~torch.isfinite(y.cpu()), bad)
    assert bool((y[:4] == 0).all()) and bool((y[70:] == 0).all()) and bool((g[:4] == 0).all())
    assert bool((g[70:] == 0).all())
    near = torch.zeros(80, 16, dtype=torch.bool)
    near[20 - taps + 1: 20 + taps, 3] = True  # inputs that share a sum with it
    assert not bool((~torch.isfinite(g.cpu()) & ~near).any())


def test_gradient_against_differences():
    """Along random directions; the differences are good to about 1e-3 of a loss of 1e2 over 2e-2."""
    from fhemamba_amd import clear

    d = make(5, 60, 24, 4, F32, 2)
    cu = torch.tensor([0, 25, 60], dtype=torch.int32, device="cuda")
    names = ("x", "weight", "bias", "initial")

    def call(v):
        return clear.causal_conv(v["x"], v["weight"], v["bias"], initial_state=v["initial"], cu_seqlens=cu)

    leaves = {k: d[k].cuda().requires_grad_(True) for k in names}
    got = torch.autograd.grad(call(leaves), list(leaves.values()), d["dy"].cuda())
    gen = torch.Generator().manual_seed(1)
    for k, g in zip(names, got):
        way = torch.randn(d[k].shape, generator=gen)
        way = way / way.norm()
        loss = [float((call({**{n: d[n].cuda() for n in names}, k: (d[k] + s * way).cuda()}).cpu().double()
                       * d["dy"].double()).sum()) for s in (1e-2, -1e-2)]
        mine = float((g.cpu().double() * way.double()).sum())
        assert abs((loss[0] - loss[1]) / 2e-2 - mine) <= 1e-2 + 5e-3 * abs(mine), k


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("channels,taps", [(24, 4), (33, 3), (8, 8), (1, 2)])
def test_step(channels, taps, dtype):
    from fhemamba_amd import clear

    R_, cache = 6, 9
    d = make(7, R_, channels, taps, dtype, cache)
    slots = torch.tensor([4, -1, 8, 0, 9, 2], dtype=torch.int32)
    state = d["initial"].cuda()
    y = clear.causal_conv_step(state, d["x"].cuda(), d["weight"].cuda(), d["bias"].cuda(), slots=slots.cuda())
    want, y0 = d["initial"].double(), torch.zeros(R_, channels, dtype=torch.float64)
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < cache:
            got, last = R.conv(d["x"][i:i + 1].double(), d["weight"].double(), d["bias"].double(),
                               d["initial"][s:s + 1].double(), [(0, 1)])
            y0[i], want[s] = got[0], last[0]
    assert R.rel(y, y0) <= R.bound(y) and torch.equal(state.cpu().double(), want)


def test_no_tokens_and_equal_bits():
    from fhemamba_amd import clear

    w = torch.randn(8, 4, device="cuda", requires_grad=True)
    h0 = torch.randn(3, 3, 8, device="cuda", requires_grad=True)
    y, last = clear.causal_conv(torch.zeros(3, 0, 8, device="cuda"), w, initial_state=h0, return_state=True)
    assert y.shape == (3, 0, 8) and torch.equal(last, h0)
    dh, dw = torch.autograd.grad(last, [h0, w], torch.ones_like(last))
    assert bool((dh == 1).all()) and bool((dw == 0).all())
    x = torch.randn(2, 500, 8, device="cuda")
    a, b = (torch.autograd.grad(clear.causal_conv(x, w).square().sum(), w)[0] for _ in range(2))
    assert torch.equal(a, b)


def test_refusals():
    from fhemamba_amd import clear

    x, w = torch.zeros(2, 5, 8, device="cuda"), torch.zeros(8, 4, device="cuda")
    for match, a, kw in [("axes", (x[0], w), {}), ("taps", (x, torch.zeros(8, 9, device="cuda")), {}),
                         ("taps", (x, w[:, :1]), {}), ("weight has shape", (x, w[:4]), {}),
                         ("weight must be of type", (x, w.bfloat16()), {}),
                         ("float32 or bfloat16", (x.double(), w), {}),
                         ("bias has shape", (x, w, w[0]), {}),
                         ("initial_state has shape", (x, w), {"initial_state": torch.zeros(2, 4, 8, device="cuda")}),
                         ("initial_state must be of type", (x, w),
                          {"initial_state": torch.zeros(2, 3, 8, device="cuda", dtype=BF)})]:
        with pytest.raises(ValueError, match=match):
            clear.causal_conv(*a, **kw)
    state = torch.zeros(2, 3, 8, device="cuda")
    for match, a in [("state has shape", (state[:, :2], x[:, 0], w)), ("rows of the state", (state[:1], x[:, 0], w)),
                     ("contiguous", (state.transpose(0, 1).contiguous().transpose(0, 1), x[:, 0], w))]:
        with pytest.raises(ValueError, match=match):
            clear.causal_conv_step(*a)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("shift", [0, 1, 4])
def test_weights_that_begin_anywhere(shift, dtype):
    """Four taps are read as one piece where the weights are aligned to it, and singly where not."""
    from fhemamba_amd import clear

    d = make(9, 50, 48, 4, dtype, 1)
    flat = torch.zeros(48 * 4 + 8, device="cuda")
    weight = flat[shift:shift + 48 * 4].view(48, 4)
    weight.copy_(d["weight"])
    y, last = clear.causal_conv(d["x"].cuda()[None], weight, d["bias"].cuda(), initial_state=d["initial"].cuda(),
                                return_state=True)
    y0, last0 = R.conv(d["x"].double(), d["weight"].double(), d["bias"].double(), d["initial"].double(),
                       R.spans([50]))
    assert R.rel(y[0], y0) <= R.bound(y)
    assert torch.equal(last.cpu().double(), last0)
    state = d["initial"].cuda()
    step = clear.causal_conv_step(state, d["x"].cuda()[:1], weight, d["bias"].cuda())
    assert R.rel(step, y0[:1]) <= R.bound(step)
