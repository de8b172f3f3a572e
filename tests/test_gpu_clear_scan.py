"""The selective scan and its single-token form against the recurrence in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

import clear_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def normal(gen, *shape, dtype=F32):
    return torch.randn(shape, generator=gen).to(dtype)


def make(seed, tokens, H, P, N, G, dtype, seqs=None, gate=1.0):
    """Inputs on the CPU; decays around exp(-gate / 4), some tokens write nothing."""
    gen = torch.Generator().manual_seed(seed)
    d = {"x": normal(gen, tokens, H, P, dtype=dtype), "B": normal(gen, tokens, G, N, dtype=dtype),
         "C": normal(gen, tokens, G, N, dtype=dtype),
         "write": torch.rand(tokens, H, generator=gen) * (torch.rand(tokens, H, generator=gen) > 0.1),
         "log_decay": -gate * 0.5 * torch.rand(tokens, H, generator=gen), "D": normal(gen, H)}
    if seqs:
        d["initial"] = normal(gen, seqs, H, P, N)
    return d


NAMES = ("x", "write", "log_decay", "B", "C", "D")


def run(d, lengths, packed, grads=None, **kw):
    """The operator on the GPU (packed, or [sequences, tokens]): y, states and, with grads =
    (dy, dstate), the gradients."""
    from fhemamba_amd import clear

    S = len(lengths)
    leaves = {}
    for k in NAMES + ("initial",):
        if d.get(k) is None:
            leaves[k] = None
            continue
        t = d[k].cuda()
        if not packed and k not in ("D", "initial"):
            t = t.reshape(S, -1, *t.shape[1:])
        leaves[k] = t.requires_grad_(grads is not None)
    cu = None
    if packed:
        cu = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    y, h = clear.ssm_scan(*(leaves[k] for k in NAMES), initial_state=leaves["initial"], cu_seqlens=cu,
                          return_state=True, **kw)
    if grads is None:
        return y.reshape(d["x"].shape), h
    dy, dh = grads
    ins = {k: v for k, v in leaves.items() if v is not None}
    outs, gs = [y], [dy.cuda().reshape(y.shape)]
    if dh is not None:
        outs.append(h)
        gs.append(dh.cuda())
    got = torch.autograd.grad(outs, list(ins.values()), gs)
    return y.detach().reshape(d["x"].shape), h.detach(), {k: g.reshape(d[k].shape) for k, g in zip(ins, got)}


def reference(d, lengths, grads=None):
    leaves = {k: None if d.get(k) is None else d[k].double().requires_grad_(grads is not None)
              for k in NAMES + ("initial",)}
    y, h = R.scan(*(leaves[k] for k in NAMES), leaves["initial"], R.spans(lengths))
    if grads is None:
        return y, h
    dy, dh = grads
    loss = (y * dy.double()).sum() + (0.0 if dh is None else (h * dh.double()).sum())
    ins = {k: v for k, v in leaves.items() if v is not None}
    got = torch.autograd.grad(loss, list(ins.values()), allow_unused=True)
    return y, h, {k: torch.zeros_like(v) if g is None else g for (k, v), g in zip(ins.items(), got)}


SHAPES = [  # heads, head_dim, states, groups
    (4, 32, 32, 1), (2, 64, 128, 1), (3, 8, 16, 3), (4, 33, 33, 2), (1, 1, 1, 1), (6, 80, 40, 2), (5, 16, 100, 1),
    (2, 50, 65, 1),
]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("lengths", [[1], [15], [64], [65, 65], [200], [1, 0, 63, 130, 0]])
@pytest.mark.parametrize("shape", SHAPES)
def test_scan_and_gradients(shape, lengths, dtype):
    H, P, N, G = shape
    packed = len(set(lengths)) > 1
    total, S = sum(lengths), len(lengths)
    d = make(total * 7 + H * P + N, total, H, P, N, G, dtype, seqs=S)
    gen = torch.Generator().manual_seed(1)
    grads = normal(gen, total, H, P, dtype=dtype), normal(gen, S, H, P, N)
    print(f"[scan] {shape} {lengths} {dtype}", flush=True)
    y, h, got = run(d, lengths, packed, grads)
    y0, h0, want = reference(d, lengths, grads)
    assert R.rel(y, y0) <= R.bound(y) and R.rel(h, h0) <= R.F32
    for k in got:
        gates = R.GATES if dtype == BF and k in ("write", "log_decay") else R.bound(got[k])
        assert got[k].dtype == d[k].dtype
        assert R.rel(got[k], want[k]) <= gates, k


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("lengths,packed", [([1500], False), ([700, 1, 0, 900, 64], True)])
def test_long_sequences_split_into_segments(lengths, packed, dtype):
    """Lengths that are cut over the GPU, slow decays that reach across the cuts, no initial state and
    no gradient of the last state."""
    d = make(3, sum(lengths), 2, 64, 128, 1, dtype, gate=0.02)
    gen = torch.Generator().manual_seed(2)
    grads = normal(gen, sum(lengths), 2, 64, dtype=dtype), None
    y, h, got = run(d, lengths, packed, grads)
    y0, h0, want = reference(d, lengths, grads)
    assert R.rel(y, y0) <= R.bound(y) and R.rel(h, h0) <= R.F32
    for k in got:
        gates = R.GATES if dtype == BF and k in ("write", "log_decay") else R.bound(got[k])
        assert R.rel(got[k], want[k]) <= gates, k


@pytest.mark.parametrize("dtype", [F32, BF])
def test_many_sequences_stay_whole(dtype):
    """So many that none is cut: the last states and the adjoint come from the sweeps themselves."""
    H, P, N, S, T = 3, 64, 64, 150, 70
    d = make(4, S * T, H, P, N, 1, dtype, seqs=S)
    gen = torch.Generator().manual_seed(2)
    grads = normal(gen, S * T, H, P, dtype=dtype), normal(gen, S, H, P, N)
    y, h, got = run(d, [T] * S, False, grads)
    y0, h0, want = reference(d, [T] * S, grads)
    assert R.rel(y, y0) <= R.bound(y) and R.rel(h, h0) <= R.F32
    for k in got:
        gates = R.GATES if dtype == BF and k in ("write", "log_decay") else R.bound(got[k])
        assert R.rel(got[k], want[k]) <= gates, k


@pytest.mark.parametrize("dtype", [F32, BF])
def test_forgetting_decays(dtype):
    """exp(-inf), exp(-300) and exp(0): resets inside of a chunk and a tile leave nothing behind."""
    d = make(5, 150, 2, 32, 40, 1, dtype, seqs=1)
    d["log_decay"][::7] = -math.inf
    d["log_decay"][3::11] = -300.0
    d["log_decay"][5::6] = 0.0
    grads = normal(torch.Generator().manual_seed(2), 150, 2, 32, dtype=dtype), None
    y, h, got = run(d, [150], False, grads)
    y0, h0, want = reference(d, [150], grads)
    assert R.rel(y, y0) <= R.bound(y) and R.rel(h, h0) <= R.F32
    for k in ("x", "write", "B", "C", "D"):
        gates = R.GATES if dtype == BF and k == "write" else R.bound(got[k])
        assert R.rel(got[k], want[k]) <= gates, k
    assert bool(torch.isfinite(got["log_decay"]).all())
    assert R.rel(got["log_decay"], want["log_decay"].nan_to_num(0.0)) <= (R.GATES if dtype == BF else R.F32)


def test_gradient_against_differences():
    """The gradient along random directions against central differences of the operator itself.  The
    losses (about 1e2) are summed in 64 bits from outputs good to 2^-22, so differences over 2e-2 are
    good to about 1e2 2^-22 / 2e-2 = 1e-3, and the step's own error is of its square."""
    d = make(6, 100, 2, 16, 24, 1, F32, seqs=2)
    gen = torch.Generator().manual_seed(3)
    dy, dh = normal(gen, 100, 2, 16), normal(gen, 2, 2, 16, 24)
    lengths = [37, 63]
    _, _, got = run(d, lengths, True, (dy, dh))

    def loss(v):
        y, h = run(v, lengths, True)
        return float((y.cpu().double() * dy.double()).sum() + (h.cpu().double() * dh.double()).sum())

    for k in got:
        way = normal(gen, *d[k].shape)
        way = way / way.norm()
        up, down = ({**d, k: d[k] + s * 1e-2 * way} for s in (1, -1))
        diff = (loss(up) - loss(down)) / 2e-2
        mine = float((got[k].cpu().double() * way.double()).sum())
        size = float(got[k].norm()) / math.sqrt(got[k].numel())
        assert abs(diff - mine) <= 1e-2 * max(1.0, size) + 5e-3 * abs(mine), k


@pytest.mark.parametrize("dtype", [F32, BF])
def test_strided_inputs(dtype):
    """Slices at odd places of a wider tensor, heads before tokens, B shared by broadcast, gates as a
    transposed view: the same values as from contiguous copies."""
    from fhemamba_amd import clear

    gen = torch.Generator().manual_seed(7)
    S, T, H, P, N = 2, 90, 3, 24, 20
    wide = normal(gen, S, T, 3 + H * P + 2 * N, dtype=dtype).cuda()
    x = wide[..., 3: 3 + H * P].unflatten(-1, (H, P))
    C = wide[..., 3 + H * P + N:].unflatten(-1, (1, N))
    B = normal(gen, 1, T, 1, N, dtype=dtype).cuda().expand(S, T, 1, N)
    write = torch.rand(S, H, T, generator=gen).cuda().transpose(1, 2)
    g = -torch.rand(H, S, T, generator=gen).cuda().permute(1, 2, 0)
    turned = normal(gen, S, H, T, P, dtype=dtype).cuda().transpose(1, 2)
    last = normal(gen, S, T, P, H, dtype=dtype).cuda().transpose(2, 3)  # copied: its last axis is strided
    for v in (x, turned, last):
        got = clear.ssm_scan(v, write, g, B, C, return_state=True)
        want = clear.ssm_scan(v.contiguous(), write.contiguous(), g.contiguous(), B.contiguous(), C.contiguous(),
                              return_state=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # an expanded gradient
    x = x.detach().requires_grad_(True)
    (a,) = torch.autograd.grad(clear.ssm_scan(x, write, g, B, C).sum(), x)
    ones = torch.ones(S, T, H, P, dtype=dtype, device="cuda")
    (b,) = torch.autograd.grad(clear.ssm_scan(x, write, g, B, C), x, ones)
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_tokens_outside_of_every_sequence(dtype):
    """NaN before, between the ends and behind the sequences stays there; its places give zeros."""
    from fhemamba_amd import clear

    d = make(8, 100, 2, 32, 32, 1, dtype)
    for k in ("x", "B", "C", "write", "log_decay"):
        d[k][:5] = math.nan
        d[k][83:] = math.nan
    leaves = [d[k].cuda().requires_grad_(True) for k in NAMES]
    cu = torch.tensor([5, 40, 40, 83], dtype=torch.int32, device="cuda")
    y, h = clear.ssm_scan(*leaves, cu_seqlens=cu, return_state=True)
    dy = normal(torch.Generator().manual_seed(1), 100, 2, 32, dtype=dtype)
    grads = torch.autograd.grad(y, leaves, dy.cuda())
    y0, h0 = R.scan(*(d[k].double() for k in NAMES), None, [(5, 40), (40, 40), (40, 83)])
    assert R.rel(y, y0) <= R.bound(y) and R.rel(h, h0) <= R.F32
    for g in [y, *grads[:-1]]:
        assert bool((g[:5] == 0).all()) and bool((g[83:] == 0).all()) and bool(torch.isfinite(g).all())


def test_no_tokens():
    from fhemamba_amd import clear

    h0 = torch.randn(2, 3, 8, 16, device="cuda", requires_grad=True)
    z = torch.zeros
    for packed in (False, True):
        lead = (0,) if packed else (2, 0)
        cu = z(3, dtype=torch.int32, device="cuda") if packed else None
        x = z(*lead, 3, 8, device="cuda")
        b, w = z(*lead, 1, 16, device="cuda"), z(*lead, 3, device="cuda")
        D = torch.ones(3, device="cuda", requires_grad=True)
        y, h = clear.ssm_scan(x, w, w, b, b, D, initial_state=h0, cu_seqlens=cu, return_state=True)
        assert y.shape == x.shape and torch.equal(h, h0)
        dh, dD = torch.autograd.grad(h, [h0, D], torch.ones_like(h))
        assert bool((dh == 1).all()) and bool((dD == 0).all())


def test_equal_inputs_give_equal_bits_on_any_stream():
    d = make(9, 1200, 2, 64, 128, 1, BF, seqs=1)
    grads = normal(torch.Generator().manual_seed(1), 1200, 2, 64, dtype=BF), None
    first = run(d, [1200], False, grads)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        second = run(d, [1200], False, grads)
    side.synchronize()
    assert torch.equal(first[0], second[0]) and torch.equal(first[1], second[1])
    assert all(torch.equal(first[2][k], second[2][k]) for k in first[2])


# ----------------------------------------------------------------- single token
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("requests", [1, 3, 40])
@pytest.mark.parametrize("shape", SHAPES)
def test_step(shape, requests, dtype):
    from fhemamba_amd import clear

    H, P, N, G = shape
    d = make(requests + H * P, requests, H, P, N, G, dtype, seqs=requests + 5)
    gen = torch.Generator().manual_seed(1)
    slots = torch.randperm(requests + 5, generator=gen)[:requests].to(torch.int32)
    if requests > 2:
        slots[1], slots[2] = -1, requests + 5  # padding
    state = d["initial"].cuda()
    y = clear.ssm_step(state, *(d[k].cuda() for k in NAMES), slots=slots.cuda())
    want = d["initial"].double()
    y0 = torch.zeros(requests, H, P, dtype=torch.float64)
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < requests + 5:
            one = {k: d[k][i:i + 1].double() if k != "D" else d[k].double() for k in NAMES}
            got, h = R.scan(*(one[k] for k in NAMES), d["initial"][s:s + 1].double(), [(0, 1)])
            y0[i], want[s] = got[0], h[0]
    assert R.rel(y, y0) <= R.bound(y) and R.rel(state, want) <= R.F32
    left = [s for s in range(requests + 5) if s not in slots.tolist()]
    assert torch.equal(state[left].cpu(), d["initial"][left])


def test_step_continues_the_scan():
    """A prompt in one call and its last token as a step, without slots and with strided inputs."""
    from fhemamba_amd import clear

    d = make(11, 2 * 33, 2, 64, 128, 1, F32)
    v = {k: d[k].cuda().reshape(2, 33, *d[k].shape[1:]) if k != "D" else d[k].cuda() for k in NAMES}
    y, h = clear.ssm_scan(*(v[k] for k in NAMES), return_state=True)
    y1, state = clear.ssm_scan(*(v[k][:, :32] if k != "D" else v[k] for k in NAMES), return_state=True)
    last = clear.ssm_step(state, *(v[k][:, 32] if k != "D" else v[k] for k in NAMES))
    assert torch.equal(y1, y[:, :32]) or R.rel(y1, y[:, :32].cpu().double()) <= R.F32
    assert R.rel(last, y[:, 32].cpu().double()) <= R.F32 and R.rel(state, h.cpu().double()) <= R.F32


def test_step_past_32_bit_offsets():
    from fhemamba_amd import clear

    H, P, N = 24, 64, 128
    cache = 2 ** 31 // (H * P * N) + 3
    state = torch.zeros(cache, H, P, N, device="cuda")
    d = make(12, 2, H, P, N, 1, BF)
    slots = torch.tensor([cache - 1, 0], dtype=torch.int32, device="cuda")
    y = clear.ssm_step(state, *(d[k].cuda() for k in NAMES), slots=slots)
    y0, _ = R.scan(*(d[k].double() for k in NAMES), None, [(0, 1), (1, 2)])
    assert R.rel(y, y0) <= R.BF16
    assert float(state[cache - 1].abs().sum()) > 0 and float(state[1:cache - 1].abs().max()) == 0


def test_step_and_scan_in_a_graph():
    """Replays after the first, with eager work between them, give what eager calls give."""
    from fhemamba_amd import clear

    d = make(13, 70, 2, 64, 128, 1, BF)
    v = [d[k].cuda() for k in NAMES]
    one = [t[0:1] if i < 5 else t for i, t in enumerate(v)]
    cu = torch.tensor([0, 30, 70], dtype=torch.int32, device="cuda")
    state = torch.zeros(1, 2, 64, 128, device="cuda")

    def work():
        return clear.ssm_step(state, *one), *clear.ssm_scan(*v, cu_seqlens=cu, return_state=True)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        work()
    side.synchronize()
    state.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    mirror = torch.zeros_like(state)
    for i in range(4):
        v[0].mul_(-0.5 if i % 2 else -2.0)
        graph.replay()
        want = clear.ssm_step(mirror, *one), *clear.ssm_scan(*v, cu_seqlens=cu, return_state=True)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(state, mirror)


def test_refusals():
    from fhemamba_amd import clear

    d = {k: v.cuda() for k, v in make(14, 10, 4, 8, 16, 2, F32).items()}
    args = [d[k] for k in NAMES]
    cu = torch.tensor([0, 10], dtype=torch.int32, device="cuda")

    def refused(match, i=None, new=None, **kw):
        a = list(args)
        if i is not None:
            a[i] = new
        with pytest.raises(ValueError, match=match):
            clear.ssm_scan(*a, **{"cu_seqlens": cu, **kw})

    refused("axes", cu_seqlens=None)
    refused("float32 or bfloat16", 0, d["x"].half())
    refused("on the GPU", 0, d["x"].cpu())
    refused("write has shape", 1, d["write"][:5])
    refused("write must be of type", 1, d["write"].double())
    refused("B must be of type", 3, d["B"].bfloat16())
    refused("groups", 0, d["x"][:, :3])
    refused("C has shape", 4, d["C"][..., :8])
    refused("D has shape", 5, d["D"][:2])
    refused("initial_state has shape", initial_state=torch.zeros(2, 4, 8, 16, device="cuda"))
    refused("cu_seqlens must be of type", cu_seqlens=cu.long())
    refused("cu_seqlens", cu_seqlens=cu[:1])
    refused("at most 128", 3, torch.zeros(10, 2, 129, device="cuda"))
    state = torch.zeros(10, 4, 8, 16, device="cuda")
    for match, s, slots in [("contiguous", state.transpose(0, 1).contiguous().transpose(0, 1), None),
                            ("state must be of type", state.bfloat16(), None), ("rows of the state", state[:9], None),
                            ("slots must be of type", state, torch.zeros(10, dtype=torch.int64, device="cuda"))]:
        with pytest.raises(ValueError, match=match):
            clear.ssm_step(s, *args, slots=slots)
    with pytest.raises(ValueError, match="no gradient"):
        clear.ssm_step(state, d["x"].clone().requires_grad_(True), *args[1:])
