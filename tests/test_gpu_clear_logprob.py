"""Log probabilities, entropies and likeliest tokens, and their gradient, against 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

import clear_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def make(seed, rows, vocab, dtype, masked, scale=4.0):
    gen = torch.Generator().manual_seed(seed)
    logits = (scale * torch.randn(rows, vocab, generator=gen)).to(dtype)
    targets = torch.randint(0, vocab, (rows,), generator=gen)
    if masked:
        logits[torch.rand(rows, vocab, generator=gen) < 0.5] = -math.inf
        logits[torch.arange(rows), targets] = 1.0
    targets[torch.rand(rows, generator=gen) < 0.2] = -1
    return logits, targets


def check_top(got, logits, top):
    """Values and indices by a stable order: the lower index first among equals."""
    want = logits.double() + 0.0
    order = torch.sort(want, dim=-1, descending=True, stable=True)
    assert torch.equal(got.top_index.cpu().long(), order.indices[:, :top])
    logp = torch.log_softmax(want, -1)
    torch.testing.assert_close(got.top_logprob.cpu().double(), logp.gather(1, order.indices[:, :top]),
                               rtol=R.F32, atol=R.F32)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 63), (2, 4096), (4, 4097), (3, 8191), (2, 50280),
                                        (1, 131075)])
def test_rows(rows, vocab, masked, dtype):
    from fhemamba_amd import clear

    logits, targets = make(rows * vocab, rows, vocab, dtype, masked)
    top = min(vocab, 20)
    print(f"[logprob] {rows} x {vocab} {dtype} {masked}", flush=True)
    leaf = logits.cuda().requires_grad_(True)
    got = clear.token_logprobs(leaf, targets.cuda(), top=top)
    gen = torch.Generator().manual_seed(1)
    da, db = (torch.randn(rows, generator=gen) for _ in range(2))
    (grad,) = torch.autograd.grad([got.logprob, got.entropy], leaf, [da.cuda(), db.cuda()])
    ref = logits.double().requires_grad_(True)
    lp, ent = R.logprob(ref, targets)
    (want,) = torch.autograd.grad((lp * da.double()).sum() + (ent * db.double()).sum(), ref)
    # entropy and log probability are differences of numbers around 10: absolute errors of 2^-16
    torch.testing.assert_close(got.logprob.detach().cpu().double(), lp.detach(), rtol=R.F32, atol=R.F32)
    torch.testing.assert_close(got.entropy.detach().cpu().double(), ent.detach(), rtol=R.F32, atol=R.F32)
    check_top(got, logits, top)
    # one allowed token: the gradient is the difference of equal numbers
    assert float((grad.cpu().double() - want).norm()) <= R.bound(grad) * float(want.norm()) + R.F32 * float(da.norm())


def test_ties_and_signed_zeros():
    from fhemamba_amd import clear

    logits = torch.zeros(4, 9000)
    logits[1, ::3] = -0.0
    logits[2, 8000:] = 1.0
    logits[3] = torch.arange(9000) // 1000
    for dtype in (F32, BF):
        got = clear.token_logprobs(logits.to(dtype).cuda(), torch.zeros(4, dtype=torch.int64, device="cuda"), top=32)
        check_top(got, logits, 32)


def test_sorted_rows_fill_the_candidates():
    """Rows in order put as many of the best into one thread's share as can be."""
    from fhemamba_amd import clear

    up = torch.arange(20000, dtype=F32)
    logits = torch.stack([up, -up, up % 4096, -(up % 4096), (up * 2654435761 % 4294967296) / 4e5])
    got = clear.token_logprobs(logits.cuda(), torch.zeros(5, dtype=torch.int64, device="cuda"), top=32)
    check_top(got, logits, 32)


def test_rows_without_tokens_and_bad_targets():
    from fhemamba_amd import clear

    logits = torch.randn(6, 5000)
    logits[0] = -math.inf
    logits[1] = -math.inf
    logits[2, 1:] = -math.inf
    logits[4, 7] = math.nan
    logits[5, 7] = math.inf
    targets = torch.tensor([3, -1, 0, 5000, 1, 2])
    leaf = logits.cuda().requires_grad_(True)
    got = clear.token_logprobs(leaf, targets.cuda(), top=2)
    lp, ent = got.logprob.tolist(), got.entropy.tolist()
    assert lp[0] == -math.inf and lp[1] == 0.0 and lp[2] == 0.0 and all(math.isnan(v) for v in lp[3:])
    assert ent[:3] == [0.0, 0.0, 0.0] and math.isfinite(ent[3]) and all(math.isnan(v) for v in ent[4:])
    assert got.top_index[0].tolist() == [0, 1] and got.top_logprob[0].tolist() == [-math.inf] * 2
    assert got.top_logprob[2].tolist() == [0.0, -math.inf]
    one = torch.ones(6, device="cuda")
    (g,) = torch.autograd.grad([got.logprob, got.entropy], leaf, [one, one])
    assert bool((g[:3] == 0).all()) and bool(torch.isfinite(g[3]).all()) and not bool(torch.isfinite(g[4:]).any())


def test_extreme_logits():
    from fhemamba_amd import clear

    logits = torch.tensor([[3e38, -3e38, 0.0], [-3e38, -3e38, -3.4028235e38], [88.0, 87.0, -100.0]])
    targets = torch.tensor([1, 0, 2])
    got = clear.token_logprobs(logits.cuda(), targets.cuda())
    want = torch.log_softmax(logits.double(), -1).gather(1, targets[:, None])[:, 0]
    assert got.logprob[0].item() == -math.inf or abs(got.logprob[0].item()) > 3e38
    torch.testing.assert_close(got.logprob[1:].cpu().double(), want[1:], rtol=R.F32, atol=R.F32)
    assert got.top_index is None and bool(torch.isfinite(got.entropy).all())


@pytest.mark.parametrize("dtype", [F32, BF])
def test_strides_and_axes(dtype):
    """Rows inside wider storage at odd places, leading axes, one row for all, gradients of either output."""
    from fhemamba_amd import clear

    wide = (3 * torch.randn(4, 6, 1500, generator=torch.Generator().manual_seed(2))).to(dtype).cuda()
    part = wide[..., 3:1250]
    targets = torch.randint(0, 1247, (4, 6), device="cuda")
    got, want = clear.token_logprobs(part, targets, top=3), clear.token_logprobs(part.contiguous(), targets, top=3)
    assert got.logprob.shape == (4, 6) and got.top_index.shape == (4, 6, 3)
    assert all(torch.allclose(a.float(), b.float(), rtol=1e-6, atol=1e-6) for a, b in zip(got, want))
    row = part[0, 0].expand(5, 1247)
    five = clear.token_logprobs(row, torch.arange(5, device="cuda"))
    torch.testing.assert_close(five.logprob.cpu().double(), torch.log_softmax(row[0].cpu().double(), -1)[:5],
                               rtol=R.F32, atol=R.F32)
    leaf = part.detach().clone().requires_grad_(True)
    for pick in ("logprob", "entropy"):
        (g,) = torch.autograd.grad(getattr(clear.token_logprobs(leaf, targets), pick).sum(), leaf)
        ref = leaf.detach().cpu().double().reshape(24, -1).requires_grad_(True)
        lp, ent = R.logprob(ref, targets.cpu().reshape(-1))
        (w,) = torch.autograd.grad((lp if pick == "logprob" else ent).sum(), ref)
        assert R.rel(g.reshape(24, -1), w) <= R.bound(g)


def test_gradient_against_differences():
    """Central differences of losses around 1 in 64 bits from outputs good to 2^-22: 1e-4 over 2e-2."""
    from fhemamba_amd import clear

    logits, targets = make(5, 6, 300, F32, False, scale=1.0)
    gen = torch.Generator().manual_seed(1)
    da, db, way = torch.randn(6, generator=gen), torch.randn(6, generator=gen), torch.randn(6, 300, generator=gen)
    way = way / way.norm()
    leaf = logits.cuda().requires_grad_(True)
    got = clear.token_logprobs(leaf, targets.cuda())
    (g,) = torch.autograd.grad([got.logprob, got.entropy], leaf, [da.cuda(), db.cuda()])

    def loss(v):
        r = clear.token_logprobs(v.cuda(), targets.cuda())
        return float((r.logprob.cpu().double() * da.double()).sum() + (r.entropy.cpu().double() * db.double()).sum())

    diff = (loss(logits + 1e-2 * way) - loss(logits - 1e-2 * way)) / 2e-2
    assert abs(diff - float((g.cpu().double() * way.double()).sum())) <= 1e-3


def test_past_32_bit_offsets():
    from fhemamba_amd import clear

    rows, vocab = 43000, 50280  # 2.16e9 logits
    logits = torch.zeros(rows, vocab, dtype=BF, device="cuda")
    logits[-1] = torch.randn(vocab, generator=torch.Generator().manual_seed(3)).to(BF).cuda()
    targets = torch.full((rows,), 17, device="cuda")
    got = clear.token_logprobs(logits, targets, top=2)
    want = torch.log_softmax(logits[-1].cpu().double(), -1)
    assert abs(float(got.logprob[-1]) - float(want[17])) <= R.F32 * 16
    assert int(got.top_index[-1, 0]) == int(want.argmax())
    assert abs(float(got.logprob[0]) + math.log(vocab)) <= R.F32 * 16


def test_no_rows_and_graph():
    from fhemamba_amd import clear

    nobody = torch.zeros(0, dtype=torch.int64, device="cuda")
    none = clear.token_logprobs(torch.zeros(0, 9, device="cuda"), nobody, top=2)
    assert none.logprob.shape == (0,) and none.top_index.shape == (0, 2)
    logits = torch.randn(3, 6000, device="cuda")
    targets = torch.tensor([1, -1, 5], device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        clear.token_logprobs(logits, targets, top=4)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = clear.token_logprobs(logits, targets, top=4)
    for _ in range(4):
        logits.copy_(torch.randn_like(logits))
        graph.replay()
        want = clear.token_logprobs(logits, targets, top=4)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    from fhemamba_amd import clear

    logits, targets = torch.zeros(3, 40, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for match, a, kw in [("float32 or bfloat16", (logits.half(), targets), {}),
                         ("on the GPU", (logits.cpu(), targets), {}),
                         ("targets has shape", (logits, targets[:2]), {}),
                         ("targets must be of type", (logits, targets.int()), {}),
                         ("top", (logits, targets), {"top": 33}),
                         ("top", (logits[:, :4].contiguous(), targets), {"top": 5}),
                         ("top", (logits, targets), {"top": -1})]:
        with pytest.raises(ValueError, match=match):
            clear.token_logprobs(*a, **kw)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("order", ["random", "rising", "falling", "equal", "few"])
def test_most_of_a_long_row(order, dtype):
    """32 of 300001, in every order of the sets of entries that they are picked from, at an odd row stride."""
    from fhemamba_amd import clear

    vocab, rows = 300001, 2
    logits, _ = make(5, rows, vocab, dtype, False)
    if order in ("rising", "falling"):
        logits = torch.sort(logits, dim=1, descending=order == "falling").values
    elif order == "equal":
        logits[:] = 0.5
    elif order == "few":  # fewer allowed tokens than places: the rest are masked ones, lowest first
        keep = logits[:, 77777::100000].clone()
        logits[:] = -math.inf
        logits[:, 77777::100000] = keep
    wide = torch.full((rows, vocab + 3), 9.0, dtype=dtype)
    wide[:, 2:vocab + 2] = logits
    print(f"[logprob] long {order} {dtype}", flush=True)
    got = clear.token_logprobs(wide.cuda()[:, 2:vocab + 2], torch.zeros(rows, dtype=torch.int64, device="cuda"), top=32)
    check_top(got, logits, 32)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_tokens_of_a_row_of_nan_are_in_it(dtype):
    """What they are is not defined, but an index never leaves its row."""
    from fhemamba_amd import clear

    logits, targets = make(6, 3, 5000, dtype, False)
    logits[0, 7] = math.nan
    logits[1] = math.nan
    logits[2] = torch.full((5000,), -1, dtype=torch.int16 if dtype == BF else torch.int32).view(dtype)  # NaN of all ones
    got = clear.token_logprobs(logits.cuda(), targets.cuda(), top=32)
    assert bool(((got.top_index >= 0) & (got.top_index < 5000)).all())
    assert bool(torch.isnan(got.top_logprob).all())
