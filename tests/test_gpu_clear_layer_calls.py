"""The operators round the mixer as programs call them: captured and replayed, on other streams, in inference mode,
with forward-mode tangents, their results changed in place."""
import pytest

torch = pytest.importorskip("torch")
fwd = torch.autograd.forward_ad

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def serving_state(rows, vocab=700, width=96, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    from fhemamba_amd import clear

    return {"table": r(vocab, width), "ids": torch.randint(0, vocab, (rows, 4), generator=gen, device="cuda"),
            "norm": r(width), "update": r(rows, 4, width), "gate": r(rows, 4, width),
            "head": clear.quantize_rows(r(vocab, width)), "scores": -r(rows, 4).abs(), "cache": r(rows * 4 + 2, 33),
            "slots": torch.randperm(rows * 4, generator=gen, device="cuda").reshape(rows, 4).to(torch.int32)}


@torch.no_grad()
def serve(s):
    """A step of a search: every operator without a gradient."""
    from fhemamba_amd import clear

    x = clear.embed(s["table"], s["ids"], scale=2.0)
    normed, hidden = clear.add_norm(x, s["update"], s["norm"])
    gated = clear.rms_norm(normed, s["norm"], gate=s["gate"], groups=3)
    logits = clear.int8_linear(gated, s["head"].values, s["head"].scale)
    choice = clear.beam_select(logits, s["scores"], 4)
    clear.reorder_states([s["cache"]], choice.parent, slots=s["slots"])
    return (hidden, logits, *choice, *clear.quantize_rows(gated))


def train_state(seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    return {"table": r(500, 72), "ids": torch.randint(-1, 60, (300,), generator=gen, device="cuda"), "norm": r(72),
            "update": r(300, 72), "gate": r(300, 72), "scale": r(72), "d": r(300, 72)}


def train(s):
    """Every operator with a gradient, forwards and backwards."""
    from fhemamba_amd import clear

    leaves = [s[k].detach().requires_grad_(True) for k in ("table", "norm", "update", "gate", "scale")]
    table, norm, update, gate, scale = leaves
    normed, hidden = clear.add_norm(clear.embed(table, s["ids"]), update, norm, scale=scale)
    out = clear.rms_norm(normed, norm, gate=gate, groups=2) + clear.add_norm(hidden, update, norm).normed
    return (out.detach(), *torch.autograd.grad(out, leaves, s["d"]))


def refill(s, other):
    for k, v in s.items():
        for a, b in zip(v, other[k]) if isinstance(v, tuple) else ((v, other[k]),):
            a.copy_(b)


@pytest.mark.parametrize("rows", [1, 2, 40, 700])
def test_captured_searches(rows):
    """Two graphs of two states, replayed in turn with eager work between: each replay is the eager result."""
    states = [serving_state(rows, seed=k) for k in (1, 2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in states:
            serve(s)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for s in states:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(serve(s))
    for turn in range(3):
        fresh = [serving_state(rows, seed=10 + 2 * turn + k) for k in range(2)]
        for s, f in zip(states, fresh):
            refill(s, f)
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        wants = [serve(f) for f in fresh]
        for s, f, out, want in zip(states, fresh, outs, wants):
            assert torch.equal(s["cache"], f["cache"])
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_captured_training():
    s = train_state(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train(s)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = train(s)
    for turn in range(1, 4):
        fresh = train_state(turn)
        refill(s, fresh)
        graph.replay()
        want = train(fresh)
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_other_streams_and_inference_mode():
    want, grads = serve(serving_state(50, seed=3)), train(train_state(4))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got, again = serve(serving_state(50, seed=3)), train(train_state(4))
    side.synchronize()
    with torch.inference_mode():
        third = serve(serving_state(50, seed=3))
    for a, b, c in zip(want, got, third):
        assert torch.equal(a, b) and torch.equal(a, c)
    for a, b in zip(grads, again):
        assert torch.equal(a, b)


def test_calls_behind_each_other_share_nothing():
    """Workspaces that the caller's allocator hands out again at once: 30 calls without a wait."""
    states = [serving_state(60, seed=k) for k in range(30)]
    torch.cuda.synchronize()
    got = [serve(s) for s in states]
    torch.cuda.synchronize()
    for k in (0, 13, 29):
        want = serve(serving_state(60, seed=k))
        torch.cuda.synchronize()
        for a, b in zip(got[k], want):
            assert torch.equal(a, b)


def test_results_are_tensors_of_their_own():
    from fhemamba_amd import clear

    s = serving_state(5)
    with torch.no_grad():
        results = [*clear.add_norm(s["update"], s["gate"], s["norm"]), *clear.quantize_rows(s["update"]),
                   *clear.beam_select(torch.randn(5, 4, 9, device="cuda"), s["scores"])]
    assert len({t.untyped_storage().data_ptr() for t in results}) == len(results)
    leaf = s["update"].clone().requires_grad_(True)
    normed, hidden = clear.add_norm(leaf, s["gate"], s["norm"], scale=s["norm"])
    (want,) = torch.autograd.grad((normed * s["gate"]).sum() + hidden.sum(), leaf)
    normed, hidden = clear.add_norm(leaf, s["gate"], s["norm"], scale=s["norm"])
    (got,) = torch.autograd.grad(normed.mul_(s["gate"]).sum() + hidden.mul_(1.0).sum(), leaf)
    assert torch.equal(got, want)


def test_tangents_are_refused():
    from fhemamba_amd import clear

    z = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
    ids, parent = torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    table = torch.zeros(4, 8, dtype=torch.int8, device="cuda")
    with fwd.dual_level(), torch.no_grad():
        for call in (lambda: clear.rms_norm(z(2, 8), dual(z(8))),
                     lambda: clear.rms_norm(z(2, 8), z(8), gate=dual(z(2, 8))),
                     lambda: clear.add_norm(z(2, 8), dual(z(2, 8)), z(8)), lambda: clear.quantize_rows(dual(z(2, 8))),
                     lambda: clear.int8_linear(dual(z(2, 8)), table, z(4)), lambda: clear.embed(dual(z(4, 8)), ids),
                     lambda: clear.beam_select(dual(z(1, 2, 8)), z(1, 2)),
                     lambda: clear.reorder_states([z(2, 8), dual(z(2, 8))], parent)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()


def test_gradients_where_only_some_are_wanted():
    from fhemamba_amd import clear

    s = train_state(5)
    full = train(s)
    for k in range(5):
        leaves = [s[n].detach().clone() for n in ("table", "norm", "update", "gate", "scale")]
        leaves[k].requires_grad_(True)
        table, norm, update, gate, scale = leaves
        normed, hidden = clear.add_norm(clear.embed(table, s["ids"]), update, norm, scale=scale)
        out = clear.rms_norm(normed, norm, gate=gate, groups=2) + clear.add_norm(hidden, update, norm).normed
        assert torch.equal(out.detach(), full[0])
        (g,) = torch.autograd.grad(out, leaves[k], s["d"])
        assert torch.equal(g, full[1 + k])
