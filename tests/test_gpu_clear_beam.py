"""A beam search's choice against a search candidate by candidate in 64 bits, and the states behind it."""
import math

import pytest

torch = pytest.importorskip("torch")

import layer_reference as L  # noqa: E402

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def make(seed, R, B, V, dtype, masked=0.0, step=None):
    gen = torch.Generator().manual_seed(seed)
    logits = 3 * torch.randn(R, B, V, generator=gen)
    if step:
        logits = torch.round(logits / step) * step  # many ties
    logits[torch.rand(R, B, V, generator=gen) < masked] = -math.inf
    return logits.to(dtype), -10 * torch.rand(R, B, generator=gen)


def compare(logits, scores, width, finished=None, end=None):
    from fhemamba_amd import clear

    got = clear.beam_select(logits.cuda(), scores.cuda(), width, finished=None if finished is None else finished.cuda(),
                            end=end)
    score, parent, token = L.beam(logits, scores, width, finished, end)
    assert got.score.shape == got.parent.shape == got.token.shape == (logits.shape[0], width)
    assert torch.equal(got.parent.cpu().long(), parent) and torch.equal(got.token.cpu().long(), token)
    # log sums good to 2^-22, the score rounded to 32 bits
    torch.testing.assert_close(got.score.cpu().double(), score, rtol=2.0 ** -23, atol=2.0 ** -22, equal_nan=True)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("R,B,V,width", [(1, 1, 1, 1), (2, 3, 1, 3), (1, 4, 2, 8), (3, 2, 5, 10), (2, 1, 100, 5),
                                         (1, 4, 4096, 4), (2, 5, 4097, 5), (1, 3, 8193, 32), (2, 32, 700, 32),
                                         (1, 32, 33, 32), (3, 8, 50280, 8), (1, 2, 131075, 32), (40, 2, 300, 4)])
def test_choice(R, B, V, width, dtype):
    print(f"[beam] {R} x {B} x {V} -> {width} {dtype}", flush=True)
    compare(*make(R * V + B, R, B, V, dtype), width)
    compare(*make(R * V + B + 1, R, B, V, dtype, masked=0.5), width)


@pytest.mark.parametrize("V", [7, 4100, 9001])
def test_ties_take_the_lower_beam_then_the_lower_token(V):
    """Equal beams (equal logits and scores, rows at any alignment) and equal tokens within them."""
    for dtype in (F32, BF):
        logits, scores = make(V, 3, 1, V, dtype, step=2.0)
        compare(logits.expand(3, 6, V).contiguous(), scores.expand(3, 6).contiguous(), 20)
    compare(torch.zeros(1, 3, V), torch.zeros(1, 3), 5)


def test_finished_dead_and_masked_beams():
    logits, scores = make(1, 6, 4, 300, F32, masked=0.2)
    finished = torch.zeros(6, 4, dtype=torch.bool)
    scores[0, 1:] = -math.inf                      # the first step: one live beam
    scores[1] = -math.inf                          # none, and one of them is finished
    finished[1, 0] = True
    finished[2, 1] = finished[2, 3] = True
    finished[3] = True                             # all
    logits[4, 0] = -math.inf                       # no token is allowed
    logits[4, 1:, 5:] = -math.inf                  # few are
    scores[5, 1:] = -math.inf
    finished[5, 0] = True                          # one candidate in all
    for width in (1, 4, 20):
        for end in (0, 2, 299):
            compare(logits, scores, width, finished, end)


def test_masks_of_the_lowest_value():
    low = torch.finfo(F32).min
    logits, scores = make(2, 2, 3, 500, F32)
    logits[0, 0] = low            # all tokens masked alike: all as likely
    logits[0, 1, 7:] = low
    logits[1, :, ::2] = low
    compare(logits, scores, 8)
    logits[1, 0] = 200.0
    logits[1, 0, 3] = 1e30        # far above all others
    compare(logits, scores, 4)


def test_values_that_are_no_order():
    """A NaN or an infinity makes its beam's candidates NaN, before all others; other requests keep theirs."""
    from fhemamba_amd import clear

    logits, scores = make(3, 5, 3, 200, F32)
    clean = clear.beam_select(logits.cuda(), scores.cuda())
    logits[0, 1, 50] = math.nan
    logits[1, 2, 0] = math.inf
    scores[2, 0] = math.nan
    scores[3, 1] = math.inf
    got = clear.beam_select(logits.cuda(), scores.cuda())
    assert bool(torch.isnan(got.score[:4]).all())
    assert got.parent[:4].tolist() == [[1] * 3, [2] * 3, [0] * 3, [1] * 3]
    assert got.token[:4].tolist() == [[0, 1, 2]] * 4
    for a, b in zip(got, clean):
        assert torch.equal(a[4], b[4])
    # beams that are not read may hold anything
    dead = scores.clone()
    dead[:2], dead[2:4] = -math.inf, 0.0
    dead[0, 0] = -1.0
    finished = torch.zeros(5, 3, dtype=torch.bool)
    finished[1] = True
    got = clear.beam_select(logits.cuda(), dead.cuda(), finished=finished.cuda(), end=9)
    assert bool(torch.isfinite(got.score[0]).all()) and got.parent[0].tolist() == [0] * 3
    assert got.score[1].tolist() == [-math.inf] * 3


def test_views_and_default_width():
    from fhemamba_amd import clear

    logits, scores = make(4, 6, 4, 1001, F32)
    logits, scores = logits.cuda(), scores.cuda()
    wide = torch.cat([logits, logits], -1)
    want = clear.beam_select(logits, scores)
    assert want.score.shape == (6, 4)
    for view in (wide[..., :1001], wide[..., 1001:], logits.transpose(0, 1).contiguous().transpose(0, 1),
                 logits.permute(2, 0, 1).contiguous().permute(1, 2, 0)):
        for a, b in zip(clear.beam_select(view, scores.t().contiguous().t()), want):
            assert torch.equal(a, b)
    one = logits[:1, :1].expand(6, 4, 1001)  # one row for all
    for a, b in zip(clear.beam_select(one, scores), clear.beam_select(one.contiguous(), scores)):
        assert torch.equal(a, b)


def test_logits_past_32_bits():
    from fhemamba_amd import clear

    requests, beams, vocab = 1400, 32, 50280
    logits = torch.zeros(requests, beams, vocab, dtype=BF, device="cuda")
    scores = torch.full((requests, beams), -1.0, device="cuda")
    some, own = make(8, 1, beams, vocab, BF)
    logits[-1], scores[-1] = some[0].cuda(), own[0].cuda()
    got, alone = clear.beam_select(logits, scores, 4), clear.beam_select(some.cuda(), own.cuda(), 4)
    for a, b in zip(got, alone):
        assert torch.equal(a[-1], b[0])
    assert got.token[0].tolist() == [0, 1, 2, 3] and got.parent[0].tolist() == [0] * 4
    assert bool((got.token[:-1] == got.token[0]).all())


def test_refusals():
    from fhemamba_amd import clear

    logits, scores = torch.zeros(2, 3, 10, device="cuda"), torch.zeros(2, 3, device="cuda")
    none = torch.zeros(2, 3, dtype=torch.bool, device="cuda")
    parent = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    state = torch.zeros(6, 4, device="cuda")
    bad = [(lambda: clear.beam_select(logits.half(), scores), "float32 or bfloat16"),
           (lambda: clear.beam_select(logits[0], scores), "axes"),
           (lambda: clear.beam_select(logits, scores[:1]), "shape"),
           (lambda: clear.beam_select(logits, scores, 33), "width"),
           (lambda: clear.beam_select(logits, scores, 0), "width"),
           (lambda: clear.beam_select(logits[..., :2], scores, 7), "width"),
           (lambda: clear.beam_select(logits, scores, finished=none), "end"),
           (lambda: clear.beam_select(logits, scores, finished=none, end=10), "end"),
           (lambda: clear.beam_select(logits, scores, finished=none.int(), end=1), "type"),
           (lambda: clear.beam_select(logits[:0], scores[:0]), "requests"),

           (lambda: clear.beam_select(torch.zeros(1, 33, 4, device="cuda"), torch.zeros(1, 33, device="cuda")), "32 beams"),
           (lambda: clear.beam_select(logits, scores.clone().requires_grad_(True)), "no gradient"),
           (lambda: clear.reorder_states([], parent), "no states"),
           (lambda: clear.reorder_states(state, parent.long()), "type"),
           (lambda: clear.reorder_states(state[:5], parent), "6 beams and 5 rows"),
           (lambda: clear.reorder_states(state, parent[0]), "requests"),
           (lambda: clear.reorder_states(state.t(), parent, slots=parent), "contiguous"),
           (lambda: clear.reorder_states([state, state[:4]], parent, slots=parent), "same number"),
           (lambda: clear.reorder_states(state, parent, slots=parent[:1]), "shape"),
           (lambda: clear.reorder_states([state, state.cpu()], parent), "one GPU"),
           (lambda: clear.reorder_states(state.cpu(), parent), "on the GPU"),
           (lambda: clear.reorder_states(state.clone().requires_grad_(True), parent), "no gradient"),
           (lambda: clear.reorder_states(torch.zeros(6, device="cuda")[:0], parent, slots=parent), "rows")]
    for call, match in bad:
        with pytest.raises(ValueError, match=match):
            call()


@pytest.mark.parametrize("B", [1, 2, 4, 5, 8, 16, 17, 32])
def test_states_follow(B):
    from fhemamba_amd import clear

    gen = torch.Generator().manual_seed(B)
    R = 5
    cache = R * B + 3
    for slotted in (False, True):
        slots = torch.randperm(cache, generator=gen)[: R * B].reshape(R, B).to(torch.int32) if slotted else None
        parent = torch.randint(0, B, (R, B), generator=gen).to(torch.int32)
        parent[0] = torch.arange(B).flip(0)  # rows change places
        parent[1] = torch.arange(B)
        parent[2, 0], parent[2, -1] = -1, B
        if slotted:
            slots[3, 0], slots[4, -1] = -1, cache
        states = [torch.randn(cache, 3, 16, 20, generator=gen), torch.randn(cache, 3, 7, generator=gen).to(BF),
                  torch.randn(cache, 5, generator=gen), torch.randint(0, 255, (cache, 13), generator=gen).to(torch.uint8),
                  torch.randn(cache, 1031, generator=gen).double(), torch.randn(cache, 0)]
        mine = [s.cuda() for s in states]
        clear.reorder_states(mine, parent.cuda(), slots=None if slots is None else slots.cuda())
        for got, s in zip(mine, states):
            assert torch.equal(got.cpu(), L.moved(s, parent, slots))


def test_more_states_than_a_launch_takes():
    from fhemamba_amd import clear

    states = [torch.randn(4, 1 + i % 9, device="cuda") for i in range(200)]
    parent = torch.tensor([[1, 0], [1, 1]], dtype=torch.int32, device="cuda")
    want = [s[[1, 0, 3, 3]].clone() for s in states]
    clear.reorder_states(states, parent)
    assert all(torch.equal(a, b) for a, b in zip(states, want))
    one = torch.randn(4, 33, device="cuda")
    view = one[1:3]  # rows of a larger cache, at any address
    want = view[[1, 0]].clone()
    clear.reorder_states(view, parent[:1])
    assert torch.equal(one[1:3], want)


def test_states_past_32_bits():
    from fhemamba_amd import clear

    state = torch.zeros(40, 1 << 26, device="cuda")  # rows of 2^28 bytes
    state[39], state[20, -1] = 3.0, 5.0
    parent = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    clear.reorder_states(state, parent, slots=torch.tensor([[20, 39]], dtype=torch.int32, device="cuda"))
    assert bool((state[20] == 3.0).all()) and float(state[39].sum()) == 5.0 and float(state[39, -1]) == 5.0


def test_a_saved_state_that_moved_is_seen():
    from fhemamba_amd import clear

    state, w = torch.randn(2, 8, device="cuda"), torch.randn(2, 8, device="cuda", requires_grad=True)
    y = (state * w).sum()
    clear.reorder_states([state], torch.tensor([[1, 0]], dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("B,width", [(4, 2), (8, 1), (32, 5), (2, 3), (1, 4), (3, 32)])
def test_states_follow_into_another_number_of_beams(B, width):
    """A choice that keeps fewer beams, or more, than there were: the states in the first rows, or slots, of each
    request; the other rows as they were."""
    from fhemamba_amd import clear

    gen = torch.Generator().manual_seed(B)
    R, pitch = 3, max(B, width)
    cache = R * pitch + 2
    choice = clear.beam_select(torch.randn(R, B, 50, generator=gen).cuda(), torch.randn(R, B, generator=gen).cuda(), width)
    for slots in (None, torch.randperm(cache, generator=gen)[: R * pitch].reshape(R, pitch).to(torch.int32)):
        states = [torch.randn(cache, 3, 8, generator=gen), torch.randn(cache, 7, generator=gen).to(BF)]
        at = torch.arange(R * pitch).reshape(R, pitch) if slots is None else slots.long()
        mine = [s.cuda() for s in states]
        clear.reorder_states(mine, choice.parent, beams=B, slots=None if slots is None else slots.cuda())
        for got, s in zip(mine, states):
            want = s.clone()
            for r in range(R):
                for j in range(width):
                    want[at[r, j]] = s[at[r, int(choice.parent[r, j])]]
            assert torch.equal(got.cpu(), want)
    state = torch.randn(6, 4, device="cuda")  # a parent that is no beam of those that were
    want = state[[1, 0, 2, 3, 4, 3]].clone()
    clear.reorder_states(state, torch.tensor([[1, 0, 2], [0, -1, 0]], dtype=torch.int32, device="cuda"), beams=2)
    assert torch.equal(state, want)
    state, parent = torch.zeros(12, 4, device="cuda"), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    for call, match in [(lambda: clear.reorder_states(state, parent, beams=33), "32 beams"),
                        (lambda: clear.reorder_states(state, parent, beams=0), "32 beams"),
                        (lambda: clear.reorder_states(state, parent, beams=7), "14 beams and 12 rows"),
                        (lambda: clear.reorder_states(state, parent, beams=4, slots=parent), "shape")]:
        with pytest.raises(ValueError, match=match):
            call()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("V", [40, 300, 5000, 50280])
def test_beams_whose_totals_are_near(V, dtype):
    """Two beams with the same logits in another order, but one: their best tokens' totals differ by 2^-33 at least
    and 2^-28 at most, either way, which the reference's sums, good to 2^-44, tell apart."""
    R = 60
    gen = torch.Generator().manual_seed(V)
    logits, scores = make(V, R, 2, V, dtype)
    for r in range(R):
        logits[r, 1] = logits[r, 0][torch.randperm(V, generator=gen)]
        sums = torch.exp(logits[r, 0].double()).sum().item()
        # one token of one of the beams gives way: its part of the sum is what the totals differ by
        want = sums * 2.0 ** (-33 + 5 * float(torch.rand((), generator=gen)))
        both = [logits[r, b].argmin() for b in range(2)]
        for b in range(2):
            logits[r, b, both[b]] = -math.inf
        logits[r, r % 2, both[r % 2]] = math.log(want)
    scores[:] = -2.0
    totals = logits.double().log_softmax(-1).amax(-1)
    apart = (totals[:, 0] - totals[:, 1]).abs()
    assert bool((apart > 2.0 ** -34).all()) and bool((apart < 2.0 ** -27).all())
    compare(logits, scores, 2)


def test_logits_far_apart():
    """One token far above the others of its thread and row, at any size: the sum is its own 1."""
    for top in (50.0, 800.0, 1e5, 1e30):
        for V in (3, 500, 5000):
            logits, scores = make(V, 4, 2, V, F32)
            logits[0, 0, 1], logits[1, 1, 0], logits[2, 0, 2], logits[3, :, V - 1] = top, top, top, top
            logits[2, 1] = -top
            compare(logits, scores, 1)
            if top <= 1e5:  # of 1e30 numbers of 64 bits keep nothing smaller than 1e14: the others would be ties there
                compare(logits, scores, 3)
