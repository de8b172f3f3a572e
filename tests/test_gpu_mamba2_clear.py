"""The model in the clear against the payload's plain references in 64 bits, its states, its gradient."""
import json
import os

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from fhemamba_amd import mamba2_payload as M  # noqa: E402

pytestmark = pytest.mark.gpu
GOLDEN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden")


@pytest.fixture(scope="module")
def synthetic(tmp_path_factory):
    """Two layers of 4 heads of 16, 32 states, five test tokens."""
    return M.synthetic_chain(str(tmp_path_factory.mktemp("clear")), seed=3, n_layers=2, n_test_tokens=5, d_model=32,
                             d_inner=64, num_heads=4, head_dim=16, state_size=32,
                             degrees={k: 8 for k in M.DEGREES})


def states_near(mine, plain):
    for a, b in zip(mine, plain):
        assert np.linalg.norm(a.ssm - b.ssm) <= 1e-4 * np.linalg.norm(b.ssm)
        assert np.linalg.norm(np.stack(a.fifo) - np.stack(b.fifo)) <= 1e-4 * np.linalg.norm(np.stack(b.fifo))


@pytest.mark.parametrize("name", ["m2_chain_tiny", "m2_chain_tiny_ar"])
def test_golden_payloads(name, tmp_path):
    """The exporter's chains through the command: prompt in one call, then token by token."""
    from fhemamba_amd import mamba2_clear as C

    out, states = str(tmp_path / "r.json"), str(tmp_path / "s.npz")
    assert C.main([os.path.join(GOLDEN, name), out, "--states", states]) == 0
    report = json.load(open(out))
    chain = M.read_chain_payload(os.path.join(GOLDEN, name))
    _, plain = M.decode_tokens(chain, chain.input_embeddings, False)
    got = np.load(states)
    for i, s in enumerate(plain):
        assert np.linalg.norm(got[f"ssm_{i:02d}"] - s.ssm) <= 1e-4 * np.linalg.norm(s.ssm)
    if name.endswith("_ar"):
        head = report["head"]
        finals, _ = M.decode_tokens(chain, chain.input_embeddings, False)
        assert head["greedy"] == [chain.autoregressive.select(f) for f in finals]
        assert [t[0] for t in head["top_index"]] == head["greedy"]
        np.testing.assert_allclose([t[0] for t in head["top_logprob"]], head["logprob"], atol=1e-5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_then_steps(synthetic, dtype):
    from fhemamba_amd import mamba2_clear as C

    for k in (1, 3, 5):
        report = C.run(synthetic, prompt_tokens=k, dtype=dtype)
        assert report["passed"] and report["step_tokens"] == 5 - k and "head" not in report


def test_packed_prompts_and_slots(synthetic):
    """Prompts of 2, 0 and 3 tokens packed, then a token each from slots: as each on its own."""
    from fhemamba_amd import mamba2_clear as C

    model = C.ClearMamba2(synthetic)
    rng = np.random.default_rng(1)
    tokens = rng.normal(0, 1, (5, 32)).astype(np.float32)
    cu = torch.tensor([0, 2, 2, 5], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        hidden, states = model.forward(torch.as_tensor(tokens, device="cuda"), cu_seqlens=cu)
    nexts = rng.normal(0, 1, (3, 32)).astype(np.float32)
    slots = torch.tensor([2, 0, 1], dtype=torch.int32, device="cuda")
    step = model.step(torch.as_tensor(nexts, device="cuda"), states, slots=slots)
    for row, (a, b) in enumerate([(0, 2), (2, 2), (2, 5)]):
        plain = [M.zero_state(lay) for lay in synthetic.layers]
        if b > a:
            want, plain = M.decode_tokens(synthetic, tokens[a:b], False)
            np.testing.assert_allclose(hidden[a:b].cpu().numpy(), want, atol=1e-3)
        want, plain = M.decode_tokens(synthetic, nexts[[slots.tolist().index(row)]], False, plain)
        np.testing.assert_allclose(step[slots.tolist().index(row)].cpu().numpy(), want[0], atol=1e-3)
        states_near(C.layer_states(states, row), plain)


def test_prompt_state_starts_the_plain_decode(synthetic):
    from fhemamba_amd import mamba2_clear as C

    model = C.ClearMamba2(synthetic)
    tokens = torch.as_tensor(synthetic.input_embeddings, dtype=torch.float32, device="cuda")
    with torch.no_grad():
        _, states = model.forward(tokens[None, :4])
    got, _ = M.decode_tokens(synthetic, synthetic.input_embeddings[4:], False, C.layer_states(states))
    assert np.linalg.norm(got[0] - synthetic.expected_final[4]) <= 1e-4 * np.linalg.norm(synthetic.expected_final[4])


def test_loss_and_its_gradient():
    """The loss is the plain decode's, its gradient the differences', and a step against it lowers it."""
    from fhemamba_amd import mamba2_clear as C

    chain = M.read_chain_payload(os.path.join(GOLDEN, "m2_chain_tiny_ar"))
    model = C.ClearMamba2(chain)
    gen = torch.Generator().manual_seed(1)
    ids = torch.randint(0, chain.autoregressive.vocab, (11,), generator=gen).cuda()
    cu = torch.tensor([0, 6, 6, 11], dtype=torch.int32, device="cuda")
    params = [p.requires_grad_(True) for p in model.parameters()]
    loss = model.loss(ids, cu_seqlens=cu)
    grads = torch.autograd.grad(loss, params)
    loss = loss.item()
    ar = chain.autoregressive
    head = ar.embedding_w if ar.lm_head_w is None else ar.lm_head_w
    want = []
    for a, b in ((0, 6), (6, 11)):
        mine = ids[a:b].cpu().numpy()
        finals, _ = M.decode_tokens(chain, chain.autoregressive.embedding_w[mine], False)
        for f, t in zip(finals[:-1], mine[1:]):
            logits = head @ f
            if chain.autoregressive.lm_head_b is not None:
                logits = logits + chain.autoregressive.lm_head_b
            want.append(np.logaddexp.reduce(logits) - logits[t])
    assert abs(loss - np.mean(want)) <= 1e-4 * np.mean(want)
    with torch.no_grad():
        before = [p.clone() for p in params]
        scale = 1e-2 / float(sum(g.square().sum() for g in grads).sqrt())
        moved = []
        for s in (1.0, -1.0):
            for p, b, g in zip(params, before, grads):
                p.copy_(b + s * scale * g)
            moved.append(model.loss(ids, cu_seqlens=cu).item())
    # along the gradient: its own norm, from losses around 5 good to 2^-20 over steps of 1e-2
    slope, norm = (moved[0] - moved[1]) / 2e-2, float(sum(g.double().square().sum() for g in grads).sqrt())
    assert moved[1] < loss < moved[0]
    assert abs(slope - norm) <= 2e-2 * norm + 1e-3


def test_refusals(synthetic):
    from fhemamba_amd import mamba2_clear as C

    model = C.ClearMamba2(synthetic)
    with pytest.raises(ValueError, match="no client head"):
        model.logits(torch.zeros(1, 32, device="cuda"))
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        C.ClearMamba2(synthetic, torch.float16)
    with pytest.raises(ValueError, match="prompt tokens"):
        C.run(synthetic, prompt_tokens=9)
