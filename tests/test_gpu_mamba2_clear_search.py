"""The model's own run of the operators round the mixer: training through embeddings and norms, projections in 8
bits, a beam search from a prompt."""
import json
import os

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from fhemamba_amd import mamba2_payload as M  # noqa: E402

pytestmark = pytest.mark.gpu
GOLDEN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden")


@pytest.fixture(scope="module")
def chain():
    return M.read_chain_payload(os.path.join(GOLDEN, "m2_chain_tiny_ar"))


def log_probs(chain, ids):
    """Log probabilities of the token behind `ids`, by the plain decode in 64 bits."""
    ar = chain.autoregressive
    final = M.decode_tokens(chain, ar.embedding_w[np.asarray(ids)], False)[0][-1]
    logits = (ar.embedding_w if ar.lm_head_w is None else ar.lm_head_w) @ final
    logits = logits if ar.lm_head_b is None else logits + ar.lm_head_b
    return logits - np.logaddexp.reduce(logits)


def search(chain, prompt, steps, beams, end):
    held = [(0.0, [])]
    for _ in range(steps):
        new = []
        for score, tokens in held:
            if end is not None and end in tokens:
                new.append((score, tokens + [end]))
            else:
                new += [(score + lp, tokens + [t]) for t, lp in enumerate(log_probs(chain, list(prompt) + tokens))]
        held = sorted(new, key=lambda c: -c[0])[:beams]
    return held


@pytest.mark.parametrize("beams,end", [(1, None), (3, None), (4, 2)])
def test_search_is_the_plain_search(chain, beams, end):
    from fhemamba_amd import mamba2_clear as C

    model = C.ClearMamba2(chain)
    vocab = chain.autoregressive.vocab
    prompts = [[1 % vocab, 3 % vocab, 0], [2 % vocab, 2 % vocab, 5 % vocab]]
    found = model.beam_search(torch.tensor(prompts, device="cuda"), 4, beams=beams, end=end)
    assert found.tokens.shape == (2, beams, 4) and found.score.shape == (2, beams)
    for r, prompt in enumerate(prompts):
        want = search(chain, prompt, 4, beams, end)
        assert found.tokens[r].tolist() == [t for _, t in want]
        np.testing.assert_allclose(found.score[r].cpu().numpy(), [s for s, _ in want], atol=1e-3)
    # prompts of other lengths, packed, find what each finds alone
    cu = torch.tensor([0, 3, 4], dtype=torch.int32, device="cuda")
    packed = model.beam_search(torch.tensor(prompts[0] + prompts[1][:1], device="cuda"), 4, beams=beams, end=end,
                               cu_seqlens=cu)
    assert torch.equal(packed.tokens[0], found.tokens[0])
    want = search(chain, prompts[1][:1], 4, beams, end)
    assert packed.tokens[1].tolist() == [t for _, t in want]


def test_one_beam_is_the_greedy_decode(chain):
    from fhemamba_amd import mamba2_clear as C

    ar = chain.autoregressive
    model = C.ClearMamba2(chain)
    found = model.beam_search(torch.tensor([ar.prompt_ids], device="cuda"), 3, beams=1)
    ids = list(ar.prompt_ids)
    for _ in range(3):
        ids.append(int(np.argmax(log_probs(chain, ids))))
    assert found.tokens[0, 0].tolist() == ids[len(ar.prompt_ids):]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_command_in_8_bits_with_beams(tmp_path, dtype):
    from fhemamba_amd import mamba2_clear as C

    out = str(tmp_path / "r.json")
    assert C.main([os.path.join(GOLDEN, "m2_chain_tiny_ar"), out, "--int8", "--dtype", dtype, "--beams", "3"]) == 0
    report = json.load(open(out))
    assert report["int8"] and max(report["relative_errors"]) <= C.INT8_TOLERANCE
    beams = report["beams"]
    chain = M.read_chain_payload(os.path.join(GOLDEN, "m2_chain_tiny_ar"))
    assert len(beams["tokens"]) == 3 and all(len(t) == chain.autoregressive.generate_tokens for t in beams["tokens"])
    assert beams["score"] == sorted(beams["score"], reverse=True)


def test_a_model_in_8_bits_serves_and_is_not_trained(chain):
    from fhemamba_amd import mamba2_clear as C

    model, exact = C.ClearMamba2(chain, int8=True), C.ClearMamba2(chain)
    ids = torch.tensor([[1, 2, 0, 3]], device="cuda") % chain.autoregressive.vocab
    with torch.no_grad():
        a, b = model.forward(model.embed(ids))[0], exact.forward(exact.embed(ids))[0]
        assert float((a - b).norm() / b.norm()) <= C.INT8_TOLERANCE
        states, alone = model.zero_states(1), []
        for t in range(4):  # token by token: the rows are rounded alike
            alone.append(model.step(model.embed(ids[:, t]), states))
        assert float((torch.stack(alone, 1) - a).norm() / a.norm()) <= 2e-2
    with pytest.raises(ValueError, match="not trained"):
        model.parameters()


def test_gradients_reach_embeddings_and_norms(chain):
    """The loss's gradient in the embeddings and each norm's weight, against differences of the loss."""
    from fhemamba_amd import mamba2_clear as C

    model = C.ClearMamba2(chain)
    ids = torch.randint(0, chain.autoregressive.vocab, (2, 9), generator=torch.Generator().manual_seed(1)).cuda()
    leaves = [model.embedding, model.norm_w] + [lay.weights[k] for lay in model.layers
                                                for k in ("block_norm_w", "gated_norm_w")]
    head = model.head = model.head.clone()  # the head stays as it is where it is tied
    for t in leaves:
        t.requires_grad_(True)
    grads = torch.autograd.grad(model.loss(ids), leaves)
    for t, g in zip(leaves, grads):
        with torch.no_grad():
            before, way = t.clone(), g / g.norm()
            f = []
            for s in (1.0, -1.0):
                t.copy_(before + s * 1e-2 * way)
                f.append(model.loss(ids).item())
            t.copy_(before)
        # losses around 5, good to 2^-20, over steps of 1e-2; the third derivative's part below 2%
        assert abs((f[0] - f[1]) / 2e-2 - float(g.norm())) <= 2e-2 * float(g.norm()) + 1e-3
    assert model.head is head


def test_ids_from_the_end_count_as_before(chain):
    from fhemamba_amd import mamba2_clear as C

    model = C.ClearMamba2(chain)
    ids = torch.tensor([-1, 0, -chain.autoregressive.vocab], device="cuda")
    assert torch.equal(model.embed(ids), model.embedding[ids])


def test_refusals(chain):
    from fhemamba_amd import mamba2_clear as C

    model = C.ClearMamba2(chain)
    ids = torch.zeros(1, 2, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="steps"):
        model.beam_search(ids, 0)
    with pytest.raises(ValueError, match="width"):
        model.beam_search(ids, 2, beams=33)
    bare = C.ClearMamba2(M.read_chain_payload(os.path.join(GOLDEN, "m2_chain_tiny")))
    with pytest.raises(ValueError, match="no client head"):
        bare.beam_search(ids, 2)
    with pytest.raises(ValueError, match="client head"):
        C.run(M.read_chain_payload(os.path.join(GOLDEN, "m2_chain_tiny")), beams=2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_model_in_8_bits_is_the_model_of_its_integers(chain, dtype, monkeypatch):
    """The same layers with the plain form of each 8-bit product.  The two round alike but where a quotient lies within
    32 bits' rounding of the middle of two integers, which moves one entry of a row by a 127th of the largest."""
    import layer_reference as L
    from fhemamba_amd import clear, mamba2_clear as C

    model = C.ClearMamba2(chain, dtype, int8=True)
    ids = torch.randint(0, chain.autoregressive.vocab, (3, 11), generator=torch.Generator().manual_seed(5)).cuda()

    def plain(x, weight, scale, bias=None):
        rows = x.cpu().reshape(-1, x.shape[-1])
        y = L.int8_linear(rows, weight.cpu(), scale.cpu(), None if bias is None else bias.cpu())
        return y.to(x.dtype).cuda().reshape(*x.shape[:-1], -1)

    with torch.no_grad():
        got = model.forward(model.embed(ids))[0]
        logits = model.logits(got)
        monkeypatch.setattr(clear, "int8_linear", plain)
        want = model.forward(model.embed(ids))[0]
        assert float((got - want).norm() / want.norm()) <= 2.0 ** -7
        want = model.logits(got)
        # each from the same hidden vectors: exact sums, then two 32-bit products and the type's rounding
        off = 2.0 ** -8 if dtype == torch.bfloat16 else 4 * 2.0 ** -24
        assert float((logits.float() - want.float()).norm() / want.float().norm()) <= 2 * off
