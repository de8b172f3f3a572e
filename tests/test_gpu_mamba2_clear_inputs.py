"""What callers hand to the model: a stream of 64 bits, ids that are no tokens, prompts without a token."""
import os

import pytest

torch = pytest.importorskip("torch")

from fhemamba_amd import mamba2_payload as M  # noqa: E402

pytestmark = pytest.mark.gpu
GOLDEN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden")


@pytest.fixture(scope="module")
def chain():
    return M.read_chain_payload(os.path.join(GOLDEN, "m2_chain_tiny_ar"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_stream_of_64_bits_stays_one(chain, dtype):
    """With output projections of nothing the layers add nothing, and the final norm is the input's to 64 bits; its
    gradient too."""
    from fhemamba_amd import mamba2_clear as C

    model = C.ClearMamba2(chain, dtype)
    x = torch.randn(1, 6, model.norm_w.shape[0], generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    want = x / torch.sqrt((x * x).mean(-1, keepdim=True) + model.norm_eps) * model.norm_w.double().cpu()
    plain = model.forward(x.cuda())[0]
    assert plain.dtype == torch.float64  # with what the layers add, in 32 bits, near the stream of 32 bits
    narrow = model.forward(x.float().cuda())[0]
    assert float((plain - narrow).norm() / narrow.norm()) <= C.TOLERANCE[dtype]
    for lay in model.layers:
        lay.weights["out_proj_w"].zero_()
    leaf = x.cuda().requires_grad_(True)
    got = model.forward(leaf)[0]
    assert got.dtype == torch.float64 and float((got.detach().cpu() - want).norm() / want.norm()) <= 1e-14
    assert float((model.step(x[0].cuda(), model.zero_states(6)).cpu() - want[0]).norm() / want.norm()) <= 1e-14
    ref = x.clone().requires_grad_(True)
    way = torch.randn(want.shape, generator=torch.Generator().manual_seed(2), dtype=torch.float64)
    (e,) = torch.autograd.grad(ref / torch.sqrt((ref * ref).mean(-1, keepdim=True) + model.norm_eps)
                               * model.norm_w.double().cpu(), ref, way)
    (g,) = torch.autograd.grad(got, leaf, way.cuda())
    # two sums of some tens of terms each, 2^-53 a term
    assert float((g.cpu() - e).norm() / e.norm()) <= 1e-13


def test_ids_outside_of_the_table_are_refused(chain):
    from fhemamba_amd import mamba2_clear as C

    model, vocab = C.ClearMamba2(chain), chain.autoregressive.vocab
    good = torch.tensor([[1, 0, vocab - 1], [-1, 2, -vocab]], device="cuda")
    cu = torch.tensor([0, 2, 6], dtype=torch.int32, device="cuda")
    assert bool(torch.isfinite(model.loss(good))) and bool(torch.isfinite(model.loss(good.reshape(-1), cu_seqlens=cu)))
    found = model.beam_search(good, 2, beams=2)
    for bad in (vocab, -vocab - 1, 2 ** 62, -2 ** 63):
        ids = good.clone()
        ids[1, 1] = bad
        for call in (lambda: model.loss(ids), lambda: model.loss(ids.reshape(-1), cu_seqlens=cu),
                     lambda: model.beam_search(ids, 2, beams=2),
                     lambda: model.beam_search(ids.reshape(-1), 2, beams=2, cu_seqlens=cu)):
            with pytest.raises(ValueError, match="outside of the table"):
                call()
        rows = model.embed(ids)  # without a wait: no row of the table, and none of zeros
        assert bool(torch.isnan(rows[1, 1]).all()) and torch.equal(rows[0], model.embed(good[0]))
    again = model.beam_search(good, 2, beams=2)
    assert torch.equal(found.tokens, again.tokens) and torch.equal(found.score, again.score)


@pytest.mark.parametrize("ends", [[0, 0, 3], [0, 3, 3], [0, 1, 1, 3], [2, 1, 3], [0, 4], [-1, 3]])
def test_prompts_without_a_token_are_refused(chain, ends):
    from fhemamba_amd import mamba2_clear as C

    model = C.ClearMamba2(chain)
    ids = torch.tensor([1, 2, 0], device="cuda")
    with pytest.raises(ValueError, match="one token or more"):
        model.beam_search(ids, 2, beams=2, cu_seqlens=torch.tensor(ends, dtype=torch.int32, device="cuda"))


def test_captured_loss(chain):
    """A capture waits for nothing: there the ids are not looked at."""
    from fhemamba_amd import mamba2_clear as C

    model, vocab = C.ClearMamba2(chain), chain.autoregressive.vocab
    ids = torch.tensor([[1, 2, 0, 3]], device="cuda") % vocab
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad(), torch.cuda.stream(side):
        model.loss(ids)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        loss = model.loss(ids)
    for turn in range(3):
        ids.copy_((ids + 1) % vocab)
        graph.replay()
        with torch.no_grad():
            assert torch.equal(loss, model.loss(ids))
