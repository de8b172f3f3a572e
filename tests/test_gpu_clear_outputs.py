"""Log probabilities and entropies are tensors of their own, also where they are changed in place."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lead", [(6,), (2, 3)])
def test_log_probabilities_changed_in_place(lead):
    from fhemamba_amd import clear

    leaf = torch.randn(*lead, 300, device="cuda", requires_grad=True)
    targets = torch.randint(0, 300, lead, device="cuda")
    mask = torch.rand(lead, device="cuda")
    got = clear.token_logprobs(leaf, targets)
    (want,) = torch.autograd.grad((got.logprob * mask).sum() + got.entropy.sum(), leaf)
    got = clear.token_logprobs(leaf, targets)
    (grad,) = torch.autograd.grad(got.logprob.mul_(mask).sum() + got.entropy.sum(), leaf)
    assert torch.equal(grad, want)


def test_outputs_without_gradients_share_nothing():
    """What a later backward pass keeps of one of them is not touched by a change of the other."""
    from fhemamba_amd import clear

    logits, targets = torch.randn(5, 100, device="cuda"), torch.zeros(5, dtype=torch.int64, device="cuda")
    with torch.no_grad():
        got = clear.token_logprobs(logits, targets, top=2)
    kept = got.logprob.clone()
    weight = torch.ones(5, device="cuda", requires_grad=True)
    loss = (weight * got.logprob).sum()
    got.entropy.zero_()
    loss.backward()
    assert torch.equal(weight.grad, kept)
