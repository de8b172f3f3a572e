"""Forward-mode derivatives, which the operators do not have, are refused and not dropped."""
import pytest

torch = pytest.importorskip("torch")
fwd = torch.autograd.forward_ad

pytestmark = pytest.mark.gpu


def test_tangents_are_refused():
    from fhemamba_amd import clear

    def dual(t):
        return fwd.make_dual(t, torch.ones_like(t))

    z = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    targets = torch.zeros(2, dtype=torch.int64, device="cuda")
    with fwd.dual_level(), torch.no_grad():
        calls = [lambda: clear.ssm_scan(dual(z(1, 4, 2, 8)), z(1, 4, 2), z(1, 4, 2), z(1, 4, 1, 8), z(1, 4, 1, 8)),
                 lambda: clear.ssm_scan(z(1, 4, 2, 8), z(1, 4, 2), z(1, 4, 2), z(1, 4, 1, 8), z(1, 4, 1, 8),
                                        initial_state=dual(z(1, 2, 8, 8))),
                 lambda: clear.ssm_step(z(1, 2, 8, 8), dual(z(1, 2, 8)), z(1, 2), z(1, 2), z(1, 1, 8), z(1, 1, 8)),
                 lambda: clear.causal_conv(z(1, 4, 8), dual(z(8, 4))),
                 lambda: clear.causal_conv_step(z(1, 3, 8), dual(z(1, 8)), z(8, 4)),
                 lambda: clear.token_logprobs(dual(z(2, 9)), targets)]
        for call in calls:
            with pytest.raises(ValueError, match="forward-mode"):
                call()
    with fwd.dual_level(), pytest.raises(ValueError, match="forward-mode"):  # the same where gradients are on
        clear.token_logprobs(dual(z(2, 9)).requires_grad_(True), targets)
    with fwd.dual_level():  # a level without a tangent refuses nothing
        assert clear.token_logprobs(z(2, 9), targets).logprob.shape == (2,)
