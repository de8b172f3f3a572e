"""What torch's autograd is told: states that are updated in place, tangents, outputs of their own."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def scan_args(tokens=40, heads=2, head_dim=16, states=24):
    gen = torch.Generator().manual_seed(1)
    n = lambda *s: torch.randn(s, generator=gen).cuda()  # noqa: E731
    return [n(1, tokens, heads, head_dim), torch.rand(1, tokens, heads, generator=gen).cuda(),
            -torch.rand(1, tokens, heads, generator=gen).cuda(), n(1, tokens, 1, states), n(1, tokens, 1, states),
            n(heads)]


@pytest.mark.parametrize("through", ["itself", "a view"])
def test_a_step_of_a_saved_state_is_seen(through):
    """A scan from a cache, whose backward pass needs the state as it was, and a step of that cache between."""
    from fhemamba_amd import clear

    args = scan_args()
    whole = torch.randn(3, 2, 16, 24, device="cuda")
    state = whole[:1]
    args[0].requires_grad_(True)
    y = clear.ssm_scan(*args, initial_state=state)
    one = [a[:, 0].detach() if i < 5 else a for i, a in enumerate(args)]
    with torch.no_grad():
        clear.ssm_step(state if through == "itself" else whole, *one)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("through", ["itself", "a view"])
def test_a_convolution_step_of_a_saved_state_is_seen(through):
    from fhemamba_amd import clear

    x, w = torch.randn(1, 20, 8, device="cuda"), torch.randn(8, 4, device="cuda", requires_grad=True)
    whole = torch.randn(2, 3, 8, device="cuda")
    state = whole[:1]
    y = clear.causal_conv(x, w, initial_state=state)
    with torch.no_grad():
        clear.causal_conv_step(state if through == "itself" else whole, x[:, 0], w)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_steps_of_other_states_and_in_inference_mode():
    from fhemamba_amd import clear

    args = scan_args()
    state, other = torch.randn(1, 2, 16, 24, device="cuda"), torch.randn(1, 2, 16, 24, device="cuda")
    args[0].requires_grad_(True)
    y = clear.ssm_scan(*args, initial_state=state)
    one = [a[:, 0].detach() if i < 5 else a for i, a in enumerate(args)]
    with torch.inference_mode():
        clear.ssm_step(other, *one)
        made = torch.zeros(1, 2, 16, 24, device="cuda")
        clear.ssm_step(made, *one)
        x, w = torch.randn(1, 8, device="cuda"), torch.randn(8, 4, device="cuda")
        clear.causal_conv_step(torch.zeros(1, 3, 8, device="cuda"), x, w)
    y.sum().backward()
    assert bool(torch.isfinite(args[0].grad).all())
