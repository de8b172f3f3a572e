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
