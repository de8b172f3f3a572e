"""The loss of packed texts does not depend on what lies before, behind or between them."""
import os

import pytest

torch = pytest.importorskip("torch")

from fhemamba_amd import mamba2_payload as M  # noqa: E402

pytestmark = pytest.mark.gpu
GOLDEN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden")


@pytest.mark.parametrize("before,behind", [(0, 5), (3, 0), (4, 70)])
def test_padding_of_a_packed_batch(before, behind):
    from fhemamba_amd import mamba2_clear as C

    chain = M.read_chain_payload(os.path.join(GOLDEN, "m2_chain_tiny_ar"))
    model = C.ClearMamba2(chain)
    gen = torch.Generator().manual_seed(1)
    ids = torch.randint(0, chain.autoregressive.vocab, (before + 11 + behind,), generator=gen).cuda()
    params = [p.requires_grad_(True) for p in model.parameters()]
    ends = torch.tensor([0, 6, 6, 7, 11], dtype=torch.int32, device="cuda")
    got = model.loss(ids, cu_seqlens=ends + before)
    grads = torch.autograd.grad(got, params)
    want = model.loss(ids[before:before + 11], cu_seqlens=ends)
    plain = torch.autograd.grad(want, params)
    # the same sums of 32 bits in another order
    assert abs(got.item() - want.item()) <= 2.0 ** -16 * want.item()
    for a, b in zip(grads, plain):
        assert float((a - b).norm()) <= 2.0 ** -13 * float(b.norm())


def test_nothing_to_score():
    """No tokens, and texts of a single one: nothing is scored, and the loss is zero."""
    from fhemamba_amd import mamba2_clear as C

    model = C.ClearMamba2(M.read_chain_payload(os.path.join(GOLDEN, "m2_chain_tiny_ar")))
    for n, ends in ((0, [0, 0]), (2, [0, 1, 2]), (3, [1, 1, 2])):
        ids = torch.zeros(n, dtype=torch.int64, device="cuda")
        assert model.loss(ids, cu_seqlens=torch.tensor(ends, dtype=torch.int32, device="cuda")).item() == 0.0
