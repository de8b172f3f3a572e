"""Rows of logits in which all but a NaN is masked off."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,vocab,column", [(5, 5000, 7), (5, 5000, 4999), (4, 50280, 0), (4, 50280, 4095),
                                               (4, 50280, 30001), (3, 9, 4), (5000, 70, 33)])
def test_a_nan_among_masked_tokens(rows, vocab, column, dtype):
    """log softmax of such a row is NaN throughout, as its entropy and its gradient are; the rows around it are as
    they are without it."""
    from fhemamba_amd import clear

    logits = torch.randn(rows, vocab, generator=torch.Generator().manual_seed(vocab)).to(dtype)
    logits[1] = -math.inf
    good = logits.clone()
    logits[1, column] = math.nan
    targets = torch.zeros(rows, dtype=torch.int64)
    targets[1] = column
    print(f"[logprob] nan {rows} x {vocab} {column} {dtype}", flush=True)
    leaf = logits.cuda().requires_grad_(True)
    got = clear.token_logprobs(leaf, targets.cuda(), top=3)
    one = torch.ones(rows, device="cuda")
    (grad,) = torch.autograd.grad([got.logprob, got.entropy], leaf, [one, one])
    assert math.isnan(got.logprob[1].item()) and math.isnan(got.entropy[1].item())
    assert bool(torch.isnan(got.top_logprob[1]).all())
    assert bool(torch.isnan(grad[1]).all())
    keep = [r for r in range(rows) if r != 1]
    want = clear.token_logprobs(good.cuda(), targets.cuda(), top=3)
    assert all(torch.equal(a.detach()[keep], b[keep]) for a, b in zip(got, want))
    assert bool(torch.isfinite(grad[keep]).all())


def test_masked_target_of_such_a_row():
    from fhemamba_amd import clear

    logits = torch.full((2, 6000), -math.inf, device="cuda")
    logits[:, 5000] = math.nan
    got = clear.token_logprobs(logits, torch.tensor([3, -1], device="cuda"))
    assert math.isnan(got.logprob[0].item()) and got.logprob[1].item() == 0.0
    assert bool(torch.isnan(got.entropy).all())
