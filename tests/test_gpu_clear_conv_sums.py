"""The convolution's weights' gradients over more tokens and channels than a workgroup sums, against 64 bits."""
import pytest

torch = pytest.importorskip("torch")

import clear_reference as R  # noqa: E402
import test_gpu_clear_conv as T  # noqa: E402

pytestmark = pytest.mark.gpu

# 32-bit sums of up to 2^12 products are off by 2^-24 sqrt(2^12) of their terms' norm, with a factor of 8 for terms
# that cancel
SUMS = 2.0 ** -15


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("channels,taps", [(200, 4), (1792, 4), (264, 8), (131, 3)])
@pytest.mark.parametrize("lengths", [[1500, 1500], [700, 1, 0, 2100, 300, 2]])
def test_sums_over_many_workgroups(lengths, channels, taps, dtype):
    from fhemamba_amd import clear

    S, total = len(lengths), sum(lengths)
    assert total > 16 * 128  # each of the last sums' sixteen wavefronts has several parts
    d = T.make(channels, total, channels, taps, dtype, S)
    packed = len(set(lengths)) > 1
    print(f"[conv sums] {channels} x {taps} {lengths} {dtype}", flush=True)
    names = ("x", "weight", "bias", "initial")
    shape = d["x"].shape if packed else (S, lengths[0], channels)
    leaves = {k: (d[k].cuda().reshape(shape) if k == "x" else d[k].cuda()).requires_grad_(True) for k in names}
    ends = torch.tensor(lengths).cumsum(0).tolist()
    cu = torch.tensor([0, *ends], dtype=torch.int32, device="cuda") if packed else None
    y, last = clear.causal_conv(leaves["x"], leaves["weight"], leaves["bias"], initial_state=leaves["initial"],
                                cu_seqlens=cu, return_state=True)
    got = torch.autograd.grad([y, last], list(leaves.values()), [d["dy"].cuda().reshape(shape), d["dstate"].cuda()])
    ref = {k: d[k].double().requires_grad_(True) for k in names}
    y0, last0 = R.conv(ref["x"], ref["weight"], ref["bias"], ref["initial"], R.spans(lengths))
    loss = (y0 * d["dy"].double()).sum() + (last0 * d["dstate"].double()).sum()
    want = torch.autograd.grad(loss, list(ref.values()))
    assert R.rel(y.reshape(d["x"].shape), y0) <= R.bound(y)
    assert torch.equal(last.cpu().double(), last0.detach())
    for k, a, b in zip(names, got, want):
        bound = SUMS if k in ("weight", "bias") else R.bound(a)
        assert R.rel(a.reshape(d[k].shape), b) <= bound, k
        if k in ("weight", "bias"):  # each channel by itself: a part that is lost or counted twice is seen
            rows, whole = (a.double().cpu() - b).reshape(channels, -1), b.reshape(channels, -1)
            assert bool((rows.norm(dim=1) <= 16 * SUMS * whole.norm(dim=1).clamp(min=1.0)).all()), k
