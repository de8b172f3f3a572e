"""The batched 64-bit scan against the plain one, and how the scan cuts sequences.  No GPU is needed."""
import pytest

torch = pytest.importorskip("torch")

import clear_batched as B  # noqa: E402
import test_gpu_clear_scan as T  # noqa: E402
import test_gpu_clear_scan_segments as S  # noqa: E402


@pytest.mark.parametrize("initial", [True, False])
def test_batched_reference(initial):
    lengths = [3, 0, 17, 1]
    d = T.make(1, 21, 4, 3, 5, 2, torch.float32, seqs=4 if initial else None)
    gen = torch.Generator().manual_seed(2)
    grads = T.normal(gen, 21, 4, 3), T.normal(gen, 4, 4, 3, 5)
    y, h, got = B.scan(d, lengths, grads, device="cpu")
    y0, h0, want = T.reference(d, lengths, grads)
    assert set(got) == set(want)
    for a, b in [(y, y0), (h, h0), *((got[k], want[k]) for k in want)]:
        torch.testing.assert_close(a, b.detach(), rtol=1e-12, atol=1e-12)


def test_segments_of_the_test_shapes():
    """Short tests' sequences are cut at 64 tokens; a long prompt of many heads is cut longer."""
    assert B.segment_lengths([1500], False, (2, 64, 128, 1), torch.bfloat16)[0] == 64
    assert B.segment_lengths([70] * 150, False, (3, 64, 64, 1), torch.float32) == []
    assert min(B.segment_lengths([30011], False, (24, 64, 128, 1), torch.bfloat16)) > 64


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", list(S.PLANS))
def test_segments_of_the_long_test_shapes(name, dtype):
    """What the GPU tests of long segments rely on, so that another rule for them is seen here too."""
    S.plan_of(name, dtype)
