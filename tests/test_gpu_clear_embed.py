"""Embedding lookup and the table's gradient by sorted tokens, against 64 bits."""
import pytest

torch = pytest.importorskip("torch")

import clear_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def lookup(weight, ids, scale):
    real = (ids >= 0)[..., None]
    return torch.where(real, weight[ids.clamp(min=0)] * scale, torch.zeros((), dtype=torch.float64))


def compare(weight, ids, scale, seed=0):
    from fhemamba_amd import clear

    gen = torch.Generator().manual_seed(seed)
    dy = torch.randn(*ids.shape, weight.shape[1], generator=gen).to(weight.dtype)
    ref = weight.double().requires_grad_(True)
    want = lookup(ref, ids, scale)
    (grad,) = torch.autograd.grad(want, ref, dy.double())
    mine = weight.cuda().requires_grad_(True)
    got = clear.embed(mine, ids.cuda(), scale=scale)
    assert got.dtype == weight.dtype and got.shape == want.shape
    assert R.rel(got, want) <= R.bound(got)
    (back,) = torch.autograd.grad(got, mine, dy.cuda(), retain_graph=True)
    assert back.dtype == weight.dtype
    assert R.rel(back, grad) <= R.bound(back)
    assert not bool(back.cpu()[grad.abs().sum(-1) == 0].any())  # rows that no token names
    (again,) = torch.autograd.grad(got, mine, dy.cuda())
    assert torch.equal(back, again)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("vocab,channels", [(1, 1), (2, 3), (93, 64), (255, 5), (256, 256), (257, 333), (513, 1100),
                                            (9973, 8), (50280, 16)])
@pytest.mark.parametrize("tokens", [1, 2, 63, 64, 65, 128, 129, 1000, 5001])
def test_lookup_and_gradient(tokens, vocab, channels, dtype):
    print(f"[embed] {tokens} of {vocab} x {channels} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(tokens + vocab)
    weight = torch.randn(vocab, channels, generator=gen).to(dtype)
    ids = torch.randint(0, vocab, (tokens,), generator=gen)
    ids = torch.where(torch.rand(tokens, generator=gen) < 0.3, ids % 3 % vocab, ids)  # some often
    ids[torch.rand(tokens, generator=gen) < 0.1] = -1
    compare(weight, ids, 1.0 if tokens % 2 else 27.5, tokens)


@pytest.mark.parametrize("counts", [(64, 65), (63, 1, 64, 1, 200), (1, 64, 128, 129), (700,), (65, 65, 65), (0, 3000, 0, 1),
                                    (130, 0, 62, 66)])
def test_runs_at_the_ends_of_pieces(counts):
    """Tokens that occur as often as the pieces are long, one more, and over many pieces."""
    ids = torch.cat([torch.full((n,), 7 * i, dtype=torch.int64) for i, n in enumerate(counts)])
    gen = torch.Generator().manual_seed(len(ids))
    weight = torch.randn(300, 70, generator=gen)
    compare(weight, ids[torch.randperm(len(ids), generator=gen)], 1.0)
    compare(weight.to(BF), ids, 2.0)


def test_many_tokens():
    """Longer pieces: 150001 tokens, half of them of one row; and none at all of any row."""
    gen = torch.Generator().manual_seed(3)
    weight = torch.randn(1000, 12, generator=gen)
    ids = torch.randint(0, 1000, (150001,), generator=gen)
    ids[torch.rand(150001, generator=gen) < 0.5] = 300
    compare(weight, ids, 1.0)
    compare(weight, torch.full((500,), -1), 1.0)
    for n in (100, 128, 129):  # of one row, and of none
        compare(weight, torch.full((n,), 999), 1.0)
        compare(weight, torch.full((n,), -1), 1.0)


def test_axes_strides_and_no_tokens():
    from fhemamba_amd import clear

    weight = torch.randn(50, 40, device="cuda")
    ids = torch.randint(0, 50, (6, 8), device="cuda")
    for w in (weight[:, 3:24], weight[::2], weight.t()[:, :33], weight[:1].expand(50, 40)):
        some = ids % w.shape[0]
        assert torch.equal(clear.embed(w, some), w[some])
        leaf = w.detach().requires_grad_(True)
        (g,) = torch.autograd.grad(clear.embed(leaf, some[:, ::2]).sum(), leaf)
        want = torch.zeros(leaf.shape, device="cuda").index_add_(
            0, some[:, ::2].reshape(-1), torch.ones(24, leaf.shape[1], device="cuda"))
        assert torch.equal(g, want)
    leaf = weight.requires_grad_(True)
    assert clear.embed(weight, ids[0, 0]).shape == (40,)
    none = clear.embed(leaf, ids[:0])
    assert none.shape == (0, 8, 40)
    (g,) = torch.autograd.grad(none.sum(), leaf)
    assert not bool(g.any())
    # a scaled table of a tied head: both gradients arrive
    (g,) = torch.autograd.grad(clear.embed(leaf, ids).sum() + (leaf * leaf).sum(), leaf)
    (e,) = torch.autograd.grad(leaf[ids].sum() + (leaf * leaf).sum(), leaf)
    torch.testing.assert_close(g, e, rtol=R.F32, atol=R.F32)


def test_ids_that_are_no_tokens():
    from fhemamba_amd import clear

    leaf = torch.randn(10, 21, device="cuda", requires_grad=True)
    ids = torch.tensor([3, -1, 10, 2 ** 40, -2 ** 63, 9, 3], device="cuda")
    y = clear.embed(leaf, ids)
    assert torch.equal(y[[0, 5, 6]], leaf[[3, 9, 3]]) and not bool(y[[1, 4]].any())
    assert bool(torch.isnan(y[[2, 3]]).all())
    dy = torch.randn(7, 21, device="cuda")
    dy[[1, 2, 3, 4]] = float("nan")  # no gradient from them
    (g,) = torch.autograd.grad(y, leaf, dy)
    want = torch.zeros(10, 21, device="cuda")
    want[3], want[9] = dy[0] + dy[6], dy[5]
    assert torch.equal(g, want)


def test_table_past_32_bits():
    """Rows and gradients behind 2^31 elements."""
    from fhemamba_amd import clear

    vocab, channels = 1 << 21, 1100
    weight = torch.zeros(vocab, channels, dtype=BF, device="cuda")
    at = torch.tensor([vocab - 1, 5, 1 << 20, vocab - 1], device="cuda")
    weight[at] = torch.randn(4, channels, device="cuda").to(BF)
    leaf = weight.requires_grad_(True)
    y = clear.embed(leaf, at)
    assert torch.equal(y, weight[at])
    (g,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert bool((g[vocab - 1] == 2).all()) and bool((g[5] == 1).all()) and bool((g[1 << 20] == 1).all())
    assert float(g[:, 0].float().sum()) == 4.0


def test_gradient_of_differences():
    from fhemamba_amd import clear

    gen = torch.Generator().manual_seed(4)
    w = torch.randn(30, 17, generator=gen).cuda().requires_grad_(True)
    ids, c = torch.randint(0, 30, (40,), generator=gen).cuda(), torch.randn(40, 17, generator=gen).cuda()
    loss = lambda t: (clear.embed(t, ids, scale=1.5) * c).double().sum()  # noqa: E731
    (g,) = torch.autograd.grad(loss(w), w)
    d = torch.randn(30, 17, generator=gen).cuda()
    with torch.no_grad():  # linear: the difference is the gradient, up to 2^-24 of 680 terms over a step of 2
        slope = (loss(w + d) - loss(w - d)).item() / 2
    want = float((g * d).double().sum())
    assert abs(slope - want) <= 2.0 ** -16 * float((g * d).norm()) + 1e-4


def test_refusals():
    from fhemamba_amd import clear

    w, ids = torch.randn(5, 4, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for call, match in [(lambda: clear.embed(w.half(), ids), "float32 or bfloat16"),
                        (lambda: clear.embed(w[0], ids), "axes"),
                        (lambda: clear.embed(w, ids.int()), "type"), (lambda: clear.embed(w, ids.cpu()), "cpu"),
                        (lambda: clear.embed(w, [1]), "tensor"), (lambda: clear.embed(w[:0], ids), "vocabulary"),
                        (lambda: clear.embed(w, ids, scale=float("inf")), "finite")]:
        with pytest.raises(ValueError, match=match):
            call()


def ids_of(counts):
    return torch.cat([torch.full((n,), 3 * i, dtype=torch.int64) for i, n in enumerate(counts)])


# 129 to 32768 tokens are cut into pieces of 32: a row of as many, one more and one less, at a piece's begin, at its
# end and across it
@pytest.mark.parametrize("counts", [(32,) * 5, (33,) * 5, (31,) * 6, (32, 33, 31, 64, 65, 63, 96), (1, 31, 32, 33, 32, 96),
                                    (1, 32, 31, 32, 33, 31, 40), (16, 32, 16, 33, 63, 64, 65), (31, 33, 31, 33, 1, 64),
                                    (95, 33, 32, 97, 1), (32, 0, 160, 32), (128, 1, 128, 31, 1)])
def test_rows_as_long_as_a_piece(counts):
    ids = ids_of(counts)
    assert 128 < len(ids) <= 32768
    gen = torch.Generator().manual_seed(len(ids))
    weight = torch.randn(3 * len(counts) + 2, 70, generator=gen)
    compare(weight, ids, 1.0)
    compare(weight, ids[torch.randperm(len(ids), generator=gen)], 1.0)
    compare(weight.to(BF), torch.cat([ids, torch.full((9,), -1)]), 2.0)


@pytest.mark.parametrize("last,piece", [(1, 63), (500, 64)])
def test_rows_as_long_as_a_longer_piece(last, piece):
    """Over 64000 tokens: rows of one less, as many and one more."""
    counts = [62, 63, 64, 65, 1, 62, 63, 126, 127, 128, 129] * 72 + [last]
    ids = ids_of(counts)
    assert (len(ids) + 1023) // 1024 == piece
    weight = torch.randn(3 * len(counts), 12, generator=torch.Generator().manual_seed(last))
    compare(weight, ids, 1.0)
