"""Norms with the gate or the residual before them, and their gradients, against 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

import clear_reference as R  # noqa: E402
import layer_reference as L  # noqa: E402

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
SIZES = [(1, 1), (3, 3), (5, 64), (2, 255), (7, 256), (4, 257), (9, 333), (130, 768), (3, 1001), (6, 1536), (2, 1537),
         (3, 4096), (2, 5000), (2, 8192), (2, 16384), (2, 20001), (1, 32768)]


def n(gen, *shape, dtype=F32):
    return torch.randn(shape, generator=gen).to(dtype)


def check(got, want, dtype, terms=None):
    """`terms`: what `want` is a difference of, each with the rounding of a 32-bit sum."""
    got, want = got.detach().cpu(), want.detach()
    assert got.dtype == dtype and got.shape == want.shape and bool(torch.isfinite(got).all())
    more = R.F32 * float(terms.detach().norm()) if terms is not None else 0.0
    off = float((got.double() - want).norm())
    assert off <= R.bound(got) * float(want.norm()) + more, (off, float(want.norm()), more)


def leaf(t):
    return t.double().requires_grad_(True)


@pytest.mark.parametrize("types", [(F32, F32), (F32, BF), (BF, BF)])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,channels", SIZES)
def test_norm(rows, channels, gated, types):
    from fhemamba_amd import clear

    print(f"[norm] {rows} x {channels} {gated} {types}", flush=True)
    gen = torch.Generator().manual_seed(rows * channels)
    x, w, dn = n(gen, rows, channels, dtype=types[0]), 1 + 0.2 * n(gen, channels), n(gen, rows, channels, dtype=types[1])
    z = n(gen, rows, channels, dtype=types[0]) if gated else None
    ref = [leaf(t) for t in ((x, w, z) if gated else (x, w))]
    want = L.norm(ref[0], ref[1], ref[2] if gated else None, 1, 1e-5)
    grads = torch.autograd.grad(want, ref, dn.double())
    mine = [t.cuda().requires_grad_(True) for t in ((x, w, z) if gated else (x, w))]
    got = clear.rms_norm(mine[0], mine[1], gate=mine[2] if gated else None, dtype=types[1])
    check(got, want, types[1])
    # the gradient of v is r (g - unit mean(g unit)); both of its terms are as large as r g
    v = ref[0].detach() if not gated else (ref[0] * ref[2] * torch.sigmoid(ref[2])).detach()
    rg = dn.double() * ref[1].detach() / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-5)
    mine = torch.autograd.grad(got, mine, dn.cuda())
    act = ref[2].detach() * torch.sigmoid(ref[2].detach()) if gated else torch.ones(())
    check(mine[0], grads[0], types[0], rg * act)
    check(mine[1], grads[1], F32)
    if gated:
        check(mine[2], grads[2], types[0], rg * ref[0].detach())


@pytest.mark.parametrize("types", [(F32, F32), (F32, BF), (BF, BF)])
@pytest.mark.parametrize("scaled", [False, True])
@pytest.mark.parametrize("rows,channels", SIZES)
def test_add_norm(rows, channels, scaled, types):
    from fhemamba_amd import clear

    print(f"[add_norm] {rows} x {channels} {scaled} {types}", flush=True)
    gen = torch.Generator().manual_seed(rows + channels)
    h, u, w = n(gen, rows, channels, dtype=types[0]), n(gen, rows, channels, dtype=types[1]), 1 + 0.2 * n(gen, channels)
    s = 0.5 + 0.1 * n(gen, channels) if scaled else None
    dn, dh = n(gen, rows, channels, dtype=types[1]), n(gen, rows, channels, dtype=types[0])
    ref = [leaf(t) for t in ((h, u, w, s) if scaled else (h, u, w))]
    want = L.add_norm(ref[0], ref[1], ref[2], ref[3] if scaled else None, 1e-5)
    mine = [t.cuda().requires_grad_(True) for t in ((h, u, w, s) if scaled else (h, u, w))]
    got = clear.add_norm(mine[0], mine[1], mine[2], scale=mine[3] if scaled else None)
    check(got.normed, want[0], types[1])
    check(got.hidden, want[1], types[0])
    total = want[1].detach()
    rg = dn.double() * ref[2].detach() / torch.sqrt((total * total).mean(-1, keepdim=True) + 1e-5)
    for outs in ((0, 1), (0,), (1,)):  # a result that nothing uses has no gradient
        d = [(dn, dh)[i] for i in outs]
        grads = torch.autograd.grad([want[i] for i in outs], ref, [t.double() for t in d], retain_graph=True,
                                    allow_unused=True)
        back = torch.autograd.grad([got[i] for i in outs], mine, [t.cuda() for t in d], retain_graph=True)
        for i, t in enumerate((types[0], types[1], F32, F32)[:len(ref)]):
            exact = torch.zeros_like(ref[i]) if grads[i] is None else grads[i]
            terms = (rg, rg, None, rg * ref[1].detach())[i] if 0 in outs else None
            check(back[i], exact, t, terms)


@pytest.mark.parametrize("rows,channels,groups", [(4, 12, 3), (5, 666, 2), (3, 7, 7), (9, 1536, 4), (2, 40000, 2),
                                                  (3, 3075, 3)])
def test_groups(rows, channels, groups):
    from fhemamba_amd import clear

    gen = torch.Generator().manual_seed(channels)
    x, z, dn, w = n(gen, rows, channels), n(gen, rows, channels), n(gen, rows, channels), n(gen, channels)
    ref = [leaf(t) for t in (x, w, z)]
    want = L.norm(ref[0], ref[1], ref[2], groups, 1e-5)
    grads = torch.autograd.grad(want, ref, dn.double())
    mine = [t.cuda().requires_grad_(True) for t in (x, w, z)]
    got = clear.rms_norm(mine[0], mine[1], gate=mine[2], groups=groups)
    check(got, want, F32)
    back = torch.autograd.grad(got, mine, dn.cuda())
    v = (ref[0] * ref[2] * torch.sigmoid(ref[2])).detach().reshape(rows, groups, -1)
    r = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-5)
    rg = (r * (dn.double() * ref[1].detach()).reshape(v.shape)).reshape(rows, channels)
    check(back[0], grads[0], F32, rg * ref[2].detach())
    check(back[1], grads[1], F32)
    check(back[2], grads[2], F32, rg * ref[0].detach())


@pytest.mark.parametrize("rows,channels", [(5000, 64), (1100, 1537), (300001, 4)])
def test_many_rows(rows, channels):
    """More rows than wavefronts, either way; sums over many rows."""
    from fhemamba_amd import clear

    gen = torch.Generator().manual_seed(rows)
    h, u, w, s = n(gen, rows, channels), n(gen, rows, channels), n(gen, channels), n(gen, channels)
    dn, dh = n(gen, rows, channels), n(gen, rows, channels)
    ref = [leaf(t) for t in (h, u, w, s)]
    want = L.add_norm(*ref, 1e-5)
    grads = torch.autograd.grad(want, ref, (dn.double(), dh.double()))
    mine = [t.cuda().requires_grad_(True) for t in (h, u, w, s)]
    got = clear.add_norm(*mine[:3], scale=mine[3])
    back = torch.autograd.grad(got, mine, (dn.cuda(), dh.cuda()))
    again = torch.autograd.grad(clear.add_norm(*mine[:3], scale=mine[3]), mine, (dn.cuda(), dh.cuda()))
    for g, e, a in zip(back, grads, again):
        check(g, e, F32)
        assert torch.equal(g, a)


def test_strides_alignment_and_axes():
    from fhemamba_amd import clear

    gen = torch.Generator().manual_seed(5)
    whole = n(gen, 4, 6, 1000).cuda()
    w = n(gen, 97).cuda()
    for dtype in (F32, BF):
        t = whole.to(dtype)
        for view in (t[..., 3:100], t[:, ::2, 1:98], t.transpose(0, 1)[..., 900:997], t[0, :, 5:102],
                     t[2, 3, 7:104], t[:1, :1, :97].expand(3, 5, 97), t[..., :1].expand(4, 6, 97),
                     t[..., ::10][..., :97]):
            for z in (None, view.flip(0)):
                got = clear.rms_norm(view, w, gate=z)
                want = clear.rms_norm(view.contiguous(), w, gate=None if z is None else z.contiguous())
                assert got.shape == view.shape and torch.equal(got, want)
    x = whole[..., 1:98].requires_grad_(True)  # gradients that autograd makes of one number, and of broadcast rows
    (g,) = torch.autograd.grad(clear.rms_norm(x, w).sum(), x)
    (e,) = torch.autograd.grad(clear.rms_norm(x, w), x, torch.ones(4, 6, 97, device="cuda"))
    assert torch.equal(g, e)
    one = whole[:1, :1, :97].detach().requires_grad_(True)
    (g,) = torch.autograd.grad(clear.rms_norm(one.expand(4, 6, 97), w).sum(), one)
    (e,) = torch.autograd.grad(clear.rms_norm(one, w).sum(), one)
    torch.testing.assert_close(g, 24 * e, rtol=R.F32, atol=R.F32)


def test_no_rows():
    from fhemamba_amd import clear

    w = torch.randn(8, device="cuda", requires_grad=True)
    x = torch.randn(0, 3, 8, device="cuda", requires_grad=True)
    y = clear.rms_norm(x, w, gate=x.detach())
    assert y.shape == (0, 3, 8)
    g = torch.autograd.grad(y.sum(), (x, w))
    assert g[0].shape == x.shape and not bool(g[1].any())
    got = clear.add_norm(x, x.detach(), w, scale=w.detach())
    assert got.normed.shape == got.hidden.shape == (0, 3, 8)
    assert not bool(torch.autograd.grad(got.normed.sum(), w)[0].any())


def test_values_that_are_not_finite_stay_in_their_rows():
    from fhemamba_amd import clear

    x = torch.randn(9, 300, device="cuda")
    z = torch.randn(9, 300, device="cuda")
    clean = clear.rms_norm(x, torch.ones(300, device="cuda"), gate=z)
    x[1, 7], x[3, 299], z[5, 0] = math.nan, math.inf, math.nan
    z[7] = z[7].clamp(max=0) * 1e30
    z[7, 1] = -3e38
    got = clear.rms_norm(x, torch.ones(300, device="cuda"), gate=z)
    for row in (1, 5):
        assert bool(torch.isnan(got[row]).all())
    assert not bool(torch.isfinite(got[3]).all())
    assert bool(torch.isfinite(got[7]).all())  # a closed gate is nothing
    rest = [0, 2, 4, 6, 8]
    assert torch.equal(got[rest], clean[rest])


def test_zeros_and_eps():
    from fhemamba_amd import clear

    x, w = torch.zeros(2, 40, device="cuda", requires_grad=True), torch.ones(40, device="cuda")
    y = clear.rms_norm(x, w, eps=1e-12)
    (g,) = torch.autograd.grad(y.sum(), x)
    assert not bool(y.any())
    torch.testing.assert_close(g, torch.full_like(g, 1e6), rtol=2.0 ** -20, atol=0)
    assert bool(torch.isnan(clear.rms_norm(x, w, eps=0.0)).all())
    got = clear.rms_norm(torch.full((1, 40), -3.0, device="cuda"), w, eps=0.0)
    torch.testing.assert_close(got, torch.full_like(got, -1.0), rtol=2.0 ** -20, atol=0)


def test_offsets_past_32_bits():
    from fhemamba_amd import clear

    rows, channels = 70000, 32768
    x = torch.zeros(rows, channels, dtype=BF, device="cuda")
    picked = [0, 65535, 65536, rows - 1]
    gen = torch.Generator().manual_seed(1)
    some = n(gen, 4, channels, dtype=BF)
    x[picked] = some.cuda()
    w = n(gen, channels)
    leaf = x.requires_grad_(True)
    y = clear.rms_norm(leaf, w.cuda())
    ref = some.double().requires_grad_(True)
    want = L.norm(ref, w.double(), None, 1, 1e-5)
    check(y[picked], want, BF)
    assert not bool(y[1:65535].any())
    dn = n(gen, 4, channels, dtype=BF)
    (grad,) = torch.autograd.grad(want, ref, dn.double())
    dy = torch.zeros_like(x)
    dy[picked] = dn.cuda()
    (back,) = torch.autograd.grad(y, leaf, dy)
    # the terms are about as large as the gradient: rows of 32768 are hardly along it
    check(back[picked], grad, BF, grad)
    assert not bool(back[1:65535].any())


def test_differences():
    """The gradient along a random direction is the loss's difference, in 32 bits over a step of 2^-6."""
    from fhemamba_amd import clear

    gen = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    h, u, w, s, z, c = r(6, 50), r(6, 50), r(50), r(50), r(6, 50), r(6, 50)

    def loss(h, u, w, s, z):
        normed, hidden = clear.add_norm(h, u, w, scale=s, eps=0.1)
        return (clear.rms_norm(normed, w, gate=z, groups=5, eps=0.1) * c).double().sum() + (hidden * c).double().sum()

    leaves = [t.requires_grad_(True) for t in (h, u, w, s, z)]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    ways = [r(*t.shape) for t in leaves]
    with torch.no_grad():
        f = [loss(*(t + k * 2.0 ** -6 * d for t, d in zip(leaves, ways))).item() for k in (-2, -1, 1, 2)]
    # fourth order: the step's error is of 2^-24 times a fifth derivative; the values' 2^-24 over the step 2^-18
    slope = (f[0] - 8 * f[1] + 8 * f[2] - f[3]) / (12 * 2.0 ** -6)
    want = sum(float((g * d).double().sum()) for g, d in zip(grads, ways))
    size = sum(float((g.double() * d.double()).square().sum()) for g, d in zip(grads, ways)) ** 0.5
    assert abs(slope - want) <= 2e-3 * size


def test_saved_tensors_that_change_are_seen():
    from fhemamba_amd import clear

    w = torch.ones(16, device="cuda", requires_grad=True)
    h, u = torch.randn(3, 16, device="cuda"), torch.randn(3, 16, device="cuda")
    got = clear.add_norm(h, u, w)
    got.hidden.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        got.normed.sum().backward()
    got = clear.add_norm(h, u, w)
    h.add_(1.0)  # not needed
    got.normed.sum().backward()


def test_refusals():
    from fhemamba_amd import clear

    x, w = torch.randn(3, 16, device="cuda"), torch.ones(16, device="cuda")
    bad = [(lambda: clear.rms_norm(x.half(), w), "float32 or bfloat16"), (lambda: clear.rms_norm(x, w[:8]), "shape"),
           (lambda: clear.rms_norm(x, w.to(BF)), "type"), (lambda: clear.rms_norm(x, w, groups=3), "groups"),
           (lambda: clear.rms_norm(x, w, groups=0), "groups"), (lambda: clear.rms_norm(x, w, gate=x.to(BF)), "type"),
           (lambda: clear.rms_norm(x, w, gate=x[:2]), "shape"), (lambda: clear.rms_norm(x, w, eps=-1.0), "eps"),
           (lambda: clear.rms_norm(x, w, eps=math.nan), "eps"),
           (lambda: clear.rms_norm(x.to(BF), w, dtype=F32), "dtype"),
           (lambda: clear.rms_norm(x, w.cpu()), "cpu"), (lambda: clear.rms_norm(x[:, :0], w[:0]), "channels"),
           (lambda: clear.rms_norm(x.new_empty(1, 32769), x.new_empty(32769)), "32768"),
           (lambda: clear.add_norm(x.to(BF), x, w), "type"), (lambda: clear.add_norm(x, x[:2], w), "shape"),
           (lambda: clear.add_norm(x, x, w, scale=w[:3]), "shape"),
           (lambda: clear.add_norm(x, x, w, eps=math.inf), "eps"),
           (lambda: clear.add_norm(x.new_empty(1, 32769), x.new_empty(1, 32769), x.new_empty(32769)), "32768")]
    for call, match in bad:
        with pytest.raises(ValueError, match=match):
            call()
    leaf = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(clear.rms_norm(leaf, w).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# (size of the values, eps): r = 1 / size leaves r^3 no room in 32 bits from about 1e13 on, or below 1e-12
RANGES = [(1e13, 1e-5), (1e15, 1e-5), (1e17, 1e-5), (1e18, 0.0), (1e-13, 0.0), (1e-13, 1e-30), (1e-16, 1e-30), (0.0, 1e-30)]


@pytest.mark.parametrize("size,eps", RANGES)
@pytest.mark.parametrize("form", ["plain", "gated", "sum", "scaled"])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_gradients_of_very_large_and_very_small_rows(dtype, form, size, eps):
    """The squares' sum is far from 32 bits' ends, and so are the gradients, of the size of r g."""
    from fhemamba_amd import clear

    rows, channels = 5, 97
    gen = torch.Generator().manual_seed(7)
    x, other = (size * n(gen, rows, channels)).to(dtype), n(gen, rows, channels, dtype=dtype)
    w, s, dn = 1 + 0.2 * n(gen, channels), 0.5 + 0.1 * n(gen, channels), n(gen, rows, channels, dtype=dtype)
    if form == "gated":
        tensors, call = (x, w, other), lambda a, b, c: clear.rms_norm(a, b, gate=c, eps=eps)
        plain = lambda a, b, c: L.norm(a, b, c, 1, eps)  # noqa: E731
        v = x.double() * other.double() * torch.sigmoid(other.double())
    elif form == "plain":
        tensors, call = (x, w), lambda a, b: clear.rms_norm(a, b, eps=eps)
        plain = lambda a, b: L.norm(a, b, None, 1, eps)  # noqa: E731
        v = x.double()
    else:
        update = (size * other.double()).to(dtype)
        scaled = form == "scaled"
        tensors = (x, update, w, s) if scaled else (x, update, w)
        call = lambda a, b, c, d=None: clear.add_norm(a, b, c, scale=d, eps=eps).normed  # noqa: E731
        plain = lambda a, b, c, d=None: L.add_norm(a, b, c, d, eps)[0]  # noqa: E731
        v = x.double() + update.double() * (s.double() if scaled else 1.0)
    ref, mine = [leaf(t) for t in tensors], [t.cuda().requires_grad_(True) for t in tensors]
    want, got = plain(*ref), call(*mine)
    check(got, want, dtype)
    # both terms of the gradient of v are as large as r g
    rg = dn.double() * w.double() / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    act = other.double() * torch.sigmoid(other.double())
    terms = {"plain": (rg, None), "gated": (rg * act, None, rg * x.double()), "sum": (rg, rg, None),
             "scaled": (rg, rg * s.double(), None, (rg * other.double() * size).norm(dim=0))}[form]
    grads = torch.autograd.grad(want, ref, dn.double())
    for g, e, t, term in zip(torch.autograd.grad(got, mine, dn.cuda()), grads, tensors, terms):
        check(g, e, t.dtype, term)


@pytest.mark.parametrize("low,high", [(-8, -4), (-20, -10), (-60, -40), (-85, -75), (-2, 2), (4, 40)])
def test_gates_element_by_element(low, high):
    """Each result for itself: a closed gate's is as exact as an open one's.

    In steps of 2^-24 of a result: the sigmoid's exponential 2 (a unit of the hardware's), its factor 2, 1 + e 1, the
    reciprocal 2, the products with the gate and x 2, together 9; the row's size as much from its
    products, 5.5 from ten sums and a square, 0.5 from eps, the root's unit 2; two more products: 28."""
    from fhemamba_amd import clear

    gen = torch.Generator().manual_seed(-low)
    rows, channels = 400, 64
    z = low + (high - low) * torch.rand(rows, channels, generator=gen)
    # so that the row's values are all of the same size
    x = (torch.exp(-z.double().clamp(max=0)) * (1 + torch.rand(rows, channels, generator=gen))).float()
    w = 1 + torch.rand(channels, generator=gen)
    got = clear.rms_norm(x.cuda(), w.cuda(), gate=z.cuda()).cpu().double()
    want = L.norm(x.double(), w.double(), z.double(), 1, 1e-5)
    off = ((got - want) / want).abs().max().item() * 2.0 ** 24
    assert off <= 28, off


def test_gates_at_the_ends_of_their_type():
    """Open ones pass x on, closed ones nothing, and one that is no number spoils its row."""
    from fhemamba_amd import clear

    w = torch.ones(8, device="cuda")
    z = torch.tensor([[3e38, 1e4, 200.0, 89.0, 0.0, -200.0, -1e4, -3e38], [1.0] * 7 + [math.nan],
                      [1.0] * 7 + [-math.inf], [-104.0] * 8, [0.0] * 8], device="cuda")
    x = torch.full((5, 8), 1e-38, device="cuda")
    x[0, 1:] = 1.0
    got = clear.rms_norm(x, w, gate=z)
    assert bool(torch.isfinite(got[0]).all()) and not bool(got[0, 4:].any()) and bool((got[0, :4] > 0).all())
    assert bool(torch.isnan(got[1]).all()) and bool(torch.isnan(got[2]).all())
    assert not bool(got[3:].any())


@pytest.mark.parametrize("low,high", [(-8, -4), (-60, -40), (-85, -75), (-2, 2), (4, 40)])
def test_gates_of_16_bits_element_by_element(low, high):
    """The 28 steps of 2^-24 above beneath the rounding to 16 bits: half a step of the result's own size."""
    from fhemamba_amd import clear

    gen = torch.Generator().manual_seed(-low)
    rows, channels = 400, 64
    z = (low + (high - low) * torch.rand(rows, channels, generator=gen)).to(BF)
    x = (torch.exp(-z.double().clamp(max=0)) * (1 + torch.rand(rows, channels, generator=gen))).to(BF)
    w = 1 + torch.rand(channels, generator=gen)
    got = clear.rms_norm(x.cuda(), w.cuda(), gate=z.cuda()).cpu().double()
    want = L.norm(x.double(), w.double(), z.double(), 1, 1e-5)
    step = torch.exp2(torch.floor(torch.log2(want.abs())) - 7)
    over = ((got - want).abs() - step / 2) / want.abs()
    assert over.max().item() * 2.0 ** 24 <= 28, over.max().item() * 2.0 ** 24


def test_squares_at_the_ends_of_32_bits():
    """What counts is the squares' sum: beyond 2^128 a row gives zeros, and so does its gradient."""
    from fhemamba_amd import clear

    w = torch.ones(768, device="cuda")
    x = torch.zeros(4, 768, device="cuda")
    x[0, 5] = 2.0 ** 63.5                 # its square is 2^127
    x[1] = 2.0 ** 60                      # 768 of 2^120
    x[2] = 2.0 ** 59                      # 768 of 2^118, below 2^128
    x[3] = 2.0 ** -60                     # 768 of 2^-120
    leaf = x.requires_grad_(True)
    y = clear.rms_norm(leaf, w, eps=0.0)
    want = torch.zeros(4, 768, device="cuda")
    want[0, 5], want[2:] = 768 ** 0.5, 1.0
    torch.testing.assert_close(y, want, rtol=2.0 ** -16, atol=0)
    dy = torch.arange(768, device="cuda") % 2 * 2.0 - 1.0
    (g,) = torch.autograd.grad(y, leaf, dy.expand(4, 768))
    assert bool(torch.isfinite(g).all()) and not bool(g[1].any())
    torch.testing.assert_close(g[2], dy * 2.0 ** -59, rtol=2.0 ** -16, atol=0)
    torch.testing.assert_close(g[3], dy * 2.0 ** 60, rtol=2.0 ** -16, atol=0)
