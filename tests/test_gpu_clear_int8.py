"""Rows in 8-bit integers and products of them, against exact integer sums."""
import math

import pytest

torch = pytest.importorskip("torch")

import clear_reference as R  # noqa: E402
import layer_reference as L  # noqa: E402

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def rows_of(gen, rows, channels, dtype):
    return (torch.exp(torch.randn(rows, 1, generator=gen)) * torch.randn(rows, channels, generator=gen)).to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,channels", [(1, 1), (3, 2), (5, 3), (7, 4), (2, 63), (9, 255), (4, 257), (130, 768),
                                           (3, 1001), (2, 1537), (2, 4096), (2, 5001), (1, 16384), (2, 32768)])
def test_rounding(rows, channels, dtype):
    from fhemamba_amd import clear

    gen = torch.Generator().manual_seed(rows * channels)
    x = rows_of(gen, rows, channels, dtype)
    got = clear.quantize_rows(x.cuda())
    values, scale = L.quantize(x)
    assert torch.equal(got.values.cpu(), values) and torch.equal(got.scale.cpu(), scale)


def test_rounding_of_special_rows():
    from fhemamba_amd import clear

    x = torch.zeros(10, 40)
    x[1, 3] = math.nan
    x[2, 39] = -math.inf
    x[3] = torch.linspace(-1, 1, 40)
    x[4, 0] = 1.0
    x[4, 1:] = 0.5  # 63.5: to the even one
    x[5] = 3.4e38
    x[6, 7] = 1e-44  # its scale is 0 in 32 bits
    x[7] = 2.0 ** -140 * torch.arange(40)
    x[8, 5] = -0.0
    x[9] = torch.arange(40) - 127.0
    got = clear.quantize_rows(x.cuda())
    values, scale = L.quantize(x)
    keep = [0, 3, 4, 5, 7, 8, 9]
    assert torch.equal(got.values.cpu()[keep], values[keep]) and torch.equal(got.scale.cpu()[keep], scale[keep])
    assert got.values[4, 1].item() == 64
    for row in (1, 2):
        assert not bool(got.values[row].any()) and math.isnan(got.scale[row].item())
    assert not bool(got.values[6].any()) and got.scale[6].item() == 0.0


def test_rounding_of_views_and_many_rows():
    from fhemamba_amd import clear

    t = torch.randn(4, 5, 300, device="cuda")
    for view in (t[..., 1:98], t.transpose(0, 1), t[..., ::2], t[:1].expand(4, 5, 300), t[1, 2]):
        a, b = clear.quantize_rows(view), clear.quantize_rows(view.contiguous())
        assert a.values.shape == view.shape and a.scale.shape == view.shape[:-1]
        assert torch.equal(a.values, b.values) and torch.equal(a.scale, b.scale)
    none = clear.quantize_rows(t[:0])
    assert none.values.shape == (0, 5, 300) and none.scale.shape == (0, 5)
    rows = 70000
    x = torch.zeros(rows, 32768, dtype=BF, device="cuda")
    x[rows - 1] = 1.0
    got = clear.quantize_rows(x)
    assert bool((got.values[-1] == 127).all()) and not bool(got.values[: rows - 1].any())


def compare(rows, inputs, outputs, dtype, bias=True, seed=0):
    from fhemamba_amd import clear

    print(f"[int8] {rows} x {inputs} x {outputs} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(seed + rows + 3 * inputs + 7 * outputs)
    x = rows_of(gen, rows, inputs, dtype)
    w = torch.randint(-128, 128, (outputs, inputs), generator=gen, dtype=torch.int8)
    ws, b = torch.rand(outputs, generator=gen) / 127, torch.randn(outputs, generator=gen) if bias else None
    got = clear.int8_linear(x.cuda(), w.cuda(), ws.cuda(), None if b is None else b.cuda())
    want = L.int8_linear(x, w, ws, b)
    assert got.dtype == dtype and got.shape == want.shape
    # an exact sum to 24 bits, two products, one addition: four roundings in 32 bits of what is added, then the type's
    values, scale = L.quantize(x)
    size = (values.double() @ w.double().t()).abs() * scale.double()[:, None] * ws.double()
    size = size + (0 if b is None else b.double().abs())
    off = (got.cpu().double() - want).abs()
    limit = 4 * 2.0 ** -24 * size + (2.0 ** -8 * want.abs() if dtype == BF else 0.0) + 1e-40
    assert bool((off <= limit).all()), float((off - limit).max())


@pytest.mark.parametrize("inputs", [1, 15, 16, 17, 63, 64, 65, 96, 128, 129, 255, 333, 768, 1001, 1536, 4100])
@pytest.mark.parametrize("rows,outputs", [(1, 1), (1, 643), (2, 17), (7, 130), (8, 64), (15, 16), (16, 643),
                                          (17, 15), (33, 64), (64, 65), (65, 3), (100, 130), (250, 768)])
def test_few_rows(rows, outputs, inputs):
    compare(rows, inputs, outputs, BF if (rows + inputs) % 2 else F32, bias=outputs % 2 == 0)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,inputs,outputs", [(1300, 96, 3352), (700, 129, 6401), (2049, 64, 2048), (1281, 768, 3353),
                                                 (4097, 1, 1100), (2300, 1001, 2001), (130, 333, 40000),
                                                 (65, 768, 66000), (9000, 256, 500)])
def test_many_rows(rows, inputs, outputs, dtype):
    compare(rows, inputs, outputs, dtype, bias=rows % 2 == 0)


@pytest.mark.parametrize("rows", [3, 2500])
def test_largest_sums(rows):
    """32768 products of -127 and -128: as large as the sums can be."""
    from fhemamba_amd import clear

    x = torch.full((rows, 32768), -2.0, device="cuda")
    w = torch.full((2000, 32768), -128, dtype=torch.int8, device="cuda")
    got = clear.int8_linear(x, w, torch.ones(2000, device="cuda"))
    want = 32768 * 2.0 * 128
    assert float((got.double() - want).abs().max()) <= 4 * 2.0 ** -24 * want


def test_results_past_32_bits():
    """2.5e9 results; and more rows than a launch rounds."""
    from fhemamba_amd import clear

    gen = torch.Generator().manual_seed(3)
    rows, outputs = 50000, 50280
    x, w = rows_of(gen, 8, 64, BF), torch.randint(-127, 128, (outputs, 64), generator=gen, dtype=torch.int8)
    wide = torch.zeros(rows, 64, dtype=BF, device="cuda")
    picked = [0, 1, 42700, 42711, 42712, 49151, 49998, 49999]
    wide[picked] = x.cuda()
    ws = torch.rand(outputs, generator=gen)
    got = clear.int8_linear(wide, w.cuda(), ws.cuda())
    want = L.int8_linear(x, w, ws, None)
    assert float((got[picked].cpu().double() - want).norm()) <= R.BF16 * float(want.norm())
    assert not bool(got[2:42700].any()) and not bool(got[49152:49998].any())
    rows = (1 << 20) + 5
    many = torch.arange(rows, device="cuda").float()[:, None].expand(rows, 3)
    q = clear.quantize_rows(many)
    assert bool((q.values[1:] == 127).all()) and not bool(q.values[0].any())
    assert torch.equal(q.scale, torch.arange(rows).div(127.0).cuda())


def test_views_axes_and_alignment():
    from fhemamba_amd import clear

    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(3, 4, 200, generator=gen, device="cuda")
    flat = torch.randint(-127, 128, (70 * 96 + 64,), generator=gen, device="cuda").to(torch.int8)
    ws = torch.rand(70, generator=gen, device="cuda")
    for shift in (0, 1, 4, 16):  # a table that begins anywhere
        w = flat[shift: shift + 70 * 96].view(70, 96)
        for view in (x[..., 5:101], x.transpose(0, 1)[..., :96], x[1, 2, 100:196], x[..., ::2][..., :96],
                     x[:1, :1, :96].expand(3, 4, 96)):
            got = clear.int8_linear(view, w, ws)
            want = clear.int8_linear(view.contiguous(), w.clone(), ws)
            assert got.shape == (*view.shape[:-1], 70) and torch.equal(got, want)
    got = clear.int8_linear(x[..., :70], flat[:4900].view(70, 70).t(), ws)
    assert torch.equal(got, clear.int8_linear(x[..., :70], flat[:4900].view(70, 70).t().contiguous(), ws))
    assert clear.int8_linear(x[:0, :, :96], flat[:6720].view(70, 96), ws).shape == (0, 4, 70)


@pytest.mark.parametrize("rows,outputs", [(5, 70), (1000, 6000)])
def test_rows_that_are_not_finite(rows, outputs):
    from fhemamba_amd import clear

    x = torch.randn(rows, 96, device="cuda")
    w = torch.randint(-127, 128, (outputs, 96), device="cuda").to(torch.int8)
    ws, b = torch.rand(outputs, device="cuda"), torch.randn(outputs, device="cuda")
    clean = clear.int8_linear(x, w, ws, b)
    x[1, 5], x[3, 95] = math.nan, math.inf
    x[2] = 0.0
    got = clear.int8_linear(x, w, ws, b)
    assert bool(torch.isnan(got[[1, 3]]).all()) and torch.equal(got[2], b)
    assert torch.equal(got[4:], clean[4:]) and torch.equal(got[0], clean[0])


def test_a_table_of_its_own_rows():
    """quantize_rows' own output as a table: the product is near that of the numbers themselves."""
    from fhemamba_amd import clear

    gen = torch.Generator(device="cuda").manual_seed(7)
    x, w = (torch.randn(n, 512, generator=gen, device="cuda") for n in (40, 300))
    table = clear.quantize_rows(w)
    got, want = clear.int8_linear(x, table.values, table.scale), x.double() @ w.double().t()
    # each operand is off by up to half of max / 127: a uniform error of max / (127 sqrt(12)), max about 3.2 of unit
    # rows: 7e-3 of each, 1e-2 of both
    assert float((got - want).norm() / want.norm()) <= 1.5e-2


def test_refusals():
    from fhemamba_amd import clear

    x, w = torch.randn(3, 16, device="cuda"), torch.zeros(4, 16, dtype=torch.int8, device="cuda")
    ws = torch.ones(4, device="cuda")
    bad = [(lambda: clear.int8_linear(x.half(), w, ws), "float32 or bfloat16"),
           (lambda: clear.int8_linear(x, w.int(), ws), "type"),
           (lambda: clear.int8_linear(x, w[:, :8], ws), "shape"), (lambda: clear.int8_linear(x, w, ws[:2]), "shape"),
           (lambda: clear.int8_linear(x, w[0], ws), "outputs"), (lambda: clear.int8_linear(x, w, ws, ws[:2]), "shape"),
           (lambda: clear.int8_linear(x, w[:0], ws[:0]), "no outputs"),
           (lambda: clear.int8_linear(x, w, ws.double()), "type"),
           (lambda: clear.int8_linear(x.clone().requires_grad_(True), w, ws), "no gradient"),
           (lambda: clear.int8_linear(x, w, ws.clone().requires_grad_(True)), "no gradient"),
           (lambda: clear.int8_linear(x, w.cpu(), ws), "cpu"), (lambda: clear.quantize_rows(x.int()), "float32"),
           (lambda: clear.quantize_rows(x.clone().requires_grad_(True)), "no gradient"),
           (lambda: clear.quantize_rows(x.new_empty(1, 32769)), "32768"),
           (lambda: clear.int8_linear(x.new_empty(1, 32769), w.new_empty(1, 32769), ws[:1]), "32768"),
           (lambda: clear.quantize_rows(x[:, :0]), "channels")]
    for call, match in bad:
        with pytest.raises(ValueError, match=match):
            call()
