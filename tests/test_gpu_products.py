"""Products with learned weights, by species too, and dropout against plain forms in 64 bits.  Tolerances: see
tests/_products.py."""

import pytest

from tests import _products as plain
from tests._util import flush

pytestmark = pytest.mark.gpu

TYPES = ["float32", "bfloat16"]
# rows, inputs, outputs: one of each, ends of tiles, odd sizes, long and short contractions
SIZES = [(1, 1, 1), (1, 256, 512), (2, 7, 9), (5, 1030, 40), (31, 33, 65), (33, 161, 96), (64, 64, 64), (65, 8, 130),
         (130, 515, 257), (300, 16, 1), (1000, 1, 33), (700, 96, 161), (4097, 72, 40), (2050, 264, 520), (9000, 129, 700)]


def normal(shape, dtype, seed, gpu, sd=1.0):
    import torch

    t = torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * sd
    return t.to(getattr(torch, dtype)).to(gpu)


def weights(shape, dtype, seed, gpu, turned):
    if turned:
        return normal((*shape[:-2], shape[-1], shape[-2]), dtype, seed, gpu, shape[-2] ** -0.5).transpose(-1, -2)
    return normal(shape, dtype, seed, gpu, shape[-2] ** -0.5)


def run(x, w, b, r, g, species=None, activation=None, dropout=0.0, seed=None, layer=0):
    """{name: tensor} of the forward and its gradients through the functions themselves."""
    from ye3t_amd import runtime

    kw = dict(activation=activation, dropout=dropout, seed=seed, layer=layer)
    groups, forward, backward = (), runtime.linear, runtime.linear_adjoint
    if species is not None:
        groups = (runtime.species_groups(species, len(w)),)
        forward, backward = runtime.species_linear, runtime.species_linear_adjoint
    y, z = forward(x, w, *groups, b, residual=r, return_preactivation=True, **kw)
    dx, dw, db = backward(g, x, w, *groups, preactivation=None if activation is None else z, bias=b is not None, **kw)
    return {"out": y, "preactivation": z, "input": dx, "weight": dw, "bias": db}


def compare(got, x, w, b, r, g, dtype, species=None, activation=None, keep=None):
    want = plain.forward(x, w, b, r, species, activation, keep)
    want |= plain.backward(g, x, w, got["preactivation"], species, activation, keep)
    for n, t in got.items():
        if t is not None:
            plain.check(n, t, want[n], dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("rows,inputs,outputs", SIZES)
def test_linear(gpu, dtype, turned, rows, inputs, outputs):
    flush(f"linear {rows} x {inputs} x {outputs}, turned {turned}, {dtype}")
    x, w = normal((rows, inputs), dtype, 1, gpu), weights((inputs, outputs), dtype, 2, gpu, turned)
    b, g = normal((outputs,), dtype, 3, gpu), normal((rows, outputs), dtype, 4, gpu)
    compare(run(x, w, b, None, g), x, w, b, None, g, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("dropout", [0.0, 0.3])
@pytest.mark.parametrize("bias,residual", [(False, False), (True, True)])
@pytest.mark.parametrize("rows,inputs,outputs", [(3, 40, 21), (70, 33, 130), (600, 24, 64)])
def test_epilogue(gpu, dtype, activation, dropout, bias, residual, rows, inputs, outputs):
    flush(f"linear {rows} x {inputs} x {outputs}, {activation}, dropout {dropout}, {bias}, {dtype}")
    x, w = normal((rows, inputs), dtype, 1, gpu, 1.5), weights((inputs, outputs), dtype, 2, gpu, False)
    b = normal((outputs,), dtype, 3, gpu) if bias else None
    r = normal((rows, outputs), dtype, 5, gpu, 2.0) if residual else None
    g = normal((rows, outputs), dtype, 4, gpu)
    got = run(x, w, b, r, g, None, activation, dropout, 2 ** 63 + 12345, 7)
    keep = plain.kept(rows, outputs, dropout, 2 ** 63 + 12345, 7) if dropout else None
    compare(got, x, w, b, r, g, dtype, None, activation, keep)


def species_of(rows, count, kind, gpu):
    import torch

    g = torch.Generator().manual_seed(11)
    if kind == "one":
        return torch.full((rows,), count - 1, dtype=torch.int32, device=gpu)
    s = torch.randint(count, (rows,), generator=g, dtype=torch.int64)
    if kind == "rare":  # most atoms of one species, some species missing
        s = torch.where(torch.rand(rows, generator=g) < 0.8, 0, s // 2 * 2)
    return s.to(torch.int32 if kind == "rare" else torch.int64).to(gpu)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("kind", ["any", "rare", "one"])
@pytest.mark.parametrize("rows,species,inputs,outputs", [(1, 1, 5, 3), (21, 4, 128, 128), (40, 7, 33, 65), (300, 89, 16, 40),
                                                         (900, 3, 130, 200), (5000, 300, 24, 17), (8200, 5, 70, 161)])
def test_species_linear(gpu, dtype, turned, kind, rows, species, inputs, outputs):
    flush(f"linear by {species} species ({kind}) {rows} x {inputs} x {outputs}, turned {turned}, {dtype}")
    s = species_of(rows, species, kind, gpu)
    x, w = normal((rows, inputs), dtype, 1, gpu), weights((species, inputs, outputs), dtype, 2, gpu, turned)
    b, r = normal((species, outputs), dtype, 3, gpu), normal((rows, outputs), dtype, 5, gpu)
    g = normal((rows, outputs), dtype, 4, gpu)
    got = run(x, w, b, r, g, s, "silu", 0.1, 99, 1)
    compare(got, x, w, b, r, g, dtype, s, "silu", plain.kept(rows, outputs, 0.1, 99, 1))


@pytest.mark.parametrize("rows", [0, 1, 63, 64, 4096, 4097, 30011])
@pytest.mark.parametrize("species", [1, 4, 255, 256, 70000])
def test_species_groups(gpu, rows, species):
    import torch

    from ye3t_amd import runtime

    flush(f"groups of {rows} atoms of {species} species")
    for dtype in (torch.int32, torch.int64):
        s = torch.randint(species, (rows,), generator=torch.Generator().manual_seed(rows), dtype=dtype).to(gpu)
        groups = runtime.species_groups(s, species)
        assert torch.equal(groups.order.long(), torch.argsort(s, stable=True))
        counts = torch.bincount(s.long(), minlength=species)
        assert torch.equal(groups.offsets, torch.cat([counts.new_zeros(1), counts.cumsum(0)]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [30, 900])
def test_atoms_of_no_species(gpu, dtype, rows):
    """Unchecked species outside the table: the product and the gradient are zero, the residual stays."""
    import torch

    from ye3t_amd import runtime

    flush(f"{rows} atoms, some of no species, {dtype}")
    s = species_of(rows, 4, "any", gpu)
    s[::5] = 4
    s[1::7] = -3
    with pytest.raises(RuntimeError, match="out of range"):
        runtime.species_groups(s, 4)
    x, w = normal((rows, 20), dtype, 1, gpu), normal((4, 20, 36), dtype, 2, gpu, 0.2)
    x[::5] = float("nan")
    b, r, g = normal((4, 36), dtype, 3, gpu), normal((rows, 36), dtype, 4, gpu), normal((rows, 36), dtype, 5, gpu)
    groups = runtime.species_groups(s, 4, validate=False)
    none = (s < 0) | (s > 3)
    y = runtime.species_linear(x, w, groups, b, residual=r)
    assert torch.equal(y[none], r[none])
    dx, dw, db = runtime.species_linear_adjoint(g, x, w, groups, bias=True)
    assert not dx[none].any() and torch.isfinite(dw).all() and torch.isfinite(db).all()
    clean = torch.where(none[:, None], torch.zeros_like(x), x)
    want = plain.forward(clean, w, b, r, s) | plain.backward(g, clean, w, None, s)
    for n, t in (("out", y), ("input", dx), ("weight", dw), ("bias", db)):
        plain.check(n, t, want[n], dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (64, 256), (1000, 161), (70001, 9), (5, 4096)])
@pytest.mark.parametrize("probability", [0.0, 0.1, 0.5, 1.0])
def test_dropout(gpu, dtype, residual, rows, width, probability):
    from ye3t_amd import runtime

    flush(f"dropout {rows} x {width}, {probability}, {dtype}")
    x = normal((rows, width), dtype, 1, gpu)
    r = normal((rows, width), dtype, 2, gpu) if residual else None
    for seed, layer in ((5, 0), (-1, 2 ** 32 - 1)):
        keep = plain.kept(rows, width, probability, seed, layer)
        y = runtime.dropout(x, probability, seed, layer=layer, residual=r)
        want = plain.d(x) * keep + (0 if r is None else plain.d(r))
        plain.check("out", y, (want, want.abs(), (plain.d(x) * keep).abs() + want.abs()), dtype)
        dx = runtime.dropout_adjoint(x, probability, seed, layer=layer)
        want = plain.d(x) * keep
        plain.check("input", dx, (want, want.abs(), want.abs()), dtype)
        assert bool(((dx == 0).cpu() == ((keep == 0) | (x == 0).cpu())).all())


def test_masks_of_products_and_dropout_are_one(gpu):
    """The epilogue drops what the function drops, in the rows' own places."""
    import torch

    from ye3t_amd import runtime

    x, w = normal((200, 24), "float32", 1, gpu), normal((24, 51), "float32", 2, gpu)
    whole = runtime.linear(x, w)
    for y in (runtime.linear(x, w, dropout=0.4, seed=8, layer=3),
              runtime.species_linear(x, w[None], runtime.species_groups(torch.zeros(200, dtype=torch.int32, device=gpu), 1),
                                     dropout=0.4, seed=8, layer=3)):
        assert torch.equal(y, runtime.dropout(whole, 0.4, 8, layer=3))
    other = runtime.dropout(whole, 0.4, 8, layer=4)
    assert not torch.equal(other, y)
