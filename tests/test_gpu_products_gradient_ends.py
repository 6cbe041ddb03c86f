"""Gradients of the products with learned weights at the ends of what an epilogue does: values that are dropped, units that
are dead, preactivations and adjoints that are not finite.  Tolerances: see tests/_products.py."""

import pytest

from tests import _products as plain
from tests._util import flush

pytestmark = pytest.mark.gpu

TYPES = ["float32", "bfloat16"]


def normal(shape, dtype, seed, gpu, sd=1.0):
    import torch

    t = torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * sd
    return t.to(getattr(torch, dtype)).to(gpu)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", ["relu", "silu", "gelu"])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("rows,inputs,outputs", [(40, 24, 50), (5, 1030, 9), (700, 72, 264)])
def test_dropped_values_have_no_gradient_whatever_they_hold(gpu, dtype, activation, value, rows, inputs, outputs):
    """Preactivations that are not finite at dropped places: the output does not depend on them, nor do the gradients."""
    import torch

    from ye3t_amd import runtime

    flush(f"dropped preactivations of {value}, {activation}, {rows} x {inputs} x {outputs}, {dtype}")
    x, w = normal((rows, inputs), dtype, 1, gpu), normal((inputs, outputs), dtype, 2, gpu, inputs ** -0.5)
    g = normal((rows, outputs), dtype, 3, gpu)
    kw = dict(activation=activation, dropout=0.4, seed=21, layer=5)
    keep = plain.kept(rows, outputs, 0.4, 21, 5)
    z = runtime.linear(x, w, return_preactivation=True)[1]
    z[(keep == 0).to(gpu)] = value
    clean = torch.where((keep == 0).to(gpu), torch.zeros_like(z), z)
    got = dict(zip(("input", "weight", "bias"), runtime.linear_adjoint(g, x, w, preactivation=z, bias=True, **kw)))
    want = plain.backward(g, x, w, clean, None, activation, keep)
    for n, t in got.items():
        plain.check(n, t, want[n], dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_dropped_values_through_autograd(gpu, dtype):
    """An infinite bias column: finite wherever it is dropped, and so is the gradient of those rows."""
    import torch

    from ye3t_amd import runtime

    x, w = normal((60, 24), dtype, 1, gpu).requires_grad_(), normal((24, 16), dtype, 2, gpu, 0.2)
    b = torch.zeros(16, dtype=x.dtype, device=gpu)
    b[3] = float("inf")
    y = runtime.linear(x, w, b, activation="silu", dropout=0.5, seed=4)
    gone = plain.kept(60, 16, 0.5, 4, 0)[:, 3] == 0
    assert torch.equal(torch.isfinite(y).all(1).cpu(), gone) and gone.any()
    y[gone.to(gpu)].sum().backward()
    assert torch.isfinite(x.grad[gone.to(gpu)]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dropout", [0.0, 0.25])
def test_relu_passes_or_stops(gpu, dtype, dropout):
    """relu's gradient is the adjoint where relu gave the preactivation, NaN among them, and zero where it gave zero, whatever
    the adjoint holds."""
    import torch

    from ye3t_amd import runtime

    flush(f"relu, dropout {dropout}, {dtype}")
    inf, nan = float("inf"), float("nan")
    z = torch.tensor([-inf, -1.0, -0.0, 0.0, 1e-30, 2.0, inf, nan], device=gpu).to(getattr(torch, dtype)).repeat(5, 1)
    g = torch.tensor([1.0, inf, -inf, nan, 3.0], device=gpu).to(z.dtype)[:, None].expand(5, 8).contiguous()
    # the gradient of the input is dz itself: a weight of one column for each
    x, w = torch.zeros(5, 8, dtype=z.dtype, device=gpu), torch.eye(8, dtype=z.dtype, device=gpu)
    passed = torch.where(z <= 0, torch.zeros_like(g), g)
    for k in range(8):  # a column alone: zero times infinity in the others' products is no number
        dx, _, db = runtime.linear_adjoint(g[:, k:k + 1].contiguous(), x, w[:, k:k + 1], preactivation=z[:, k:k + 1].contiguous(),
                                           bias=True, activation="relu", dropout=dropout, seed=3 if dropout else None)
        mask = plain.kept(5, 1, dropout, 3, 0).to(gpu) if dropout else torch.ones(5, 1, device=gpu)
        one = torch.where(mask == 0, torch.zeros_like(g[:, :1]), (passed[:, k:k + 1].float() * mask).to(z.dtype))
        assert torch.equal(torch.isnan(dx[:, k:k + 1]), torch.isnan(one))
        there = ~torch.isnan(one)
        assert torch.equal(dx[:, k:k + 1][there], one[there])
        total = one.double().sum(0)
        assert torch.isnan(db.double()).equal(torch.isnan(total)) and (torch.isnan(total).any() or torch.equal(db.double(), total))


def bias_check(got, dz, size, species, count):
    """One rounding, 2^-8 of the result, and float32 sums, 2e-5 of their terms."""
    import torch

    rows = plain.members(species, count, len(dz))
    want, wide = (torch.stack([t[r].sum(0) for r in rows]).reshape(got.shape) for t in (dz, size))
    assert torch.isfinite(got).all()
    worst = float(((plain.d(got) - want).abs() / (plain.BFLOAT16 * want.abs() + plain.FLOAT32 * wide + 1e-37)).max())
    flush(f"  bias: error {worst:.3f} of what is allowed")
    assert worst <= 1.0


@pytest.mark.parametrize("species", [None, 1, 7, 300])
@pytest.mark.parametrize("rows,outputs", [(1, 1), (40, 9), (255, 16), (257, 17), (700, 65), (3001, 130), (5000, 1), (70000, 40),
                                          (9000, 1032)])
def test_bias_gradients_are_sums_of_what_is_not_rounded(gpu, rows, outputs, species):
    """bfloat16 rounds dz for the matrix instructions of the other two gradients; the bias's has one rounding, its own.  Of
    values of 65536 / 65280 = 1 + 0.0039, which all round to 1 + 0.0078, sums would be off by 2^-8 before it."""
    import torch

    from ye3t_amd import runtime

    flush(f"bias gradients of {rows} x {outputs} by {species} species")
    lead = () if species is None else (species,)
    s, groups, adjoint = None, (), runtime.linear_adjoint
    if species is not None:
        s = torch.randint(species, (rows,), generator=torch.Generator().manual_seed(3)) // 2 * 2  # some have no atoms
        groups, adjoint = (runtime.species_groups(s.to(gpu), species),), runtime.species_linear_adjoint
    x, w = normal((rows, 8), "bfloat16", 1, gpu), normal((*lead, 8, outputs), "bfloat16", 2, gpu)
    one = torch.ones(rows, outputs, dtype=x.dtype, device=gpu)
    drop = 256 / 65536
    keep = plain.kept(rows, outputs, drop, 6, 2)
    _, _, db = adjoint(one, x, w, *groups, bias=True, dropout=drop, seed=6, layer=2)
    bias_check(db, keep, keep, s, species)
    g, z = normal((rows, outputs), "bfloat16", 4, gpu), normal((rows, outputs), "bfloat16", 5, gpu, 2.0)
    for activation in ("relu", "silu", "gelu"):
        _, _, db = adjoint(g, x, w, *groups, preactivation=z, bias=True, activation=activation, dropout=drop, seed=6, layer=2)
        dz = plain.d(g) * plain.slope(activation, plain.d(z)) * keep
        size = plain.d(g).abs() * plain.slope_size(activation, plain.d(z)) * keep
        bias_check(db, dz, size, s, species)
        _, _, again = adjoint(g, x, w, *groups, preactivation=z, bias=True, activation=activation, dropout=drop, seed=6, layer=2)
        assert torch.equal(db, again)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [30, 900, 26000])
def test_atoms_of_no_species_behind_an_activation(gpu, dtype, rows):
    """Their rows reach no gradient, whatever they or the memory that the call takes for itself held."""
    import torch

    from ye3t_amd import runtime

    flush(f"{rows} atoms, some of no species, {dtype}")
    s = torch.randint(5, (rows,), generator=torch.Generator().manual_seed(2))
    s[::7] = -1
    none = (s < 0) | (s > 3)
    x, w = normal((rows, 24), dtype, 1, gpu), normal((4, 24, 40), dtype, 2, gpu, 0.2)
    g, z = normal((rows, 40), dtype, 3, gpu), normal((rows, 40), dtype, 4, gpu)
    clean = [torch.where(none[:, None].to(gpu), torch.zeros_like(t), t) for t in (x, g, z)]
    for t in (x, g, z):
        t[none.to(gpu)] = float("nan")
    groups = runtime.species_groups(s.to(gpu), 4, validate=False)
    kw = dict(activation="silu", dropout=0.3, seed=8, layer=1)
    for _ in range(2):
        held = torch.full((1 << 24,), float("nan"), device=gpu)
        del held
        got = dict(zip(("input", "weight", "bias"), runtime.species_linear_adjoint(g, x, w, groups, preactivation=z, bias=True, **kw)))
        want = plain.backward(clean[1], clean[0], w, clean[2], s, "silu", plain.kept(rows, 40, 0.3, 8, 1))
        for n, t in got.items():
            plain.check(n, t, want[n], dtype)
        assert not got["input"][none.to(gpu)].any()
