"""Wide bf16 products whose workgroups go through several tiles of 256 x 256, the next tile's loads under the stores of the
last: whole and ragged tiles, one and two results, weights as they lie and transposed, rows gathered by species.  Every row
holds random values, so that a tile that is read too early shows.  Compared in 64 bits on the GPU; tolerances: see
tests/_products.py."""

import pytest

from tests import _products as plain
from tests._util import flush

pytestmark = pytest.mark.gpu

UNITS, TILE = 256, 256  # compute units, rows and columns of a tile


def tiles(rows, columns, species=0):
    return (-(-rows // TILE) + species) * -(-columns // TILE)


def normal(shape, seed, gpu, sd=1.0):
    import torch

    return (torch.randn(shape, generator=torch.Generator(device=gpu).manual_seed(seed), device=gpu) * sd).bfloat16()


def weight_of(shape, seed, gpu, turned):
    if turned:
        return normal((*shape[:-2], shape[-1], shape[-2]), seed, gpu, shape[-2] ** -0.5).transpose(-1, -2)
    return normal(shape, seed, gpu, shape[-2] ** -0.5)


def check(name, got, want, rounded, wide):
    """As in tests/_products.py: 2e-5 of what float32 sums up and 2^-8 of what is rounded to bfloat16."""
    import torch

    assert got.shape == want.shape and bool(torch.isfinite(got).all()), name
    worst = float(((got.double() - want).abs() / (plain.FLOAT32 * wide + plain.BFLOAT16 * rounded + 1e-37)).max())
    print(f"  {name}: error {worst:.3f} of what is allowed", flush=True)
    assert worst <= 1.0, f"{name}: {worst:.3f} times what is allowed"


def members(species, count, rows, gpu):
    import torch

    if species is None:
        return [torch.arange(rows, device=gpu)]
    return [torch.nonzero(species == k)[:, 0] for k in range(count)]


def product(x, w, rows):
    """Sums and the sums of magnitudes of x times each weight, rows of no weight zero."""
    import torch

    out = [torch.zeros(x.shape[0], w.shape[-1], dtype=torch.float64, device=x.device) for _ in range(2)]
    for k, of in enumerate(rows):
        out[0][of] = torch.mm(x[of].double(), w[k].double())
        out[1][of] = torch.mm(x[of].double().abs(), w[k].double().abs())
    return out


# 25 000 rows are 97 whole rows of tiles and one of 168
CASES = [(25000, 1024, 1024, 0), (25000, 1024, 1032, 0), (25000, 1032, 1024, 0), (25088, 1024, 1024, 0), (25000, 1024, 1024, 3),
         (25000, 1024, 1032, 4), (50000, 2048, 512, 5)]


@pytest.mark.parametrize("activation,dropout,residual", [(None, 0.0, False), (None, 0.2, True), ("silu", 0.0, False),
                                                         ("gelu", 0.2, True)])
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("rows,inputs,outputs,species", CASES)
def test_forward(gpu, rows, inputs, outputs, species, turned, activation, dropout, residual):
    import torch

    from ye3t_amd import runtime
    from ye3t_amd.runtime import native

    assert tiles(rows, outputs) > UNITS  # some workgroups have several tiles
    flush(f"{rows} x {inputs} x {outputs} by {species} species, turned {turned}, {activation}, dropout {dropout}")
    x, b = normal((rows, inputs), 1, gpu), normal((max(species, 1), outputs), 3, gpu)
    w = weight_of((max(species, 1), inputs, outputs), 2, gpu, turned)
    r = normal((rows, outputs), 4, gpu) if residual else None
    s, groups, forward = None, (), runtime.linear
    if species:  # some atoms of no species
        s = torch.randint(species + 1, (rows,), generator=torch.Generator().manual_seed(5)).to(gpu)
        groups, forward = (runtime.species_groups(s, species, validate=False),), runtime.species_linear
    shape = dict(activation=activation, dropout=dropout, seed=9 if dropout else None, residual=r)
    parameters = (w, *groups, b) if species else (w[0], b[0])
    of = members(s, len(w), rows, gpu)
    z, wide = product(x, w, of)
    for k, at in enumerate(of):
        z[at] += b[k].double()
        wide[at] += b[k].double().abs()
    y = plain.activated(activation, z)
    if s is not None:
        y[s >= species] = 0.0
    far = 1.13 * wide + y.abs()
    if dropout:
        keep = plain.kept(rows, outputs, dropout, 9, 0).to(gpu)
        y, far = y * keep, far * keep
    if residual:
        y, far = y + r.double(), far + r.double().abs()
    alone = forward(x, *parameters, **shape)
    assert native.last_kernel() == "row_product_rounds_kernel"
    check("out", alone, y, y.abs(), far)
    out, kept = forward(x, *parameters, return_preactivation=True, **shape)
    assert native.last_kernel() == "row_product_rounds_kernel"
    assert torch.equal(out, alone)
    check("preactivation", kept, z, z.abs(), wide)


@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("rows,inputs,outputs,species", [(25000, 1024, 1024, 0), (25000, 1032, 1024, 0), (25000, 1024, 1024, 4)])
def test_gradient_of_rows(gpu, rows, inputs, outputs, species, turned):
    import torch

    from ye3t_amd import runtime
    from ye3t_amd.runtime import native

    assert tiles(rows, inputs) > UNITS
    flush(f"gradients of {rows} x {inputs} x {outputs} by {species} species, turned {turned}")
    x, g = normal((rows, inputs), 1, gpu), normal((rows, outputs), 3, gpu)
    w = weight_of((max(species, 1), inputs, outputs), 2, gpu, turned)
    s = torch.randint(species, (rows,), generator=torch.Generator().manual_seed(5)).to(gpu) if species else None
    groups = runtime.species_groups(s, species) if species else (None, None)
    problem = native.Linear(x, w if species else w[0], None, None, *groups, 0, 0, 0, 0)
    got, _, _ = problem.adjoint(g, None, True, False, False)
    assert native.last_kernel() == "row_product_rounds_kernel"
    dx, wide = product(g, w.transpose(-1, -2).contiguous(), members(s, len(w), rows, gpu))
    check("input", got, dx, dx.abs(), wide)
