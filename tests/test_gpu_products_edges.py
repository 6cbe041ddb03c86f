"""Products with learned weights and dropout where they can go wrong: every kernel's ends of tiles, values that are not
finite, strides and alignment, empty sizes, graphs, streams, seeds in memory, and arrays of more than 2^31 values.
Tolerances: see tests/_products.py."""

import pytest

from tests import _products as plain
from tests._util import flush
from tests.test_gpu_products import TYPES, compare, normal, run, species_of, weights

pytestmark = pytest.mark.gpu


# ---- every kernel ------------------------------------------------------------------

# tiles of 256 x 256 and 128 x 128 of direct loads, 128 x 128, 128 x 64, 64 x 64, and 32 x 32 with the contraction in
# parts; rows, columns and contractions that end inside a tile; chunks that are whole and aligned, and not
KERNELS = [(12300, 1032, 1032), (5003, 264, 1000), (5003, 300, 1001), (70001, 40, 96), (9001, 31, 65), (5, 4096, 40),
           (37, 2050, 100), (2500, 1544, 520)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("rows,inputs,outputs", KERNELS)
def test_kernels(gpu, dtype, turned, rows, inputs, outputs):
    flush(f"linear {rows} x {inputs} x {outputs}, turned {turned}, {dtype}")
    x, w = normal((rows, inputs), dtype, 1, gpu), weights((inputs, outputs), dtype, 2, gpu, turned)
    b, r, g = normal((outputs,), dtype, 3, gpu), normal((rows, outputs), dtype, 5, gpu), normal((rows, outputs), dtype, 4, gpu)
    got = run(x, w, b, r, g, None, "gelu", 0.2, 17, 2)
    compare(got, x, w, b, r, g, dtype, None, "gelu", plain.kept(rows, outputs, 0.2, 17, 2))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("kind", ["any", "rare"])
@pytest.mark.parametrize("rows,species,inputs,outputs", [(12300, 3, 1032, 1032), (5003, 4, 264, 1000), (37, 5, 2050, 100)])
def test_kernels_by_species(gpu, dtype, turned, kind, rows, species, inputs, outputs):
    flush(f"linear by {species} species ({kind}) {rows} x {inputs} x {outputs}, turned {turned}, {dtype}")
    s = species_of(rows, species, kind, gpu)
    x, w = normal((rows, inputs), dtype, 1, gpu), weights((species, inputs, outputs), dtype, 2, gpu, turned)
    b, g = normal((species, outputs), dtype, 3, gpu), normal((rows, outputs), dtype, 4, gpu)
    compare(run(x, w, b, None, g, s), x, w, b, None, g, dtype, s)


def test_equal_calls_give_equal_bits(gpu):
    import torch

    flush("equal calls")
    for dtype in TYPES:
        s = species_of(7000, 6, "rare", gpu)
        x, w, g = normal((7000, 136), dtype, 1, gpu), normal((6, 136, 264), dtype, 2, gpu, 0.1), normal((7000, 264), dtype, 4, gpu)
        b = normal((6, 264), dtype, 3, gpu)
        first = run(x, w, b, None, g, s, "silu", 0.1, 5)
        again = run(x, w, b, None, g, s, "silu", 0.1, 5)
        assert all(torch.equal(t, again[n]) for n, t in first.items())


# ---- values --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inputs,outputs", [(5, 4096, 40), (20, 33, 70), (300, 40, 130), (5003, 264, 1000)])
def test_values_that_are_not_finite(gpu, dtype, rows, inputs, outputs):
    """Infinities and NaN reach what a sum of products says, no other rows or columns; the largest numbers stay numbers."""
    import torch

    from ye3t_amd import runtime

    flush(f"values that are not finite, {rows} x {inputs} x {outputs}, {dtype}")
    x, w = normal((rows, inputs), dtype, 1, gpu), normal((inputs, outputs), dtype, 2, gpu)
    largest = torch.finfo(x.dtype).max
    x[1, 3], x[2, 5], x[3, 7], w[9, 4] = float("inf"), float("nan"), -float("inf"), float("inf")
    x[4, :], x[4, 11] = 0.0, largest
    w[11], w[11, 6] = 0.25, 0.0
    y = plain.d(runtime.linear(x, w))
    want = plain.d(x) @ plain.d(w)
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    endless = torch.isinf(want)
    assert torch.equal(y[endless], want[endless]) and not torch.isinf(y[~endless]).any()
    # the row of one largest number, but for the column of the weight that is infinite (0 x infinity)
    columns = [c for c in range(outputs) if c != 4]
    assert torch.allclose(y[4, columns], want[4, columns], rtol=2.0 ** -8 if dtype == "bfloat16" else 2e-6, atol=0.0)
    g = normal((rows, outputs), dtype, 3, gpu)
    g[1, 2], g[3, 8] = float("inf"), float("nan")
    clean = torch.where(torch.isfinite(w), w, torch.zeros_like(w))
    dx, dw, db = runtime.linear_adjoint(g, x, clean, bias=True)
    for got, exact in ((dx, plain.d(g) @ plain.d(clean).T), (dw, plain.d(x).T @ plain.d(g)), (db, plain.d(g).sum(0))):
        got = plain.d(got)
        assert torch.equal(torch.isnan(got), torch.isnan(exact))
        # sums of the largest number and others may pass it or not
        endless = torch.isinf(exact) & (exact.abs() > largest)
        assert torch.equal(got[endless], exact[endless])


def test_small_values(gpu):
    """float32 keeps its digits down to 2^-100; products of smaller ones are off by the last bits of three parts, 2^-133 of the other
    factor at most (16 x 2^-133 x 30 here)."""
    from ye3t_amd import runtime

    flush("small values")
    x, w = normal((70, 16), "float32", 1, gpu), normal((16, 70), "float32", 2, gpu)
    for power in (-60, -100):
        y = runtime.linear(x * 2.0 ** power, w)
        want = plain.d(x * 2.0 ** power) @ plain.d(w)
        plain.check("out", y * 2.0 ** -power, (want * 2.0 ** -power, want, (plain.d(x).abs() @ plain.d(w).abs())), "float32")
    y = runtime.linear(x * 2.0 ** -124, w)
    want = plain.d(x * 2.0 ** -124) @ plain.d(w)
    assert float((plain.d(y) - want).abs().max()) <= 16 * 30 * 2.0 ** -133


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", ["relu", "silu", "gelu"])
def test_activations_far_out(gpu, dtype, activation):
    """Large preactivations: no overflow on the way, slopes of 0 and 1."""
    import torch

    from ye3t_amd import runtime

    z = torch.tensor([[-1e30, -1e4, -200.0, -88.0, -30.0, -1e-30, 0.0, 1e-30, 30.0, 88.0, 200.0, 1e4, 1e30]], device=gpu)
    z = z.to(getattr(torch, dtype))
    one = torch.ones(1, 1, dtype=z.dtype, device=gpu)
    # through the bias: an input of zero
    y, kept = runtime.linear(one * 0, one.expand(1, z.shape[1]).contiguous(), z[0], activation=activation, return_preactivation=True)
    assert torch.equal(kept, z)
    want = plain.activated(activation, plain.d(z))
    # exponents of up to 200: 200 x 2^-24 of the tails
    assert torch.allclose(plain.d(y), want, rtol=2.0 ** -8 if dtype == "bfloat16" else 3e-5, atol=1e-37)
    _, _, db = runtime.linear_adjoint(torch.ones_like(y), one * 0, one.expand(1, z.shape[1]).contiguous(), preactivation=kept,
                                      activation=activation, bias=True)
    want = plain.slope(activation, plain.d(z)).nan_to_num(0.0)[0]
    size = plain.slope_size(activation, plain.d(z)).nan_to_num(0.0)[0]
    assert bool(((plain.d(db) - want).abs() <= (2.0 ** -8 if dtype == "bfloat16" else 0.0) * want.abs() + 3e-5 * size + 1e-37).all())


def test_dropped_values_are_zero_whatever_they_hold(gpu):
    import torch

    from ye3t_amd import runtime

    x = torch.full((40, 50), float("nan"), device=gpu)
    gone = plain.kept(40, 50, 0.5, 3, 0) == 0
    y = runtime.dropout(x, 0.5, 3)
    assert not y.cpu()[gone].any() and torch.isnan(y.cpu()[~gone]).all()
    assert torch.equal(runtime.dropout(x, 1.0, 3), torch.zeros_like(x))


# ---- layouts ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
def test_strides(gpu, dtype):
    import torch

    from ye3t_amd import runtime

    flush(f"strides, {dtype}")
    rows, a, b = 700, 264, 136
    wide = normal((rows, 2 * a + 5), dtype, 1, gpu)
    weight = normal((2 * a, 2 * b), dtype, 2, gpu, a ** -0.5)
    bias, residual = normal((2 * b,), dtype, 3, gpu), normal((1, b), dtype, 4, gpu)
    g = normal((rows, 2 * b), dtype, 5, gpu)
    for x in (wide[:, 3:3 + a], wide[:, 8:8 + a], wide[:, :2 * a:2], wide[:1, :a].expand(rows, a)):
        for w in (weight[::2, ::2], weight[:a, 1:1 + b], weight[5:5 + a, 8:8 + b], weight.t()[1:1 + b, 7:7 + a].t()):
            y, z = runtime.linear(x, w, bias[::2], residual=residual.expand(rows, b), return_preactivation=True)
            want = plain.forward(x, w, bias[::2], residual.expand(rows, b))
            plain.check("out", y, want["out"], dtype)
            got = dict(zip(("input", "weight", "bias"), runtime.linear_adjoint(g[:, ::2], x, w, bias=True)))
            want = plain.backward(g[:, ::2], x, w, z)
            for n, t in got.items():
                plain.check(n, t, want[n], dtype)
    # one weight for all species, as a view
    s = species_of(rows, 3, "any", gpu)
    groups = runtime.species_groups(s, 3)
    x, w = wide[:, 3:3 + a], weight[:a, 8:8 + b]
    y = runtime.species_linear(x, w.expand(3, a, b), groups)
    plain.check("out", y, plain.forward(x, w, None, None)["out"], dtype)
    # every other species of a larger table
    table = normal((6, a, b), dtype, 7, gpu, a ** -0.5)
    y = runtime.species_linear(x, table[::2], groups)
    plain.check("out", y, plain.forward(x, table[::2], None, None, s)["out"], dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_more_axes(gpu, dtype):
    import torch

    from ye3t_amd import runtime

    x, w, r = normal((3, 5, 7, 24), dtype, 1, gpu), normal((24, 40), dtype, 2, gpu), normal((3, 5, 7, 40), dtype, 3, gpu)
    y, z = runtime.linear(x, w, activation="relu", residual=r, dropout=0.3, seed=1, return_preactivation=True)
    flat = runtime.linear(x.reshape(105, 24), w, activation="relu", residual=r.reshape(105, 40), dropout=0.3, seed=1)
    assert y.shape == z.shape == r.shape and torch.equal(y.reshape(105, 40), flat)
    dx, dw, db = runtime.linear_adjoint(r, x, w, preactivation=z, activation="relu", dropout=0.3, seed=1)
    assert dx.shape == x.shape and dw.shape == w.shape and db is None
    groups = runtime.species_groups(species_of(105, 2, "any", gpu), 2)
    assert runtime.species_linear(x, w.expand(2, 24, 40), groups).shape == r.shape
    one = runtime.linear(x[0, 0, 0], w)
    assert one.shape == (40,)
    assert runtime.dropout(x[0, 0, 0], 0.3, 1).shape == (24,) and runtime.dropout(x, 0.3, 1).shape == x.shape


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inputs,outputs,species", [(0, 8, 6, None), (5, 0, 6, None), (5, 8, 0, None), (0, 0, 0, None),
                                                         (0, 8, 6, 3), (5, 0, 6, 3), (5, 8, 0, 3), (0, 8, 6, 0)])
def test_empty_sizes(gpu, dtype, rows, inputs, outputs, species):
    import torch

    from ye3t_amd import runtime

    flush(f"linear {rows} x {inputs} x {outputs} by {species} species, {dtype}")
    lead = () if species is None else (species,)
    s = None if species is None else torch.zeros(rows, dtype=torch.int32, device=gpu)
    x, w, b = (normal(n, dtype, 1, gpu) for n in ((rows, inputs), (*lead, inputs, outputs), (*lead, outputs)))
    g = normal((rows, outputs), dtype, 2, gpu)
    got = run(x, w, b, None, g, s, "silu")
    compare(got, x, w, b, None, g, dtype, s, "silu")
    leaves = [t.requires_grad_() for t in (x, w, b)]
    groups = () if species is None else (runtime.species_groups(s, species),)
    y = (runtime.linear if species is None else runtime.species_linear)(x, w, *groups, b, activation="silu")
    for t, grad in zip(leaves, torch.autograd.grad(y.sum(), leaves)):
        assert grad.shape == t.shape
    assert runtime.dropout(x.detach(), 0.5, 1).shape == x.shape


@pytest.mark.parametrize("dtype", TYPES)
def test_atoms_without_any_species(gpu, dtype):
    """No species at all, and atoms: products and gradients of zero."""
    import torch

    from ye3t_amd import runtime

    for rows in (5, 3000):
        x, w, b = normal((rows, 264), dtype, 1, gpu), normal((0, 264, 136), dtype, 2, gpu), normal((0, 136), dtype, 3, gpu)
        r, g = normal((rows, 136), dtype, 4, gpu), normal((rows, 136), dtype, 5, gpu)
        groups = runtime.species_groups(torch.zeros(rows, dtype=torch.int64, device=gpu), 0, validate=False)
        assert groups.offsets.tolist() == [0]
        y, z = runtime.species_linear(x, w, groups, b, activation="gelu", residual=r, return_preactivation=True)
        assert torch.equal(y, r) and not z.any()
        dx, dw, db = runtime.species_linear_adjoint(g, x, w, groups, preactivation=z, activation="gelu", bias=True)
        assert dx.shape == x.shape and not dx.any() and dw.shape == w.shape and db.shape == b.shape


# ---- autograd --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("by_species", [False, True])
@pytest.mark.parametrize("turned", [False, True])
def test_autograd_is_the_adjoint(gpu, dtype, by_species, turned):
    import torch

    from ye3t_amd import runtime

    flush(f"autograd, by species {by_species}, turned {turned}, {dtype}")
    s = species_of(150, 3, "any", gpu)
    groups = (runtime.species_groups(s, 3),) if by_species else ()
    lead = (3,) if by_species else ()
    x, w = normal((150, 24), dtype, 1, gpu), weights((*lead, 24, 40), dtype, 2, gpu, turned)
    b, r, g = normal((*lead, 40), dtype, 3, gpu), normal((150, 40), dtype, 4, gpu), normal((150, 40), dtype, 5, gpu)
    forward = runtime.species_linear if by_species else runtime.linear
    kw = dict(activation="gelu", dropout=0.25, seed=6, layer=9)
    leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
    y = forward(leaves[0], leaves[1], *groups, leaves[2], residual=leaves[3], **kw)
    grads = torch.autograd.grad(y, leaves, g)
    want = run(x, w, b, r, g, s if by_species else None, "gelu", 0.25, 6, 9)
    assert torch.equal(y, want["out"])
    for n, t in zip(("input", "weight", "bias"), grads):
        assert torch.equal(t, want[n]), n
    assert torch.equal(grads[3], g)
    # only some of them
    for k in range(3):
        some = [t.detach().requires_grad_(i == k) for i, t in enumerate((x, w, b))]
        y = forward(some[0], some[1], *groups, some[2], **kw)
        (grad,) = torch.autograd.grad(y, some[k], g)
        assert torch.equal(grad, want[("input", "weight", "bias")[k]])
    # a weight that is used twice
    w2 = w.detach().requires_grad_()
    both = forward(x, w2, *groups, b, **kw) + forward(x, w2, *groups, b, **kw)
    (grad,) = torch.autograd.grad(both, w2, g)
    assert torch.allclose(grad.float(), 2 * want["weight"].float(), rtol=2.0 ** -7 if dtype == "bfloat16" else 1e-6, atol=1e-6)
    # the preactivation has no gradient of its own
    y, z = forward(x.detach().requires_grad_(), w, *groups, b, return_preactivation=True, **kw)
    assert not z.requires_grad and torch.equal(z, want["preactivation"])
    # dropout by itself
    x3, r3 = (normal((150, 40), dtype, n, gpu).requires_grad_() for n in (7, 8))
    dx, dr = torch.autograd.grad(runtime.dropout(x3, 0.3, 2, residual=r3), (x3, r3), g)
    assert torch.equal(dx, runtime.dropout_adjoint(g, 0.3, 2)) and torch.equal(dr, g)


def test_gradients_against_differences(gpu):
    """The slope of the sum along random directions, float32.  Steps of 2^-6 leave third derivatives, 2^-12 / 6 of values of order
    one, and float32's rounding of sums of a few hundred values over the step, 300 x 2^-24 x 64: below 2e-3 of their size."""
    import torch

    from ye3t_amd import runtime

    flush("gradients against differences")
    s = species_of(60, 3, "any", gpu)
    groups = runtime.species_groups(s, 3)
    leaves = [normal(n, "float32", k, gpu, 0.4).requires_grad_() for k, n in enumerate(((60, 20), (3, 20, 30), (3, 30)))]
    g = normal((60, 30), "float32", 9, gpu)
    for activation in ("silu", "gelu", None):
        def value(x, w, b):
            return (runtime.species_linear(x, w, groups, b, activation=activation, dropout=0.2, seed=4).double() * g.double()).sum()

        grads = torch.autograd.grad(value(*leaves), leaves)
        for k in range(3):
            for seed in range(3):
                d = normal(leaves[k].shape, "float32", 20 + seed, gpu)
                moved = [[t.detach() + (step * d if i == k else 0) for i, t in enumerate(leaves)] for step in (2.0 ** -6, -2.0 ** -6)]
                slope = float(value(*moved[0]) - value(*moved[1])) * 32.0
                exact = float((grads[k].double() * d.double()).sum())
                size = float((grads[k].double() * d.double()).norm())
                assert abs(slope - exact) <= 2e-3 * (abs(exact) + 10 * size), (activation, k, slope, exact)


# ---- seeds -----------------------------------------------------------------------------

def test_seeds_in_memory(gpu):
    import torch

    from ye3t_amd import runtime

    x, w = normal((70, 24), "float32", 1, gpu), normal((24, 40), "float32", 2, gpu)
    for seed in (0, 5, 2 ** 63 - 1, -1, -2 ** 63):
        held = torch.tensor([seed], device=gpu)
        assert torch.equal(runtime.dropout(x, 0.5, held), runtime.dropout(x, 0.5, seed))
        assert torch.equal(runtime.dropout(x, 0.5, seed), runtime.dropout(x, 0.5, seed + 2 ** 64))
        assert torch.equal(runtime.linear(x, w, dropout=0.5, seed=held), runtime.linear(x, w, dropout=0.5, seed=seed))
    # a seed that has changed before the gradient is an error, not another mask
    held = torch.tensor([3], device=gpu)
    leaf = w.clone().requires_grad_()
    outs = (runtime.linear(x, leaf, dropout=0.5, seed=held), runtime.dropout(leaf, 0.5, held))
    held.add_(1)
    for y in outs:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_shares_of_dropped_values(gpu):
    """n values dropped with probability p: p n on average, standard deviation sqrt(n p (1 - p)); within five of it, in all
    columns, rows, layers and seeds alike."""
    import torch

    from ye3t_amd import runtime

    ones = torch.ones(4096, 512, device=gpu)
    for p in (0.1, 0.5):
        a = runtime.dropout(ones, p, 1) == 0
        for gone in (a, a[:, 3::8], a[7::64], a != (runtime.dropout(ones, p, 2) == 0), a != (runtime.dropout(ones, p, 1, layer=1) == 0)):
            q = p if gone is a or gone.shape != a.shape else 2 * p * (1 - p)
            n = gone.numel()
            assert abs(float(gone.sum()) - q * n) < 5 * (n * q * (1 - q)) ** 0.5


# ---- streams and graphs ------------------------------------------------------------------

def test_graphs(gpu):
    """Captured forward and gradient, replayed with other inputs, species and seeds, with eager work between."""
    import torch

    from ye3t_amd import runtime

    flush("captured products")
    for dtype in TYPES:
        seed = torch.tensor([1], device=gpu)
        s = species_of(600, 4, "any", gpu)
        x, w, b = normal((600, 136), dtype, 1, gpu), normal((4, 136, 264), dtype, 2, gpu, 0.1), normal((4, 264), dtype, 3, gpu)
        few, wide = normal((3, 4096), dtype, 6, gpu), normal((4096, 40), dtype, 7, gpu, 0.02)  # split over the contraction
        g = normal((600, 264), dtype, 4, gpu)
        kw = dict(activation="silu", dropout=0.2, seed=seed, layer=1)

        def step():
            groups = runtime.species_groups(s, 4, validate=False)
            y, z = runtime.species_linear(x, w, groups, b, return_preactivation=True, **kw)
            grads = runtime.species_linear_adjoint(g, x, w, groups, preactivation=z, bias=True, **kw)
            return [*groups, y, z, *grads, runtime.linear(few, wide), runtime.dropout(y, 0.5, seed)]

        step()
        torch.cuda.synchronize()
        graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        with torch.cuda.graph(other, pool=graph.pool()):
            step()
        for k in range(4):
            seed.fill_(10 + k)
            x.copy_(normal((600, 136), dtype, 30 + k, gpu))
            s.copy_(torch.randint(4, (600,), generator=torch.Generator().manual_seed(k), dtype=torch.int64))
            if k % 2:
                other.replay()  # shares the graph's workspaces, before it and not after
            graph.replay()
            got = [t.clone() for t in held]
            torch.cuda.synchronize()
            for a, c in zip(got, step()):
                assert torch.equal(a, c)


def test_streams(gpu):
    """Calls on two streams at once, each with workspaces of its own."""
    import torch

    from ye3t_amd import runtime

    flush("products on two streams")
    data = []
    for k in range(2):
        s = species_of(9000, 4, "rare", gpu)
        x, w, b = normal((9000, 72), "bfloat16", k, gpu), normal((4, 72, 136), "bfloat16", k + 2, gpu, 0.1), normal((4, 136), "bfloat16", 9, gpu)
        data.append((x, w, b, None, normal((9000, 136), "bfloat16", k + 5, gpu), s, "silu", 0.1, k))
    want = [run(*d) for d in data]
    streams = [torch.cuda.Stream() for _ in data]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for d, stream in zip(data, streams):
            with torch.cuda.stream(stream):
                got.append(run(*d))
        torch.cuda.synchronize()
        for a, c in zip(got, want):
            assert all(torch.equal(t, c[n]) for n, t in a.items())


# ---- more than 2^31 values ---------------------------------------------------------------

def test_long_rows_of_input(gpu):
    """Rows, outputs and masks behind 2^31 values."""
    import torch

    from ye3t_amd import runtime

    rows, width = 600000, 4096
    flush(f"linear and dropout of {rows} x {width}")
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device=gpu)
    x[-40:] = normal((40, width), "bfloat16", 1, gpu)
    w = normal((width, 16), "bfloat16", 2, gpu, 0.02)
    y = runtime.linear(x, w)
    want = plain.forward(x[-40:], w, None, None)["out"]
    plain.check("out", y[-40:], want, "bfloat16")
    assert not y[:-40].any()
    g = torch.zeros(rows, 16, dtype=torch.bfloat16, device=gpu)
    g[-40:] = normal((40, 16), "bfloat16", 3, gpu)
    dx, dw, _ = runtime.linear_adjoint(g, x, w)
    want = plain.backward(g[-40:], x[-40:], w, None)
    plain.check("input", dx[-40:], want["input"], "bfloat16")
    plain.check("weight", dw, want["weight"], "bfloat16")
    del dx
    dropped = runtime.dropout(x, 0.5, 4)
    want = plain.d(x[-40:]) * plain.kept(40, width, 0.5, 4, 0, rows - 40)
    assert torch.equal(plain.d(dropped[-40:]), want)


def test_long_weights(gpu):
    """Species whose weights lie behind 2^31 values."""
    import torch

    from ye3t_amd import runtime

    species, a, b = 9000, 512, 512
    flush(f"linear by {species} species {a} x {b}")
    w = torch.zeros(species, a, b, dtype=torch.bfloat16, device=gpu)
    w[-3:] = normal((3, a, b), "bfloat16", 1, gpu, a ** -0.5)
    s = torch.arange(60, device=gpu) % 3 + species - 3
    x, g = normal((60, a), "bfloat16", 2, gpu), normal((60, b), "bfloat16", 3, gpu)
    groups = runtime.species_groups(s, species)
    y = runtime.species_linear(x, w, groups)
    dx, dw, _ = runtime.species_linear_adjoint(g, x, w, groups)
    want = plain.forward(x, w[-3:], None, None, s - species + 3) | plain.backward(g, x, w[-3:], None, s - species + 3)
    for n, t in (("out", y), ("input", dx), ("weight", dw[-3:])):
        plain.check(n, t, want[n], "bfloat16")
    assert not dw[:-3].any()
