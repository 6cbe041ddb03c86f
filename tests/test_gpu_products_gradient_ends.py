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
