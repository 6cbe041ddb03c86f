"""The products with learned weights make what a call asks for, once: kernels and memory by the gradients that are wanted."""

import pytest

from tests import _products as plain
from tests._util import flush
from tests.test_gpu_products import TYPES, normal, species_of

pytestmark = pytest.mark.gpu


@pytest.fixture
def calls(monkeypatch):
    """The names of the entry points that are called."""
    from ye3t_amd.runtime import native

    seen, library = [], native.lib()

    class Counting:
        def __getattr__(self, name):
            if name.startswith("ye3t_hip_linear") and not name.endswith("bytes"):
                seen.append(name)
            return getattr(library, name)

    monkeypatch.setattr(native, "lib", lambda: Counting())
    return seen


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("by_species", [False, True])
@pytest.mark.parametrize("activation", [None, "silu"])
def test_the_preactivation_under_autograd_is_of_the_same_product(gpu, calls, dtype, by_species, activation):
    import torch

    from ye3t_amd import runtime

    flush(f"preactivation under autograd, by species {by_species}, {activation}, {dtype}")
    lead = (3,) if by_species else ()
    x, w, b = normal((150, 24), dtype, 1, gpu), normal((*lead, 24, 40), dtype, 2, gpu), normal((*lead, 40), dtype, 3, gpu)
    r, g = normal((150, 40), dtype, 4, gpu), normal((150, 40), dtype, 5, gpu)
    groups = (runtime.species_groups(species_of(150, 3, "any", gpu), 3),) if by_species else ()
    forward = runtime.species_linear if by_species else runtime.linear
    kw = dict(activation=activation, residual=r, dropout=0.2, seed=3)
    y, z = forward(x, w, *groups, b, return_preactivation=True, **kw)
    leaf = w.clone().requires_grad_()
    del calls[:]
    out, kept = forward(x, leaf, *groups, b, return_preactivation=True, **kw)
    assert calls == ["ye3t_hip_linear"]
    assert torch.equal(out, y) and torch.equal(kept, z) and out.requires_grad and not kept.requires_grad
    (grad,) = torch.autograd.grad(out, leaf, g)
    other = w.clone().requires_grad_()
    (want,) = torch.autograd.grad(forward(x, other, *groups, b, **kw), other, g)
    assert torch.equal(grad, want)
