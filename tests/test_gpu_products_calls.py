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


def memory(call):
    """The result and the bytes that the call took at most beside what was held before it."""
    import torch

    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    result = call()
    torch.cuda.synchronize()
    return result, torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inputs,outputs", [(700, 24, 40), (0, 8, 6), (9000, 40, 130), (300, 2048, 1024), (70001, 33, 9)])
@pytest.mark.parametrize("by_species", [False, True])
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("activation", [None, "silu"])
def test_a_bias_without_its_weight(gpu, dtype, rows, inputs, outputs, by_species, turned, activation):
    """Frozen weights: the biases' gradients alone and with the input's are what they are beside the weight's, to the order of
    their sums, and no gradient of the weight is made."""
    import torch

    from ye3t_amd import runtime

    flush(f"biases of {rows} x {inputs} x {outputs}, by species {by_species}, turned {turned}, {activation}, {dtype}")
    lead = (3,) if by_species else ()
    x = normal((rows, inputs), dtype, 1, gpu)
    w = normal((*lead, outputs, inputs), dtype, 2, gpu, inputs ** -0.5).transpose(-1, -2) if turned else \
        normal((*lead, inputs, outputs), dtype, 2, gpu, inputs ** -0.5)
    b, g = normal((*lead, outputs), dtype, 3, gpu), normal((rows, outputs), dtype, 5, gpu)
    s = species_of(rows, 3, "rare", gpu) if by_species else None
    groups = (runtime.species_groups(s, 3),) if by_species else ()
    forward = runtime.species_linear if by_species else runtime.linear
    kw = dict(activation=activation, dropout=0.2, seed=3) if activation else {}
    z = forward(x, w, *groups, b, return_preactivation=True, **kw)[1]
    want = plain.backward(g, x, w, z, s, activation, plain.kept(rows, outputs, 0.2, 3, 0) if activation else None)
    for with_input in (False, True):
        leaf, rows_of = b.clone().requires_grad_(), x.clone().requires_grad_(with_input)
        y = forward(rows_of, w, *groups, leaf, **kw)
        grads, taken = memory(lambda: torch.autograd.grad(y, [leaf, rows_of] if with_input else [leaf], g))
        plain.check("bias", grads[0], want["bias"], dtype)
        if with_input:
            plain.check("input", grads[1], want["input"], dtype)
        if inputs >= 2048 and not with_input:
            assert taken < w.numel() * w.element_size()
        again = torch.autograd.grad(forward(rows_of, w, *groups, leaf, **kw), leaf, g)[0]
        assert torch.equal(again, grads[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_the_rows_gradient_takes_no_shares_of_the_weights(gpu, dtype):
    """Frozen weights: beside the result only the memory of the allocator's rounding."""
    import torch

    from ye3t_amd import runtime

    rows, inputs, outputs = 16384, 2048, 1024
    flush(f"memory of the gradient of {rows} x {inputs} x {outputs} by 8 species, {dtype}")
    x, w = normal((rows, inputs), dtype, 1, gpu), normal((8, inputs, outputs), dtype, 2, gpu, inputs ** -0.5)
    g, s = normal((rows, outputs), dtype, 3, gpu), species_of(rows, 8, "any", gpu)
    leaf = x.clone().requires_grad_()
    y = runtime.species_linear(leaf, w, runtime.species_groups(s, 8))
    (dx,), taken = memory(lambda: torch.autograd.grad(y, leaf, g))
    assert taken < dx.numel() * dx.element_size() + (4 << 20)
    plain.check("input", dx, plain.backward(g, x, w, None, s)["input"], dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("frozen", [False, True])
def test_a_captured_training_step(gpu, dtype, frozen):
    """Forward and autograd's gradients in one graph, biases with and without their weights' gradients, replayed with other
    inputs and seeds beside a second graph of the same pool, with eager work between."""
    import torch

    from ye3t_amd import runtime

    flush(f"captured training step, frozen weights {frozen}, {dtype}")
    rows, a, b = 3000, 136, 264
    seed = torch.tensor([1], device=gpu)
    s = species_of(rows, 4, "rare", gpu)
    x, g = normal((rows, a), dtype, 1, gpu), normal((rows, b), dtype, 4, gpu)
    w, bias = normal((4, a, b), dtype, 2, gpu, 0.1), normal((4, b), dtype, 3, gpu)

    def step(leaves):
        groups = runtime.species_groups(s, 4, validate=False)
        y = runtime.species_linear(x, leaves[0], groups, leaves[1], activation="gelu", dropout=0.2, seed=seed, layer=1)
        return [y.detach(), *torch.autograd.grad(y, leaves[1:] if frozen else leaves, g)]

    fresh = lambda: [w.clone().requires_grad_(not frozen), bias.clone().requires_grad_()]  # noqa: E731
    step(fresh())
    torch.cuda.synchronize()
    leaves, others = fresh(), fresh()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(leaves)
    with torch.cuda.graph(other, pool=graph.pool()):
        step(others)
    for k in range(4):
        seed.fill_(10 + k)
        x.copy_(normal((rows, a), dtype, 30 + k, gpu))
        s.copy_(species_of(rows, 4, "any" if k % 2 else "rare", gpu))
        if k % 2:
            other.replay()
        graph.replay()
        got = [t.clone() for t in held]
        torch.cuda.synchronize()
        for n, c in zip(got, step(fresh())):
            assert torch.equal(n, c)


@pytest.mark.parametrize("dtype", TYPES)
def test_two_streams_of_gradients(gpu, dtype):
    """Gradients on two streams at once, each with workspaces of its own."""
    import torch

    from ye3t_amd import runtime

    flush(f"gradients on two streams, {dtype}")
    data = []
    for k in range(2):
        x, w = normal((9000, 72), dtype, k, gpu), normal((72, 136), dtype, k + 2, gpu, 0.1)
        data.append((normal((9000, 136), dtype, k + 5, gpu), x, w, normal((9000, 136), dtype, k + 7, gpu)))
    call = lambda d: runtime.linear_adjoint(*d[:3], preactivation=d[3], bias=True, activation="silu", dropout=0.1, seed=3)  # noqa: E731,E501
    want = [call(d) for d in data]
    streams = [torch.cuda.Stream() for _ in data]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for d, stream in zip(data, streams):
            with torch.cuda.stream(stream):
                got.append(call(d))
        torch.cuda.synchronize()
        for one, other in zip(got, want):
            assert all(torch.equal(t, c) for t, c in zip(one, other))
