"""The layer that runs the species vectors, norms and attention on ACE features."""

import pytest

from tests._util import flush, rotation

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(gpu):
    import torch

    from ye3t_amd.ace.atom_block import AceFeatures, AtomBlock, synthetic_structures

    features = AceFeatures(3, device=gpu)
    torch.manual_seed(4)
    block = AtomBlock(features.width, 3, width=64, heads=4, cap=8.0).to(gpu)
    return features, block, synthetic_structures(3, 12, 3, seed=2, device=gpu)


def test_energies_are_invariant_and_additive(model):
    import torch

    flush("energies under rotation, translation, and of structures by themselves")
    features, block, (positions, species, offsets) = model
    with torch.no_grad():
        energies = block(features(positions, species, offsets), species, positions, offsets)
        turn = torch.as_tensor(rotation(5), dtype=torch.float32, device=positions.device)
        moved = positions @ turn.T + 3.0
        again = block(features(moved, species, offsets), species, moved, offsets)
        # fp32 features of a few hundred terms, two norms and the attention: below 1e-4 of the energies' size
        size = float(energies.abs().max())
        assert float((energies - again).abs().max()) < 1e-4 * size
        for s in range(3):
            a, b = int(offsets[s]), int(offsets[s + 1])
            own = torch.tensor([0, b - a], device=positions.device)
            one = block(features(positions[a:b], species[a:b], own), species[a:b], positions[a:b], own)
            assert abs(float(one[0] - energies[s])) < 1e-4 * size
        mask = torch.ones(len(species), dtype=torch.bool, device=positions.device)
        mask[0] = False
        masked = block(features(positions, species, offsets), species, positions, offsets, key_mask=mask)
        assert abs(float(masked[0] - energies[0])) > 1e-6 and float((masked - energies)[1:].abs().max()) < 1e-4 * size


def test_forces_are_the_energies_derivative(model):
    import torch

    from ye3t_amd.ace.atom_block import energies_and_forces

    flush("forces against differences of the energies")
    features, block, (positions, species, offsets) = model
    energies, forces = energies_and_forces(features, block, positions, species, offsets)
    g = torch.Generator().manual_seed(8)
    for _ in range(4):
        direction = torch.randn(positions.shape, generator=g).to(positions.device)
        direction /= direction.norm()

        def energy(step):
            moved = positions + step * direction
            with torch.no_grad():
                return float(block(features(moved, species, offsets), species, moved, offsets).double().sum())

        # central differences: energies in fp32 (1e-6 of their size) over 2 h, and h^2 times third derivatives
        h = 4e-3
        slope = (energy(h) - energy(-h)) / (2 * h)
        got = -float((forces * direction).sum())
        flush(f"  {got:.6f} and {slope:.6f}")
        assert abs(got - slope) < 5e-3 * float(forces.norm()) + 1e-6 * float(energies.abs().sum()) / h


def test_training_gradients_reach_every_parameter(model):
    import torch

    flush("gradients of the layer's parameters; the layer in bf16; descriptors")
    features, block, (positions, species, offsets) = model
    held = features(positions, species, offsets).detach()
    energies = block(held, species, positions, offsets)
    exact_energies = energies.detach()
    grads = torch.autograd.grad(energies.square().sum(), list(block.parameters()))
    assert all(bool(g.isfinite().all()) and bool(g.any()) for g in grads)
    half = type(block)(features.width, 3, width=64, heads=4, cap=8.0).to(positions.device)
    half.load_state_dict(block.state_dict())
    half.bfloat16()
    low = half(held.bfloat16(), species, positions, offsets).detach()
    # a dozen roundings of 2^-9 on the way
    assert float((low - exact_energies).norm() / exact_energies.norm()) < 12 * 2.0 ** -9 * 3
    codes, scales = block.descriptors(held)
    values = codes.float() * scales.repeat_interleave(128, dim=1)[:, :features.width]
    from ye3t_amd import runtime

    exact = runtime.rms_norm(held, block.feature_norm.detach())
    assert float((values - exact).abs().max() / exact.abs().max()) < 2.0 ** -4
