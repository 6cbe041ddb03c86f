"""Features and energies of structures do not depend on the batch that they are in, nor on where they lie."""

import pytest

from tests._util import flush

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count,centre", [(300, 1000.0), (3000, 0.0)])
def test_features_of_the_last_structure_of_a_batch(gpu, count, centre):
    """The batch's neighbour list has the pairs that the structure has by itself: the same edge vectors in the same
    order, so features equal to within fp32 (the 2e-5 that this package holds fp32 to)."""
    import torch

    from ye3t_amd.ace.atom_block import AceFeatures, synthetic_structures

    flush(f"features of {count} structures around {centre}, and of the last ones by themselves")
    features = AceFeatures(3, device=gpu)
    positions, species, offsets = synthetic_structures(count, 20, 3, seed=6, device=gpu)
    positions = positions + centre
    ends = offsets.tolist()
    held = features(positions, species, offsets)
    for s in (0, count // 2, count - 2, count - 1):
        part = slice(ends[s], ends[s + 1])
        alone = features(positions[part], species[part], torch.tensor([0, ends[s + 1] - ends[s]], device=gpu))
        size = alone.double().square().mean(0).sqrt().clamp(min=1e-30)
        worst = float(((held[part] - alone).double().abs() / size).max())
        flush(f"  structure {s}: {worst:.2e}")
        assert worst < 2e-5


def test_what_hidden_atoms_hold_reaches_nothing(gpu):
    """Energies, forces and parameter gradients with NaN in the features and positions of hidden atoms."""
    import math

    import torch

    from ye3t_amd.ace.atom_block import AtomBlock

    flush("the layer with hidden atoms that hold no numbers")
    torch.manual_seed(3)
    block = AtomBlock(40, 3, width=64, heads=4, cap=8.0).to(gpu)
    features, positions = torch.randn(30, 40, device=gpu), torch.randn(30, 3, device=gpu) * 3.0
    species = torch.randint(3, (30,), device=gpu)
    offsets = torch.tensor([0, 12, 12, 20, 30], device=gpu)
    mask = torch.ones(30, dtype=torch.bool, device=gpu)
    mask[[2, 5, *range(12, 20)]] = False  # two atoms, and a whole structure

    def everything(value):
        x, r = features.clone(), positions.clone()
        x[~mask], r[~mask] = value, value
        x.requires_grad_(), r.requires_grad_()
        energies = block(x, species, r, offsets, key_mask=mask)
        return [energies, *torch.autograd.grad(energies.square().sum(), [x, r, *block.parameters()])]

    want = everything(0.5)
    assert float(want[0][1]) == 0.0 and float(want[0][2]) == 0.0
    for value in (math.nan, math.inf):
        assert all(torch.equal(a, b) for a, b in zip(everything(value), want))


def test_batches_without_atoms_and_atoms_without_neighbours(gpu):
    """Energies and forces of nothing, of lone atoms, and of a batch with empty structures."""
    import torch

    from ye3t_amd.ace.atom_block import AceFeatures, AtomBlock, energies_and_forces

    flush("energies and forces without atoms, and of lone atoms")
    torch.manual_seed(3)
    features = AceFeatures(3, device=gpu)
    block = AtomBlock(features.width, 3, width=64, heads=4).to(gpu)
    for ends, positions in (([0], []), ([0, 0, 0], []), ([0, 1], [[1.0, 2.0, 3.0]]),
                            ([0, 0, 1, 1, 3, 3], [[0.0, 0.0, 0.0], [0.0, 0.0, 0.0], [0.0, 0.0, 30.0]])):
        positions = torch.tensor(positions, device=gpu).reshape(-1, 3)
        species = torch.zeros(len(positions), dtype=torch.int32, device=gpu)
        energies, forces = energies_and_forces(features, block, positions, species, torch.tensor(ends, device=gpu))
        assert energies.shape == (len(ends) - 1,) and forces.shape == positions.shape
        assert bool(energies.isfinite().all()) and bool(forces.isfinite().all())
        for s in range(len(ends) - 1):
            if ends[s] == ends[s + 1]:
                assert float(energies[s]) == 0.0
