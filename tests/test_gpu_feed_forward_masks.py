"""The masks of several layers on ACE features that run with one seed."""

import copy

import pytest

from tests import _products
from tests._util import flush

pytestmark = pytest.mark.gpu


def test_layers_drop_places_of_their_own(gpu):
    """A layer's two masks are those of its own two numbers: its energies are what it gives, without dropout, of features
    that are dropped by hand, and two layers of one seed drop different places."""
    import torch

    from ye3t_amd.ace.atom_block import AtomBlock, synthetic_structures

    flush("masks of two layers")
    positions, species, offsets = synthetic_structures(4, 12, 3, seed=1, device=gpu)
    features = torch.randn(len(species), 24, generator=torch.Generator().manual_seed(2)).to(gpu)
    energies = {}
    for layer in (0, 2, 7):
        torch.manual_seed(6)
        block = AtomBlock(24, 3, width=32, heads=2, dropout=0.4, layer=layer).to(gpu)
        energies[layer] = block(features, species, positions, offsets, seed=5)
        keep = _products.kept(len(species), 24, 0.4, 5, layer).float().to(gpu)
        assert torch.equal(energies[layer], block(features * keep, species, positions, offsets))
    assert not torch.equal(energies[0], energies[2]) and not torch.equal(energies[2], energies[7])
    # the feed-forward part's mask: all of it dropped but for its number
    torch.manual_seed(6)
    block = AtomBlock(24, 3, width=32, heads=2, hidden=48, dropout=0.4).to(gpu)
    other = copy.deepcopy(block)
    other.layer = 1  # its first mask is the other's second
    seen = {}
    for b in (block, other):
        for name, value in (("zeros", torch.zeros_like(features)), ("own", features)):
            seen[b.layer, name] = b(value, species, positions, offsets, seed=5)
    # features of zeros are the same however they are dropped: only the second masks are left
    assert not torch.equal(seen[0, "zeros"], seen[1, "zeros"])


@pytest.mark.parametrize("layer", [-1, 2 ** 32 - 1])
def test_numbers_of_masks(layer):
    from ye3t_amd.ace.atom_block import AtomBlock

    with pytest.raises(ValueError, match="layer"):
        AtomBlock(24, 3, width=32, heads=2, dropout=0.4, layer=layer)
