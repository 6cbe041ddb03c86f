"""The layer on ACE features with its feed-forward part and dropped values, against the same layer in 64 bits: energies,
forces' gradients and the gradients of all weights."""

import math

import pytest

from tests import _atoms, _products
from tests._util import flush

pytestmark = pytest.mark.gpu


def plain_layer(block, p, features, species, positions, offsets, seed):
    """AtomBlock.forward in 64 bits on the CPU; ``p``: its parameters by name."""
    import torch

    atoms, width = len(features), block.width
    dropped = block.dropout if seed is not None else 0.0
    keep = lambda columns, layer: _products.kept(atoms, columns, dropped, seed, layer) if dropped else 1.0  # noqa: E731
    norm = lambda x, w: _atoms.rms_norm(x, w, None, 1e-6)[0]  # noqa: E731
    x = norm(features * keep(features.shape[1], 0), p["feature_norm"]) @ p["mix"] + math.sqrt(width) * p["species"][species]
    q, k, v = (norm(x, p["attend_norm"]) @ p["project"]).reshape(atoms, 3, block.heads, -1).unbind(1)
    seen, _ = _atoms.attention(q, k, v, offsets, cap=block.cap, slopes=p["slope_logs"].exp(), positions=positions)
    x = x + seen.reshape(atoms, width) @ p["join"]
    if block.hidden:
        z = norm(x, p["hidden_norm"]) @ p["widen"] + p["widen_bias"]
        h = z * torch.sigmoid(z)
        y = torch.einsum("nh,nhw->nw", h, p["narrow"][species]) + p["narrow_bias"][species]
        x = x + y * keep(width, 1)
    each = norm(x, p["out_norm"]) @ p["readout"]
    return torch.stack([each[offsets[s]:offsets[s + 1]].sum() for s in range(len(offsets) - 1)])


@pytest.mark.parametrize("hidden,dropout,seed", [(0, 0.0, None), (136, 0.0, None), (136, 0.2, 7), (136, 0.2, None), (0, 0.3, 9)])
def test_layer(gpu, hidden, dropout, seed):
    """float32 through some ten products, norms and an attention, each within 2e-5: 2e-4 in the 2-norm of each result."""
    import torch

    from ye3t_amd.ace.atom_block import AtomBlock, synthetic_structures

    flush(f"layer with hidden width {hidden}, dropout {dropout}, seed {seed}")
    positions, species, offsets = synthetic_structures(5, 14, 4, seed=3, device=gpu)
    torch.manual_seed(6)
    block = AtomBlock(48, 4, width=64, heads=4, cap=6.0, hidden=hidden, dropout=dropout)
    if hidden:
        with torch.no_grad():
            block.widen_bias.normal_()
            block.narrow_bias.normal_()
    exact = {n: t.detach().double().requires_grad_() for n, t in block.named_parameters()}
    block = block.to(gpu)
    features = torch.randn(len(species), 48, generator=torch.Generator().manual_seed(2))
    leaves = [t.detach().double().cpu().requires_grad_() for t in (features, positions)]
    want = plain_layer(block, exact, leaves[0], species.cpu().long(), leaves[1], offsets.cpu(), seed)
    own = [features.to(gpu).requires_grad_(), positions.clone().requires_grad_()]
    got = block(own[0], species, own[1], offsets, seed=seed)
    weight = torch.randn(len(want), generator=torch.Generator().manual_seed(4)).double()
    wanted = torch.autograd.grad((want * weight).sum(), [*leaves, *exact.values()])
    (got * weight.float().to(gpu)).sum().backward()
    results = [("energies", got, want), ("features", own[0].grad, wanted[0]), ("positions", own[1].grad, wanted[1])]
    results += [(n, t.grad, g) for (n, t), g in zip(block.named_parameters(), wanted[2:])]
    for n, a, b in results:
        error = float((a.detach().double().cpu() - b).norm() / b.norm())
        flush(f"  {n} {error:.1e}")
        assert error < 2e-4, n


def test_layer_without_a_hidden_width_is_as_before(gpu):
    """The same parameters from the same seed, and values are dropped only where a seed asks for it."""
    import torch

    from ye3t_amd.ace.atom_block import AtomBlock

    torch.manual_seed(1)
    block = AtomBlock(20, 3, width=32, heads=2)
    torch.manual_seed(1)
    other = AtomBlock(20, 3, width=32, heads=2, hidden=8, dropout=0.5)
    own = dict(block.named_parameters())
    assert set(own) == {"species", "feature_norm", "mix", "attend_norm", "project", "join", "slope_logs", "out_norm", "readout"}
    for n, t in other.named_parameters():
        assert n not in own or torch.equal(t, own[n])


def test_atoms_of_no_structure_and_ghosts(gpu):
    """Ghost atoms reach nothing through the feed-forward part either; no atoms give zeros."""
    import torch

    from ye3t_amd.ace.atom_block import AtomBlock, synthetic_structures

    torch.manual_seed(6)
    block = AtomBlock(24, 3, width=32, heads=2, hidden=64, dropout=0.1).to(gpu)
    positions, species, offsets = synthetic_structures(3, 10, 3, seed=1, device=gpu)
    features = torch.randn(len(species), 24, generator=torch.Generator().manual_seed(2)).to(gpu)
    mask = torch.ones(len(species), dtype=torch.bool, device=gpu)
    mask[3] = mask[-1] = False
    clean = block(features, species, positions, offsets, key_mask=mask, seed=4)
    features[~mask] = float("nan")
    assert torch.equal(block(features, species, positions, offsets, key_mask=mask, seed=4), clean)
    none = block(features[:0], species[:0], positions[:0], torch.zeros(3, dtype=torch.int64, device=gpu), seed=4)
    assert none.shape == (2,) and not none.any()


def test_command(gpu, capsys):
    from ye3t_amd.ace import atom_block

    flush("the command with a hidden width")
    atom_block.main(steps=2, hidden=96, dropout=0.1)
    assert "energies" in capsys.readouterr().out
