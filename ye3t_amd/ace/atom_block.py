"""A learned layer on the ACE features of packed structures: species vectors,
norms and attention among the atoms of each structure, with energies and forces.

    features  = B(density(edge vectors))                      stage 1 and stage 2
    x         = scale * table[species] + norm(features) M     embedding, rms_norm
    x         = x + attention(norm(x)) O                      rms_norm, atom_attention
    x         = x + D(species' matrix of silu(norm(x) M'))    linear, species_linear, where there is a hidden width
    energy    = sum over a structure's atoms of norm(x) . r   rms_norm

In training values of the features and of what is added to x may be dropped (D; dropout).
:class:`AceFeatures` makes the features of positions, differentiable through
the fused density and the product's reverse mode; :class:`AtomBlock` is the layer.
``python -m ye3t_amd.ace.atom_block`` fits one to synthetic energies and prints
energies and forces.  The products with M, O and r and those for the attention's queries, keys and values are Torch's.
"""

import dataclasses
import math

import torch

from ye3t_amd import runtime
from ye3t_amd.ace import workloads
from ye3t_amd.ace.pipeline import ACEPipeline

CUTOFF = 5.0


class _Product(torch.autograd.Function):
    """B-features of density rows, with the product's reverse mode."""

    @staticmethod
    def forward(ctx, rows, pipe):
        ctx.save_for_backward(rows)
        ctx.pipe = pipe
        return pipe.product(rows)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (rows,) = ctx.saved_tensors
        return ctx.pipe.product_adjoint(rows, grad.contiguous()), None


class AceFeatures:
    """Invariant B-features ``[N, channels * features]`` of packed structures in
    float32, differentiable in the positions: the message couplings of l up to 3 in the
    scalar sector, one set for each of 16 channels whose neighbour weights are a
    table's rows by species."""

    def __init__(self, species_count, device="cuda", seed=0):
        g = torch.Generator().manual_seed(seed)
        base = workloads.config(4)
        self.channels, self.n_max, self.l_max = 16, 8, 3
        self.pipe = ACEPipeline(dataclasses.replace(base.feature_spec, targets=(0,)), "f32",
                                accumulate=base.accumulate, density=base.density_dtype)
        self.table = torch.randn((species_count, self.channels), generator=g).to(device)
        mix = torch.randn((self.channels, self.n_max + 1), generator=g)
        mix[:, 0] = 0.0  # the constant radial function: energies would jump where a pair crosses the cutoff
        self.mix = mix.to(device)
        self.width = self.channels * self.pipe.feature_count

    def __call__(self, positions, species, offsets):
        atoms = int(positions.shape[0])
        if atoms == 0:
            return torch.zeros((0, self.width), device=positions.device)
        owner = torch.searchsorted(offsets, torch.arange(atoms, device=offsets.device), right=True) - 1
        with torch.no_grad():
            # Structures side by side along x, further apart than the cutoff, make one neighbour list.
            # Each is laid out from its own corner, in float64: in float32 a large batch, or one far from
            # the origin, would lose digits of the distances and with them pairs.
            apart = positions.detach().double()
            corner = torch.full((offsets.numel() - 1, 3), math.inf, dtype=torch.float64, device=positions.device)
            corner.scatter_reduce_(0, owner[:, None].expand(-1, 3), apart, "amin")
            apart = apart - corner[owner]
            reach = float(apart[:, 0].max()) + 2.0 * CUTOFF
            apart[:, 0] += owner * reach
            pairs = runtime.neighbor_list(apart, CUTOFF)
            rows, centres, neighbours = pairs["target_offsets"], pairs["edge_targets"], pairs["edge_sources"]
            weights = runtime.embedding(species, self.table)
        vectors = positions[neighbours] - positions[centres]
        density = runtime.ace_density(vectors, rows, neighbours, atom_count=atoms, channel_count=self.channels,
                                      n_max=self.n_max, l_max=self.l_max, cutoff=CUTOFF, lam=workloads.LAMBDA,
                                      node_features=weights, radial_mix=self.mix, out_dtype=torch.float32,
                                      accumulate_dtype=torch.float64)
        return _Product.apply(density.reshape(-1, (self.l_max + 1) ** 2), self.pipe).reshape(atoms, self.width)


class AtomBlock(torch.nn.Module):
    """Energies of packed structures from their atoms' features and species.  ``hidden``: the width of a feed-forward
    part behind the attention, whose second matrix is the species' own (0: none); ``dropout``: the share of values that
    are dropped in training, of the features and of the feed-forward part; ``layer``: the number of the first of its two
    masks.  Blocks that run with one seed take numbers of their own (0, 2, 4, ...), or they drop the same places."""

    def __init__(self, feature_width, species_count, width=128, heads=8, cap=0.0, hidden=0, dropout=0.0, layer=0):
        super().__init__()
        if width % heads:
            raise ValueError("width must be a multiple of heads")
        if not 0 <= layer < 2 ** 32 - 1:
            raise ValueError("layer must be 0 .. 2^32 - 2")
        self.width, self.heads, self.cap = int(width), int(heads), float(cap)
        matrix = lambda a, b: torch.nn.Parameter(torch.randn(a, b) / math.sqrt(a))  # noqa: E731
        ones = lambda n: torch.nn.Parameter(torch.ones(n))  # noqa: E731
        self.species = torch.nn.Parameter(torch.randn(species_count, width) / math.sqrt(width))
        self.feature_norm, self.mix = ones(feature_width), matrix(feature_width, width)
        self.attend_norm, self.project, self.join = ones(width), matrix(width, 3 * width), matrix(width, width)
        # distances in Angstrom: from local heads to heads that see the whole structure
        self.slope_logs = torch.nn.Parameter(torch.linspace(0.0, -3.0, heads))
        self.out_norm, self.readout = ones(width), torch.nn.Parameter(torch.randn(width) / width)
        self.species_count, self.hidden = int(species_count), int(hidden)
        self.dropout, self.layer = float(dropout), int(layer)
        if hidden:
            zeros = lambda *n: torch.nn.Parameter(torch.zeros(*n))  # noqa: E731
            self.hidden_norm, self.widen, self.widen_bias = ones(width), matrix(width, hidden), zeros(hidden)
            self.narrow = torch.nn.Parameter(torch.randn(species_count, hidden, width) / math.sqrt(hidden))
            self.narrow_bias = zeros(species_count, width)

    def forward(self, features, species, positions, offsets, key_mask=None, seed=None):
        """``[structures]`` energies of ``features [N, F]``, ``species [N]``, ``positions [N, 3]``
        (float32) and row offsets ``[structures + 1]``; ``key_mask [N]`` hides ghost atoms: what their
        features and positions hold reaches nothing.  With a ``seed`` (another one each step, and for each rank of a
        data-parallel run) values are dropped."""
        atoms = int(features.shape[0])
        if key_mask is not None:
            # their rows are computed with the others', and zero times what is not a number is none either
            features, positions = (t.masked_fill(~key_mask[:, None], 0.0) for t in (features, positions))
        dropped = self.dropout if seed is not None else 0.0
        if dropped:
            features = runtime.dropout(features, dropped, seed, layer=self.layer)
        mixed = runtime.rms_norm(features, self.feature_norm) @ self.mix
        vectors = runtime.embedding(species, self.species, scale=math.sqrt(self.width))
        y, x = runtime.rms_norm(mixed, self.attend_norm, residual=vectors)
        q, k, v = (y @ self.project).reshape(atoms, 3, self.heads, self.width // self.heads).unbind(1)
        seen = runtime.atom_attention(q, k, v, offsets, cap=self.cap, slopes=self.slope_logs.float().exp(),
                                      positions=positions, key_mask=key_mask)
        joined = seen.reshape(atoms, self.width) @ self.join
        if self.hidden:
            y, x = runtime.rms_norm(joined, self.hidden_norm, residual=x)
            wide = runtime.linear(y, self.widen, self.widen_bias, activation="silu")
            groups = runtime.species_groups(species, self.species_count, validate=False)  # the embedding has checked them
            y = runtime.rms_norm(runtime.species_linear(wide, self.narrow, groups, self.narrow_bias, residual=x,
                                                        dropout=dropped, seed=seed, layer=self.layer + 1),
                                 self.out_norm)
        else:
            y, x = runtime.rms_norm(joined, self.out_norm, residual=x)
        each = (y @ self.readout).float()
        if key_mask is not None:
            each = each.masked_fill(~key_mask, 0.0)
        return torch.segment_reduce(each, "sum", offsets=offsets, axis=0, initial=0)

    def descriptors(self, features):
        """The normalised features in 8 bits with their scales, a quarter of the memory of float32."""
        return runtime.rms_norm_8bit(features.detach(), self.feature_norm.detach())


def energies_and_forces(features, block, positions, species, offsets):
    """Energies of the structures and the forces on their atoms."""
    positions = positions.detach().requires_grad_()
    energies = block(features(positions, species, offsets), species, positions, offsets)
    (gradient,) = torch.autograd.grad(energies.sum(), positions)
    return energies.detach(), -gradient


def synthetic_structures(count, atoms, species_count, seed, device="cuda"):
    """Random cells of about 15 cubic Angstrom an atom, half to one and a half times ``atoms`` each."""
    g = torch.Generator().manual_seed(seed)
    lengths = torch.randint(max(1, atoms // 2), atoms + atoms // 2 + 1, (count,), generator=g)
    offsets = torch.zeros(count + 1, dtype=torch.int64)
    offsets[1:] = lengths.cumsum(0)
    side = (15.0 * lengths.double()).pow(1.0 / 3.0).float().repeat_interleave(lengths)
    total = int(offsets[-1])
    positions = torch.rand((total, 3), generator=g) * side[:, None]
    species = torch.randint(species_count, (total,), generator=g, dtype=torch.int32)
    return positions.to(device), species.to(device), offsets.to(device)


def main(steps=20, hidden=0, dropout=0.0):
    species_count = 4
    features = AceFeatures(species_count)
    torch.manual_seed(0)
    block = AtomBlock(features.width, species_count, hidden=hidden, dropout=dropout).cuda()
    positions, species, offsets = synthetic_structures(16, 40, species_count, seed=1)
    held = features(positions, species, offsets).detach()
    atoms = (offsets[1:] - offsets[:-1]).float()
    target = torch.cos(atoms)  # energies per atom to be fitted
    optimiser = torch.optim.Adam(block.parameters(), lr=2e-3)
    for step in range(steps):
        optimiser.zero_grad()
        loss = (block(held, species, positions, offsets, seed=step) / atoms - target).square().mean()
        loss.backward()
        optimiser.step()
        if step % 5 == 0 or step == steps - 1:
            print(f"step {step:3d} loss {float(loss.detach()):.4f}", flush=True)
    energies, forces = energies_and_forces(features, block, positions, species, offsets)
    codes, scales = block.descriptors(held)
    print(f"{len(atoms)} structures, {len(positions)} atoms, {features.width} features each; energies "
          f"{[round(float(e), 3) for e in energies[:4]]} ..., largest force {float(forces.abs().max()):.4f}; descriptors "
          f"{codes.numel() + 4 * scales.numel()} bytes for {4 * held.numel()}", flush=True)


if __name__ == "__main__":
    import argparse

    parser = argparse.ArgumentParser(description="Fits a layer on ACE features to synthetic energies.")
    parser.add_argument("--steps", type=int, default=20)
    parser.add_argument("--hidden", type=int, default=0, help="width of the feed-forward part")
    parser.add_argument("--dropout", type=float, default=0.0, help="share of values dropped in training")
    main(**vars(parser.parse_args()))
