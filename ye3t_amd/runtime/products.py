"""Products of atoms' rows with learned weights, one for all atoms or one for
each species, and dropout.

``linear`` and ``species_linear`` add the bias, the activation, dropout and the
residual in the product's own kernel; ``species_groups`` orders a batch's atoms
by species once for all layers.  Storage is float32 or bfloat16; sums are held
in 32 bits and every output is rounded once.  float32 products are taken from
three bfloat16 parts of each value; what that leaves out is below 2^-26 of each
term, and the sums' own roundings are the larger part of their errors.
The gradient of what is behind the product is rounded to the storage type
before it is multiplied, but not where it is summed for the bias.  Dropped values follow from a seed and their place:
no mask is stored.  The forward operators are differentiable once; each has its
adjoint as a function of its own.  No reference counterparts.
"""

import math
from typing import NamedTuple

import torch

from ye3t_amd.runtime import native
from ye3t_amd.runtime.atoms import _check_tokens, _require_one_device, _tracked, _unit_rows

__all__ = ("SpeciesGroups", "species_groups", "linear", "linear_adjoint", "species_linear", "species_linear_adjoint",
           "dropout", "dropout_adjoint")

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3}


class SpeciesGroups(NamedTuple):
    """A batch's atoms by species, of :func:`species_groups`."""

    order: torch.Tensor    # int32 [atoms]: the atoms by species
    offsets: torch.Tensor  # int64 [species + 1]: where each species begins in it


def species_groups(species, species_count, *, validate=True):
    """The atoms of ``species`` (int32 or int64 ``[N]``) ordered by species, for
    :func:`species_linear`: one for all layers of a batch.  Atoms of one species
    keep their order.

    ``validate`` range-checks the species first (one kernel and one wait).  Atoms
    of a species outside ``[0, species_count)`` that is not checked belong to no
    group: their products are zero."""
    _require_one_device("species_groups", species)
    if species.dtype not in (torch.int32, torch.int64):
        raise ValueError("species must be int32 or int64")
    if species.ndim != 1:
        raise ValueError("species must be [atoms]")
    species_count = int(species_count)
    if species_count < 0:
        raise ValueError("species_count must be non-negative")
    species = species.contiguous()
    if validate:
        _check_tokens(species, species_count, "species_groups")
    return SpeciesGroups(*native.species_groups(species, species_count))


# ---- dropped values ------------------------------------------------------------

def _dropped(probability, seed, layer, device, name):
    """The checked ``(below, layer, seed)``."""
    probability, layer = float(probability), int(layer)
    if not 0.0 <= probability <= 1.0:
        raise ValueError(f"{name} must be a probability")
    if not 0 <= layer < 2 ** 32:
        raise ValueError("layer must be 0 .. 2^32 - 1")
    below = int(math.floor(probability * 65536.0 + 0.5))
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != device:
            raise ValueError("seed must be an int or one int64 value on the input's device")
    elif seed is None:
        if below:
            raise ValueError(f"{name} needs a seed")
        seed = 0
    else:
        seed = int(seed) & (2 ** 64 - 1)
    return below, layer, seed


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, residual, below, layer, seed):
        held = isinstance(seed, torch.Tensor)
        ctx.save_for_backward(*((seed,) if held else ()))  # a seed that has changed by then is an error
        ctx.below, ctx.layer, ctx.seed, ctx.added = below, layer, None if held else seed, residual is not None
        return native.dropout(input, residual, below, layer, seed)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        seed = ctx.saved_tensors[0] if ctx.saved_tensors else ctx.seed
        dx = native.dropout(grad.contiguous(), None, ctx.below, ctx.layer, seed) if ctx.needs_input_grad[0] else None
        return dx, grad if ctx.added else None, None, None, None


def dropout(input, probability, seed, *, layer=0, residual=None):
    """``residual + kept input / (1 - probability)``: each value is dropped with
    ``probability``, in steps of 2^-16.

    A value's fate follows from ``seed``, ``layer`` and its place (the column of
    the last axis and the number of the row): sixteen bits of Philox 4x32-10.
    Equal calls drop equal values, and no mask is kept for the gradient.  ``seed``
    is an int, or an int64 tensor of one value on the input's device, which a
    captured graph reads anew at each replay; ``layer`` keeps the masks of
    several layers apart.  float32 or bfloat16, rounded once; a dropped value is
    zero whatever it held.  Differentiable (:func:`dropout_adjoint`)."""
    _require_one_device("dropout", input, residual)
    if input.ndim < 1:
        raise ValueError("input must have at least one axis")
    if residual is not None and (residual.shape != input.shape or residual.dtype != input.dtype):
        raise ValueError("residual must have the input's shape and dtype")
    below, layer, seed = _dropped(probability, seed, layer, input.device, "probability")
    input = input.contiguous()
    residual = None if residual is None else residual.contiguous()
    if _tracked(input, residual):
        return _Dropout.apply(input, residual, below, layer, seed)
    return native.dropout(input, residual, below, layer, seed)


def dropout_adjoint(adjoint, probability, seed, *, layer=0):
    """Gradient of :func:`dropout` with respect to its input for the output's
    ``adjoint``; the residual's is the adjoint itself."""
    _require_one_device("dropout_adjoint", adjoint)
    if adjoint.ndim < 1:
        raise ValueError("adjoint must have at least one axis")
    below, layer, seed = _dropped(probability, seed, layer, adjoint.device, "probability")
    return native.dropout(adjoint.contiguous(), None, below, layer, seed)


# ---- products --------------------------------------------------------------------

def _laid_out(weight):
    """``weight``, or a contiguous copy where neither of its last two axes is laid out value after value."""
    if weight.stride(-1) == 1 or weight.shape[-1] == 1 or weight.stride(-2) == 1 or weight.shape[-2] == 1:
        return weight
    return weight.contiguous()


def _checked(name, input, weight, groups, bias, rows, rows_names, activation, probability, seed, layer):
    """Checks the arguments of a product; ``rows``: tensors of the output's shape or None, with their names for a refusal.
    ``(activation, below, layer, seed)``."""
    device, dtype, shape, matrix = input.device, input.dtype, input.shape, weight.shape
    order, offsets = (None, None) if groups is None else groups
    others = (weight, bias, order, offsets, *rows)
    if not input.is_cuda or any([t is not None and t.device != device for t in others]):
        _require_one_device(name, input, *others)  # says what is wrong
    if dtype != torch.float32 and dtype != torch.bfloat16:
        raise TypeError(f"unsupported dtype {dtype}; expected float32 or bfloat16")
    if not shape or len(matrix) != (2 if groups is None else 3) or shape[-1] != matrix[-2]:
        lead = "" if groups is None else "species, "
        raise ValueError(f"weight must be [{lead}inputs, outputs] with input [..., inputs]")
    if weight.dtype != dtype:
        raise ValueError(f"weight must have dtype {dtype}")
    if bias is not None and (bias.dtype != dtype or bias.shape != (*matrix[:-2], matrix[-1])):
        raise ValueError(f"bias must be {[*matrix[:-2], matrix[-1]]} of dtype {dtype}")
    for n, t in zip(rows_names, rows):
        if t is not None and (t.dtype != dtype or t.shape != (*shape[:-1], matrix[-1])):
            raise ValueError(f"{n} must be [..., outputs] of dtype {dtype} with input [..., inputs]")
    if groups is not None:
        if order.dtype != torch.int32 or offsets.dtype != torch.int64 or order.ndim != 1 or offsets.ndim != 1 or \
                not order.is_contiguous() or not offsets.is_contiguous():
            raise ValueError("groups must be of species_groups")
        if len(order) != math.prod(shape[:-1]):
            raise ValueError("groups must be of the input's rows")
        if len(offsets) != matrix[0] + 1:
            raise ValueError("weight must have a matrix for each species of the groups")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}")
    if seed is None and probability == 0.0 and layer == 0:
        return ACTIVATIONS[activation], 0, 0, 0
    return ACTIVATIONS[activation], *_dropped(probability, seed, layer, device, "dropout")


def _rows(t):
    """``[rows, columns]`` of ``t [..., columns]``."""
    return t if t.ndim == 2 else t.reshape(math.prod(t.shape[:-1]), t.shape[-1])


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, weight, bias, residual, order, offsets, shape, wanted):
        activation, below, layer, seed = shape
        problem = native.Linear(input, weight, bias, residual, order, offsets, *shape)
        out, kept = problem.forward(wanted or activation != 0)
        held = isinstance(seed, torch.Tensor)
        # a seed that has changed by then is an error
        ctx.save_for_backward(input, weight, kept if activation else None, order, offsets, seed if held else None)
        ctx.shape = (activation, below, layer, None if held else seed)
        ctx.set_materialize_grads(False)
        if kept is not None:
            ctx.mark_non_differentiable(kept)
        return out, kept

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _):
        if grad is None:
            return (None,) * 8
        input, weight, kept, order, offsets, seed = ctx.saved_tensors
        activation, below, layer, number = ctx.shape
        problem = native.Linear(input, weight, None, None, order, offsets, activation, below, layer,
                                number if seed is None else seed)
        need = ctx.needs_input_grad
        dx = dw = db = None
        if any(need[:3]):
            dx, dw, db = problem.adjoint(grad.contiguous(), kept, *need[:3])
        return dx, dw, db, grad if need[3] else None, None, None, None, None


def _product(name, input, weight, groups, bias, activation, residual, probability, seed, layer, return_preactivation):
    shape = _checked(name, input, weight, groups, bias, (residual,), ("residual",), activation, probability, seed, layer)
    order, offsets = (None, None) if groups is None else groups
    columns = weight.shape[-1]
    lead = input.shape[:-1]
    args = (_unit_rows(_rows(input)), _laid_out(weight), None if bias is None else bias.contiguous(),
            None if residual is None else _rows(residual).contiguous())
    if _tracked(*args):
        out, kept = _Linear.apply(*args, order, offsets, shape, return_preactivation)
    else:
        out, kept = native.Linear(*args, order, offsets, *shape).forward(return_preactivation)
    if len(lead) != 1:
        out, kept = out.reshape(*lead, columns), None if kept is None else kept.reshape(*lead, columns)
    return (out, kept) if return_preactivation else out


def _product_adjoint(name, adjoint, input, weight, groups, preactivation, bias, activation, probability, seed, layer):
    shape = _checked(name, input, weight, groups, None, (adjoint, preactivation), ("adjoint", "preactivation"), activation,
                     probability, seed, layer)
    if activation is not None and preactivation is None:
        raise ValueError(f"{name}: the gradient of {activation} needs the preactivation")
    order, offsets = (None, None) if groups is None else groups
    problem = native.Linear(_unit_rows(_rows(input)), _laid_out(weight), None, None, order, offsets, *shape)
    kept = None if preactivation is None else _rows(preactivation).contiguous()
    dx, dw, db = problem.adjoint(_rows(adjoint).contiguous(), kept, True, True, bool(bias))
    return dx.reshape(input.shape), dw, db


def linear(input, weight, bias=None, *, activation=None, residual=None, dropout=0.0, seed=None, layer=0,
           return_preactivation=False):
    """``residual + D(activation(input weight + bias))`` in one kernel.

    ``input [..., inputs]``, ``weight [inputs, outputs]`` (any strides; a transposed
    ``[outputs, inputs]`` is read as it lies), ``bias [outputs]``, ``residual
    [..., outputs]``, one dtype (float32 or bfloat16).  Returns ``[..., outputs]``.

    * ``activation``: None, ``"relu"`` (zero up to zero; NaN and its gradient
      pass), ``"silu"`` (``z / (1 + exp(-z))``) or
      ``"gelu"`` (``z`` times the normal distribution's integral up to ``z``).
    * ``dropout``, ``seed``, ``layer``: D drops values as :func:`dropout` does.
    * ``return_preactivation``: also ``input weight + bias``, rounded, which
      :func:`linear_adjoint` takes.

    Differentiable in input, weight, bias and residual; the gradient is taken at
    the rounded preactivation."""
    return _product("linear", input, weight, None, bias, activation, residual, dropout, seed, layer,
                    return_preactivation)


def linear_adjoint(adjoint, input, weight, *, preactivation=None, bias=False, activation=None, dropout=0.0, seed=None,
                   layer=0):
    """Gradients of :func:`linear` for the output's ``adjoint [..., outputs]`` with
    the same arguments: ``(input, weight, bias)``, the last None without ``bias``;
    the residual's is the adjoint itself.  ``preactivation`` is the forward's and
    needed with an activation.  Sums over rows are float32 in a fixed order."""
    return _product_adjoint("linear_adjoint", adjoint, input, weight, None, preactivation, bias, activation, dropout, seed,
                            layer)


def species_linear(input, weight, groups, bias=None, *, activation=None, residual=None, dropout=0.0, seed=None, layer=0,
                   return_preactivation=False):
    """:func:`linear` with the weights of each atom's species: ``weight [species,
    inputs, outputs]``, ``bias [species, outputs]``, ``groups`` of
    :func:`species_groups` for the input's rows.  Rows keep their places; atoms of
    no species have a product of zero and no gradient."""
    return _product("species_linear", input, weight, groups, bias, activation, residual, dropout, seed, layer,
                    return_preactivation)


def species_linear_adjoint(adjoint, input, weight, groups, *, preactivation=None, bias=False, activation=None, dropout=0.0,
                           seed=None, layer=0):
    """Gradients of :func:`species_linear` as :func:`linear_adjoint` gives them; a
    species without atoms has zeros."""
    return _product_adjoint("species_linear_adjoint", adjoint, input, weight, groups, preactivation, bias, activation,
                            dropout, seed, layer)
