"""What the products with learned weights and dropout refuse without a GPU: CPU tensors, tensors of two devices and wrong
shapes, and at the C entry points sizes, types and missing arrays."""

import ctypes

import pytest
import torch

from tests import _products as plain
from ye3t_amd import runtime
from ye3t_amd.runtime import native

F = torch.zeros(4, 8)
W = torch.zeros(8, 6)
G = runtime.SpeciesGroups(torch.zeros(4, dtype=torch.int32), torch.zeros(3, dtype=torch.int64))


@pytest.mark.parametrize("call", [
    lambda: runtime.linear(F, W),
    lambda: runtime.linear_adjoint(torch.zeros(4, 6), F, W),
    lambda: runtime.species_groups(torch.zeros(4, dtype=torch.int32), 2),
    lambda: runtime.species_linear(F, torch.zeros(2, 8, 6), G),
    lambda: runtime.species_linear_adjoint(torch.zeros(4, 6), F, torch.zeros(2, 8, 6), G),
    lambda: runtime.dropout(F, 0.1, 0),
    lambda: runtime.dropout_adjoint(F, 0.1, 0),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(NotImplementedError, match="HIP device branch"):
        call()


def test_operators_are_listed():
    for name in ("linear", "linear_adjoint", "species_groups", "species_linear", "species_linear_adjoint", "dropout",
                 "dropout_adjoint"):
        assert callable(getattr(runtime, name)) and name in runtime.FUSED_OPERATIONS


def test_generator():
    """The published answers of Philox 4x32-10, for the plain form that the kernels are held to."""
    words = lambda c, k: [int(w) for w in plain.philox(c, k)]  # noqa: E731
    assert words((0, 0, 0, 0), (0, 0)) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert words((0xffffffff,) * 4, (0xffffffff,) * 2) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert words((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0)) == \
        [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]


def error():
    return native.lib().ye3t_hip_last_error().decode()


def arguments(**changes):
    a = dict(dtype=0, rows=10, inputs=8, outputs=6, input=256, input_row_stride=8, weight=256, weight_row_stride=6)
    a.update(changes)
    return native.linear_args(**a)


def test_layout_of_the_arguments():
    """The packed bytes against the header's struct, field by field in its order."""
    import os
    import re

    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "ye3t_hip.h")).read()
    body = re.search(r"typedef struct \{([^}]*)\} ye3t_linear_args;", text).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names, codes = [], ""
    for line in filter(None, (" ".join(part.split()) for part in body.split(";"))):
        kind = re.match(r"(const \w+\*|\w+) ", line).group(1)
        for name in line[len(kind):].split(","):
            names.append(name.strip())
            codes += {"int": "i", "int64_t": "q", "uint32_t": "I", "uint64_t": "Q"}.get(kind, "P")
    assert tuple(names) == native._LINEAR_FIELDS
    assert "@" + codes == native._LINEAR_ARGS.format


@pytest.mark.parametrize("changes,code,match", [
    (dict(rows=-1), -1, "negative"), (dict(inputs=-1), -1, "negative"), (dict(groups=-1), -1, "negative"),
    (dict(dtype=1), -3, "dtype"), (dict(dtype=9), -3, "dtype"), (dict(rows=(1 << 31) - 256), -1, "2^31"),
    (dict(outputs=(1 << 24) + 1), -1, "2^24"), (dict(groups=1 << 24), -1, "2^24"), (dict(activation=4), -1, "activation"),
    (dict(activation=-1), -1, "activation"), (dict(drop_below=65537), -1, "dropped"), (dict(drop_below=-1), -1, "dropped"),
    (dict(input=0), -1, "input"), (dict(weight=0), -1, "weight"), (dict(groups_given=1, groups=2), -1, "order"),
    (dict(groups_given=1, groups=2, order=256), -1, "order"), (dict(input_row_stride=-8), -1, "strides"),
    (dict(weight_row_stride=-6), -1, "strides")])
def test_product_arguments(changes, code, match):
    L = native.lib()
    args, one = arguments(**changes), ctypes.c_void_p(256)  # never read: the calls end before
    assert L.ye3t_hip_linear(args, None, one, one, 1 << 40, None) == code and match in error()
    assert L.ye3t_hip_linear_adjoint(args, one, one, one, one, one, one, 1 << 40, None) == code and match in error()


def test_product_outputs_and_workspaces():
    L = native.lib()
    one = ctypes.c_void_p(256)
    assert L.ye3t_hip_linear(None, None, one, None, 0, None) == -1
    assert L.ye3t_hip_linear(arguments(rows=0, input=0), None, None, None, 0, None) == 0  # nothing to do
    assert L.ye3t_hip_linear(arguments(), None, None, None, 0, None) == -1 and "output" in error()
    assert L.ye3t_hip_linear_workspace_bytes(arguments()) == 0
    few = arguments(rows=3, inputs=4096, input_row_stride=4096)
    size = L.ye3t_hip_linear_workspace_bytes(few)
    assert size > 0  # split over the contraction
    assert L.ye3t_hip_linear(few, None, one, one, size - 1, None) == -1 and "workspace" in error()
    assert L.ye3t_hip_linear(few, None, one, None, 0, None) == -1 and "workspace" in error()
    assert L.ye3t_hip_linear_workspace_bytes(arguments(rows=-1)) == -1
    assert L.ye3t_hip_linear_workspace_bytes(None) == -1
    size = L.ye3t_hip_linear_adjoint_workspace_bytes(arguments(activation=2))
    assert size > L.ye3t_hip_linear_adjoint_workspace_bytes(arguments()) > 0
    adjoint = L.ye3t_hip_linear_adjoint
    assert adjoint(arguments(activation=2), one, one, one, one, one, one, size - 1, None) == -1 and "workspace" in error()
    assert adjoint(arguments(activation=2), one, None, one, one, one, one, size, None) == -1 and "preactivation" in error()
    assert adjoint(arguments(), None, None, one, one, one, one, size, None) == -1 and "adjoint" in error()
    assert adjoint(arguments(), one, None, one, None, one, one, size, None) == -1 and "bias" in error()
    assert adjoint(arguments(), one, None, one, one, one, None, size, None) == -1 and "workspace" in error()


def test_group_arguments():
    L = native.lib()
    one = ctypes.c_void_p(256)
    size = L.ye3t_hip_species_groups_workspace_bytes(10000, 5)
    assert size > 0 and L.ye3t_hip_species_groups_workspace_bytes(-1, 5) == -1
    assert L.ye3t_hip_species_groups_workspace_bytes((1 << 31) - 256, 5) == -1
    assert L.ye3t_hip_species_groups_workspace_bytes(5, 1 << 24) == -1
    call = L.ye3t_hip_species_groups
    assert call(one, 2, 10, 5, one, one, one, size, None) == -1 and "int32 or int64" in error()
    assert call(None, 4, 10, 5, one, one, one, size, None) == -1 and "species" in error()
    assert call(one, 4, 10, 5, one, None, one, size, None) == -1 and "outputs" in error()
    assert call(one, 4, 10000, 5, one, one, one, size - 1, None) == -1 and "workspace" in error()


def test_dropout_arguments():
    L = native.lib()
    one = ctypes.c_void_p(256)
    call = lambda dtype=0, x=one, rows=3, width=8, below=9, y=one: L.ye3t_hip_dropout(dtype, x, None, rows, width, below, 0, 0, None, y, None)  # noqa: E731,E501
    assert call(rows=0, x=None, y=None) == 0 and call(width=0, x=None, y=None) == 0  # nothing to do
    assert call(x=None) == -1 and call(y=None) == -1 and "output" in error()
    assert call(dtype=1) == -3 and call(below=65537) == -1 and call(below=-1) == -1 and "dropped" in error()
    assert call(rows=-1) == -1 and call(width=(1 << 24) + 1) == -1 and call(rows=1 << 62) == -1 and "rows" in error()


class OnGPU:
    """A stand-in with a GPU tensor's attributes, for refusals that come before any launch."""

    def __init__(self, *shape, dtype=torch.float32, index=0):
        self.t = torch.zeros(shape, dtype=dtype)
        self.is_cuda, self.device = True, torch.device("cuda", index)

    def __getattr__(self, name):
        return getattr(self.t, name)

    def __len__(self):
        return len(self.t)


def groups(rows=4, species=2, order=torch.int32, offsets=torch.int64):
    return runtime.SpeciesGroups(OnGPU(rows, dtype=order), OnGPU(species + 1, dtype=offsets))


@pytest.mark.parametrize("call,kind,match", [
    (lambda: runtime.linear(OnGPU(4, 8), OnGPU(8, 6, index=1)), ValueError, "cuda:1"),
    (lambda: runtime.linear(OnGPU(4, 8), OnGPU(8, 6), OnGPU(6, index=1)), ValueError, "cuda:1"),
    (lambda: runtime.linear(OnGPU(4, 8), OnGPU(8, 6), residual=OnGPU(4, 6, index=1)), ValueError, "cuda:1"),
    (lambda: runtime.linear(OnGPU(4, 8), OnGPU(7, 6)), ValueError, "weight must be"),
    (lambda: runtime.linear(OnGPU(4, 8), OnGPU(2, 8, 6)), ValueError, "weight must be"),
    (lambda: runtime.linear(OnGPU(4, 8, dtype=torch.float16), OnGPU(8, 6)), TypeError, "float16"),
    (lambda: runtime.linear(OnGPU(4, 8, dtype=torch.float64), OnGPU(8, 6)), TypeError, "float64"),
    (lambda: runtime.linear(OnGPU(4, 8), OnGPU(8, 6, dtype=torch.bfloat16)), ValueError, "weight must have dtype"),
    (lambda: runtime.linear(OnGPU(4, 8), OnGPU(8, 6), OnGPU(5)), ValueError, "bias must be"),
    (lambda: runtime.linear(OnGPU(4, 8), OnGPU(8, 6), OnGPU(6, dtype=torch.bfloat16)), ValueError, "bias must be"),
    (lambda: runtime.linear(OnGPU(4, 8), OnGPU(8, 6), residual=OnGPU(4, 8)), ValueError, "residual must be"),
    (lambda: runtime.linear(OnGPU(4, 8), OnGPU(8, 6), activation="tanh"), ValueError, "activation must be"),
    (lambda: runtime.linear(OnGPU(4, 8), OnGPU(8, 6), dropout=0.5), ValueError, "needs a seed"),
    (lambda: runtime.linear(OnGPU(4, 8), OnGPU(8, 6), dropout=1.5, seed=1), ValueError, "probability"),
    (lambda: runtime.linear(OnGPU(4, 8), OnGPU(8, 6), dropout=float("nan"), seed=1), ValueError, "probability"),
    (lambda: runtime.linear(OnGPU(4, 8), OnGPU(8, 6), dropout=0.5, seed=1, layer=-1), ValueError, "layer"),
    (lambda: runtime.linear(OnGPU(4, 8), OnGPU(8, 6), dropout=0.5, seed=1, layer=2 ** 32), ValueError, "layer"),
    (lambda: runtime.linear(OnGPU(4, 8), OnGPU(8, 6), dropout=0.5, seed=torch.zeros(1, dtype=torch.int64)), ValueError, "seed"),
    (lambda: runtime.linear_adjoint(OnGPU(4, 5), OnGPU(4, 8), OnGPU(8, 6)), ValueError, "adjoint must be"),
    (lambda: runtime.linear_adjoint(OnGPU(4, 6), OnGPU(4, 8), OnGPU(8, 6), activation="silu"), ValueError, "preactivation"),
    (lambda: runtime.linear_adjoint(OnGPU(4, 6), OnGPU(4, 8), OnGPU(8, 6), preactivation=OnGPU(6, 4)), ValueError,
     "preactivation must be"),
    (lambda: runtime.species_linear(OnGPU(4, 8), OnGPU(8, 6), groups()), ValueError, "weight must be"),
    (lambda: runtime.species_linear(OnGPU(4, 8), OnGPU(2, 8, 6), groups(5)), ValueError, "input's rows"),
    (lambda: runtime.species_linear(OnGPU(4, 8), OnGPU(2, 8, 6), groups(4, 3)), ValueError, "each species"),
    (lambda: runtime.species_linear(OnGPU(4, 8), OnGPU(2, 8, 6), groups(order=torch.int64)), ValueError, "species_groups"),
    (lambda: runtime.species_linear(OnGPU(4, 8), OnGPU(2, 8, 6), groups(), OnGPU(6)), ValueError, "bias must be"),
    (lambda: runtime.species_groups(OnGPU(4, dtype=torch.float32), 2), ValueError, "int32 or int64"),
    (lambda: runtime.species_groups(OnGPU(4, 2, dtype=torch.int32), 2), ValueError, "species must be"),
    (lambda: runtime.species_groups(OnGPU(4, dtype=torch.int32), -1), ValueError, "non-negative"),
    (lambda: runtime.dropout(OnGPU(4, 8), 0.5, None), ValueError, "needs a seed"),
    (lambda: runtime.dropout(OnGPU(4, 8), -0.1, 1), ValueError, "probability"),
    (lambda: runtime.dropout(OnGPU(4, 8), 0.1, 1, residual=OnGPU(4, 7)), ValueError, "residual must have"),
    (lambda: runtime.dropout(OnGPU(4, 8), 0.1, 1, residual=OnGPU(4, 8, index=1)), ValueError, "cuda:1"),
    (lambda: runtime.dropout(OnGPU(), 0.1, 1), ValueError, "one axis"),
])
def test_refusals(call, kind, match):
    with pytest.raises(kind, match=match):
        call()
