"""Workspaces of the products' gradients by the gradients that are asked for; no GPU."""

import ctypes

import pytest

from ye3t_amd.runtime import native


def arguments(dtype, rows, inputs, outputs, activation=0, groups=None):
    a = dict(dtype=dtype, rows=rows, inputs=inputs, outputs=outputs, input=256, input_row_stride=inputs, weight=256,
             weight_row_stride=outputs, activation=activation)
    if groups is not None:
        a.update(groups_given=1, groups=groups, order=256, offsets=256, weight_group_stride=inputs * outputs)
    return native.linear_args(**a)


@pytest.mark.parametrize("dtype", [native.F32, native.BF16])
@pytest.mark.parametrize("groups", [None, 8])
@pytest.mark.parametrize("activation", [0, 2])
@pytest.mark.parametrize("rows,inputs,outputs", [(16384, 2048, 1024), (5, 40, 4096), (70000, 33, 9), (0, 8, 6)])
def test_workspaces_of_the_gradients_that_are_wanted(dtype, groups, activation, rows, inputs, outputs):
    L, args = native.lib(), arguments(dtype, rows, inputs, outputs, activation, groups)
    size = lambda *wanted: L.ye3t_hip_linear_adjoint_workspace_bytes_of(args, *wanted)  # noqa: E731
    both = L.ye3t_hip_linear_adjoint_workspace_bytes(args)
    assert both == size(1, 1, 1) == max(size(1, 1, 1), size(1, 0, 0), size(0, 1, 0), size(0, 1, 1))
    dz = (rows * outputs * (4 if dtype == native.F32 else 2) + 255) // 256 * 256 if activation else 0
    if rows == 16384:
        assert size(1, 0, 0) == dz + 256  # no parts of either product
        assert size(0, 1, 0) > dz + 4 * inputs * outputs  # shares of the rows
    one = ctypes.c_void_p(256)
    for wanted in ((1, 0, 0), (0, 1, 0), (1, 1, 1)):
        outs = [one if w else None for w in wanted]
        bytes = size(*wanted)
        assert L.ye3t_hip_linear_adjoint(args, one, one, *outs, one, bytes - 1, None) == -1
        assert "workspace" in L.ye3t_hip_last_error().decode()


def test_invalid_arguments():
    L = native.lib()
    assert L.ye3t_hip_linear_adjoint_workspace_bytes_of(None, 1, 1, 1) == -1
    assert L.ye3t_hip_linear_adjoint_workspace_bytes_of(arguments(native.F32, -1, 8, 6), 1, 0, 0) == -1
