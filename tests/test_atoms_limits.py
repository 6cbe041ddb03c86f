"""Sizes at the ends of what the operators around the features take, at the C entry points and without a GPU."""

import ctypes

import pytest

from ye3t_amd.runtime import native
from tests.test_atoms_refusals import attention, error


def workspace(**changes):
    return native.lib().ye3t_hip_atom_attention_workspace_bytes(ctypes.byref(attention(**changes)))


def test_arrays_without_values_may_be_null():
    """What an empty tensor's address is."""
    assert workspace(queries=0, slopes=256, positions=None, key_offsets=256, key_positions=256) == 0
    assert workspace(keys=0, slopes=256, positions=256, key_offsets=256, key_positions=None, key=None, value=None) == 0
    assert workspace(queries=0, keys=0, slopes=256) == 0
    args = attention(queries=0, keys=0, slopes=256)
    assert native.lib().ye3t_hip_atom_attention_adjoint_workspace_bytes(ctypes.byref(args), 1) > 0
    assert workspace(slopes=256) == -1 and "together" in error()
    assert workspace(positions=256) == -1 and "together" in error()
    assert workspace(slopes=256, positions=256, key_offsets=256) == -1 and "key_positions" in error()
