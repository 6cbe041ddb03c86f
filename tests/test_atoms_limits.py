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


def test_rows_and_keys_of_attention():
    """The kernels count a structure's rows and keys in 32 bits, up to two tiles of 128 past its end."""
    most = 2 ** 31 - 256
    for heads in (1, 4):
        for name in ("queries", "keys"):
            for atoms, fits in ((most // heads, True), (most // heads + 1, False)):
                sizes = dict(queries=1, keys=1) | {name: atoms}
                found = workspace(**sizes, heads=heads, key_heads=1, key_offsets=256)
                assert (found >= 0) == fits, (name, atoms)
                if not fits:
                    assert "2^31 - 256" in error()


def last_indices(length, tile_keys, tile, waves):
    """The largest numbers that a walk over `length` keys forms: tiles of keys with one looked at ahead, and the keys of
    the last workgroup of the key-side gradient."""
    tiles = (length + tile_keys - 1) // tile_keys
    ahead = tiles * tile_keys + 63
    first = (length - 1) // tile * tile
    return max(length + tile_keys - 1, (tiles + 1) * tile_keys, ahead, first + 32 * (waves - 1) + 31, first + 32 * waves)


@pytest.mark.parametrize("tile_keys", [32, 64])
@pytest.mark.parametrize("waves", [1, 4])
def test_indices_of_the_longest_structure(tile_keys, waves):
    most = 2 ** 31 - 256
    assert last_indices(most, tile_keys, 32 * waves, waves) < 2 ** 31
    assert last_indices(2 ** 31 - 1, tile_keys, 32 * waves, waves) >= 2 ** 31  # what the limit is for
