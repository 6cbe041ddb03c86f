"""What the operators around the features refuse without a GPU: CPU tensors, and at the C entry points sizes, types
and missing arrays."""

import ctypes

import pytest
import torch

from ye3t_amd import runtime
from ye3t_amd.runtime import native

F = torch.zeros(4, 8)


@pytest.mark.parametrize("call", [
    lambda: runtime.embedding(torch.zeros(3, dtype=torch.int64), F),
    lambda: runtime.embedding_adjoint(torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64), 4),
    lambda: runtime.rms_norm(F, torch.ones(8)),
    lambda: runtime.rms_norm_8bit(F, torch.ones(8)),
    lambda: runtime.rms_norm_adjoint(F, F, torch.ones(8)),
    lambda: runtime.atom_attention(F[:, None], F[:, None], F[:, None], torch.tensor([0, 4])),
    lambda: runtime.atom_attention_adjoint(F[:, None], F[:, None], F[:, :1], F[:, None], F[:, None], F[:, None],
                                           torch.tensor([0, 4])),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(NotImplementedError, match="HIP device branch"):
        call()


def test_operators_are_listed():
    for name in ("embedding", "embedding_adjoint", "rms_norm", "rms_norm_adjoint", "rms_norm_8bit", "atom_attention",
                 "atom_attention_adjoint"):
        assert callable(getattr(runtime, name)) and name in runtime.FUSED_OPERATIONS


def error():
    return native.lib().ye3t_hip_last_error().decode()


def test_embedding_arguments():
    L = native.lib()
    assert L.ye3t_hip_embedding(0, None, 4, 0, None, 8, 5, 8, 1.0, None, None) == 0  # nothing to do
    assert L.ye3t_hip_embedding(0, None, 4, 3, None, 8, 5, 8, 1.0, None, None) == -1 and "tokens" in error()
    assert L.ye3t_hip_embedding(0, None, 2, 3, None, 8, 5, 8, 1.0, None, None) == -1 and "int32 or int64" in error()
    assert L.ye3t_hip_embedding(2, None, 4, 3, None, 8, 5, 8, 1.0, None, None) == -3
    assert L.ye3t_hip_embedding(0, None, 4, -1, None, 8, 5, 8, 1.0, None, None) == -1
    assert L.ye3t_hip_embedding_adjoint_workspace_bytes(0, 1 << 31, 5, 8) == -1
    assert L.ye3t_hip_embedding_adjoint_workspace_bytes(0, 100, 5, 8) > 0
    one = ctypes.c_void_p(256)  # never read: the call ends before
    assert L.ye3t_hip_embedding_adjoint(0, one, one, 4, 100, 5, 8, 1.0, one, one, 8, None) == -1 and "workspace" in error()


def test_norm_arguments():
    L = native.lib()
    one = ctypes.c_void_p(256)
    assert L.ye3t_hip_rms_norm(0, None, None, None, 0, 8, 1e-6, None, None, None) == 0
    assert L.ye3t_hip_rms_norm(0, one, None, one, 2, 8, 0.0, None, one, None) == -1 and "epsilon" in error()
    assert L.ye3t_hip_rms_norm(1, one, None, one, 2, 8, 1e-6, None, one, None) == -3
    assert L.ye3t_hip_rms_norm(0, one, one, one, 2, 8, 1e-6, None, one, None) == -1 and "residual" in error()
    assert L.ye3t_hip_rms_norm(0, one, None, one, 2, 0, 1e-6, None, one, None) == -1
    assert L.ye3t_hip_rms_norm_8bit(0, one, None, one, 2, 8, 1e-6, None, one, None, None) == -1 and "scales" in error()
    assert L.ye3t_hip_rms_norm_adjoint_workspace_bytes(0, 10, 8) >= 32
    assert L.ye3t_hip_rms_norm_adjoint(0, one, None, one, one, 10, 8, 1e-6, one, one, one, 4, None) == -1


def attention(**changes):
    a = dict(dtype=0, queries=10, keys=10, structures=2, heads=4, key_heads=2, head_width=16, query=256, key=256,
             value=256, query_row_stride=64, query_head_stride=16, key_row_stride=32, key_head_stride=16,
             value_row_stride=32, value_head_stride=16, offsets=256, scale=1.0, cap=0.0)
    a.update(changes)
    return native.AttentionArgs(**a)


@pytest.mark.parametrize("changes,code,match", [
    (dict(key_heads=3), -1, "multiple"), (dict(head_width=129), -5, "above 128"), (dict(head_width=0), -1, "positive"),
    (dict(dtype=1), -3, "dtype"), (dict(keys=11), -1, "key_offsets"), (dict(cap=-1.0), -1, "cap"),
    (dict(slopes=256), -1, "together"), (dict(slopes=256, positions=256, key_offsets=256), -1, "key_positions"),
    (dict(queries=-1), -1, "negative"), (dict(queries=1 << 30, keys=1 << 30), -1, "2^31"), (dict(offsets=None), -1, "offsets"),
    (dict(query=None), -1, "query")])
def test_attention_arguments(changes, code, match):
    L = native.lib()
    args = attention(**changes)
    one = ctypes.c_void_p(256)
    assert L.ye3t_hip_atom_attention(ctypes.byref(args), one, None, one, 1 << 40, None) == code
    assert match in error()
    assert L.ye3t_hip_atom_attention_adjoint(ctypes.byref(args), one, one, one, one, one, one, None, None, None, one, 1 << 40,
                                             None) == code


def test_attention_workspaces():
    L = native.lib()
    few = attention(queries=2, keys=100000, key_offsets=256)
    assert L.ye3t_hip_atom_attention_workspace_bytes(ctypes.byref(attention())) == 0
    assert L.ye3t_hip_atom_attention_workspace_bytes(ctypes.byref(few)) > 0  # split over the keys
    one = ctypes.c_void_p(256)
    assert L.ye3t_hip_atom_attention(ctypes.byref(few), one, None, None, 0, None) == -1 and "workspace" in error()
    plain = L.ye3t_hip_atom_attention_adjoint_workspace_bytes(ctypes.byref(attention()), 0)
    assert 0 < plain < L.ye3t_hip_atom_attention_adjoint_workspace_bytes(
        ctypes.byref(attention(slopes=256, positions=256)), 1)
    assert L.ye3t_hip_atom_attention_adjoint(ctypes.byref(attention()), one, one, one, one, one, one, None, None, None, one,
                                             plain - 1, None) == -1 and "workspace" in error()
    assert L.ye3t_hip_atom_attention_adjoint(ctypes.byref(attention()), one, one, one, one, one, one, one, one, None, one,
                                             1 << 40, None) == -1 and "slopes" in error()
