"""Tensors of two devices in one call of the operators around the features: refused, without a GPU (tensors that have a
device and no memory)."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from ye3t_amd import runtime


def tensor(*shape, on=0, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device=f"cuda:{on}")


def ids(n, on=0):
    return tensor(n, on=on, dtype=torch.int64)


def attend(where, adjoint=False):
    """One argument of the call lies on the second device."""
    on = lambda name: int(name == where)  # noqa: E731
    q, k, v = (tensor(6, 4, 8, on=on(n)) for n in ("query", "key", "value"))
    kw = dict(key_offsets=ids(3, on("key_offsets")), slopes=tensor(4, on=on("slopes")), positions=tensor(6, 3, on=on("positions")),
              key_positions=tensor(6, 3, on=on("key_positions")), key_mask=tensor(6, on=on("key_mask"), dtype=torch.bool),
              validate=False)
    if not adjoint:
        return runtime.atom_attention(q, k, v, ids(3, on("offsets")), **kw)
    return runtime.atom_attention_adjoint(tensor(6, 4, 8, on=on("adjoint")), tensor(6, 4, 8, on=on("out")),
                                          tensor(6, 4, on=on("log_sums")), q, k, v, ids(3, on("offsets")), **kw)


@pytest.mark.parametrize("call", [
    lambda: runtime.embedding(ids(3, 1), tensor(4, 8), validate=False),
    lambda: runtime.embedding_adjoint(tensor(3, 8), ids(3, 1), 4, validate=False),
    lambda: runtime.rms_norm(tensor(4, 8), tensor(8, on=1)),
    lambda: runtime.rms_norm(tensor(4, 8), tensor(8), residual=tensor(4, 8, on=1)),
    lambda: runtime.rms_norm_8bit(tensor(4, 8), tensor(8), residual=tensor(4, 8, on=1)),
    lambda: runtime.rms_norm_adjoint(tensor(4, 8, on=1), tensor(4, 8), tensor(8)),
    lambda: runtime.rms_norm_adjoint(tensor(4, 8), tensor(4, 8), tensor(8), total_adjoint=tensor(4, 8, on=1)),
    *[lambda n=n: attend(n) for n in ("key", "value", "offsets", "key_offsets", "slopes", "positions", "key_positions", "key_mask")],
    *[lambda n=n: attend(n, True) for n in ("key", "offsets", "adjoint", "out", "log_sums")]])
def test_two_devices_are_refused(call):
    with FakeTensorMode(), pytest.raises(ValueError, match="cuda:0 and cuda:1"):
        call()
