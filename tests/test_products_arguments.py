"""The arguments that a product with learned weights is called with, field by field; no GPU."""

import pytest
import torch

from ye3t_amd.runtime import native


def fields(problem):
    return dict(zip(native._LINEAR_FIELDS, native._LINEAR_ARGS.unpack(problem.args)))


def test_fields_by_name():
    """Every name reaches the place that it has in the order."""
    values = {n: k + 1 for k, n in enumerate(native._LINEAR_FIELDS)}
    assert native._LINEAR_ARGS.unpack(native.linear_args(**values)) == tuple(values.values())
    for n in native._LINEAR_FIELDS:
        alone = native._LINEAR_ARGS.unpack(native.linear_args(**{n: 7}))
        assert alone == tuple(7 if m == n else 0 for m in native._LINEAR_FIELDS)


@pytest.mark.parametrize("dtype,code", [(torch.float32, native.F32), (torch.bfloat16, native.BF16)])
@pytest.mark.parametrize("by_species", [False, True])
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("held", [False, True])
def test_arguments_of_a_product(dtype, code, by_species, turned, held):
    """Distinct values in every field."""
    x = torch.zeros(13, 40, dtype=dtype)[:, 3:14]
    w = torch.zeros(*((5,) if by_species else ()), *((17, 24) if turned else (24, 17)), dtype=dtype)[..., 1:12] if turned else \
        torch.zeros(*((5,) if by_species else ()), 24, 17, dtype=dtype)[..., 2:13, 1:10]
    w = w.transpose(-1, -2) if turned else w
    outputs = w.shape[-1]
    bias, residual = torch.zeros(*((5,) if by_species else ()), outputs, dtype=dtype), torch.zeros(13, outputs, dtype=dtype)
    order, offsets = (torch.zeros(13, dtype=torch.int32), torch.zeros(6, dtype=torch.int64)) if by_species else (None, None)
    seed = torch.zeros(1, dtype=torch.int64) if held else 2 ** 63 + 19
    problem = native.Linear(x, w, bias, residual, order, offsets, 2, 6554, 31, seed)
    assert fields(problem) == dict(
        dtype=code, rows=13, inputs=11, outputs=outputs, groups_given=by_species, groups=5 if by_species else 0,
        order=order.data_ptr() if by_species else 0, offsets=offsets.data_ptr() if by_species else 0, input=x.data_ptr(),
        input_row_stride=40, weight=w.data_ptr(), weight_group_stride=17 * 24 if by_species else 0,
        weight_row_stride=24 if turned else 17, turned=turned, bias=bias.data_ptr(), residual=residual.data_ptr(), activation=2,
        drop_below=6554, layer=31, seed=0 if held else 2 ** 63 + 19, device_seed=seed.data_ptr() if held else 0)


def test_fields_that_are_not_there():
    x, w = torch.zeros(3, 4), torch.zeros(4, 6)
    got = fields(native.Linear(x, w, None, None, None, None, 0, 0, 0, 0))
    given = {"rows": 3, "inputs": 4, "outputs": 6, "input": x.data_ptr(), "input_row_stride": 4, "weight": w.data_ptr(),
             "weight_row_stride": 6}
    assert got == {n: given.get(n, 0) for n in native._LINEAR_FIELDS}
