"""float32 products whose results are not finite: computed again value by value, to the end where the end counts."""

import pytest

from tests import _products as plain
from tests._util import flush
from tests.test_gpu_products import normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,inputs,outputs", [(7, 33, 13), (70, 130, 77), (1, 1030, 9), (3000, 40, 21)])
@pytest.mark.parametrize("at", [0, 14, 15, 16, 31, -1])
def test_columns_end_apart(gpu, rows, inputs, outputs, at):
    """One column of NaN from any place on, infinities of either sign in the others."""
    import torch

    from ye3t_amd import runtime

    flush(f"not finite at {at}, {rows} x {inputs} x {outputs}")
    x, w = normal((rows, inputs), "float32", 1, gpu), normal((inputs, outputs), "float32", 2, gpu)
    inf = float("inf")
    w[at, outputs // 2] = float("nan")
    x[0, at], x[-1, 0] = inf, -inf
    w[0, 0] = 0.0  # zero times infinity
    y, want = plain.d(runtime.linear(x, w)), plain.d(x) @ plain.d(w)
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    endless = torch.isinf(want)
    assert torch.equal(y[endless], want[endless]) and bool(torch.isfinite(y[torch.isfinite(want)]).all())
    g = normal((rows, outputs), "float32", 3, gpu)
    g[0, -1] = inf
    dx, dw, db = (plain.d(t) for t in runtime.linear_adjoint(g, x, w, bias=True))
    for got, exact in ((dx, plain.d(g) @ plain.d(w).T), (dw, plain.d(x).T @ plain.d(g)), (db, plain.d(g).sum(0))):
        assert torch.equal(torch.isnan(got), torch.isnan(exact)) and torch.equal(torch.isinf(got), torch.isinf(exact))
        assert torch.equal(got[torch.isinf(exact)], exact[torch.isinf(exact)])


def test_a_batch_of_nan_takes_about_its_time(gpu):
    """A diverged step: sums that are NaN are not followed to their end (with that 81 and 76 times the time of numbers)."""
    import torch

    from ye3t_amd import runtime

    rows, inputs, outputs = 20001, 1449, 256
    flush(f"a batch of NaN, {rows} x {inputs} x {outputs}")
    x, w = normal((rows, inputs), "float32", 1, gpu), normal((inputs, outputs), "float32", 2, gpu)
    g = normal((rows, outputs), "float32", 3, gpu)

    def time(call):
        call()
        ends = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        ends[0].record()
        for _ in range(5):
            call()
        ends[1].record()
        torch.cuda.synchronize()
        return ends[0].elapsed_time(ends[1])

    none, none_g = torch.full_like(x, float("nan")), torch.full_like(g, float("nan"))
    for name, call, other in (("forward", lambda: runtime.linear(x, w), lambda: runtime.linear(none, w)),
                              ("gradient", lambda: runtime.linear_adjoint(g, x, w, bias=True),
                               lambda: runtime.linear_adjoint(none_g, none, w, bias=True))):
        ratio = time(other) / time(call)
        flush(f"  {name}: {ratio:.1f} times")
        assert ratio < 20
