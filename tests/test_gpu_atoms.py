"""Embedding, norm and attention against plain forms in 64 bits.

Tolerances.  fp32 results take sums of at most a few thousand terms in fp32
(sqrt(n) 2^-24 relative, below 4e-6) and exponentials of scores below 30 (30 x
2^-24): within the 2e-5 that this package holds fp32 to.  bf16 results have up
to four independent roundings of 2^-9 relative (the weights of a sum, the
output a gradient starts from, the sum they are rounded from, and the result
itself): 4 x 2^-9 in the 2-norm.  Where a result vanishes (the gradient of a softmax over one key)
the error is measured against the size of the terms that cancel.
"""

import math

import pytest

from tests import _atoms
from tests._util import flush

pytestmark = pytest.mark.gpu

TOL = {"float32": 2e-5, "bfloat16": 4 * 2.0 ** -9, "float64": 1e-12}


def near(got, want, dtype, floor=0.0, what=""):
    import torch

    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape
    if not want.numel():
        return
    assert torch.isfinite(got).all(), what
    n = math.sqrt(want.numel())
    error = float((got - want).norm()) / max(float(want.norm()), floor * n, 1e-300)
    worst = float((got - want).abs().max()) / max(float(want.abs().max()), floor, 1e-300)
    flush(f"  {what} error {error:.2e}, worst {worst:.2e}")
    assert error <= TOL[dtype], what
    assert worst <= 4 * TOL[dtype], what


def normal(shape, dtype, seed, gpu, sd=1.0):
    import torch

    t = torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * sd
    return t.to(getattr(torch, dtype)).to(gpu)


# ---- embedding -----------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["float32", "float64", "bfloat16"])
@pytest.mark.parametrize("shape,rows,width", [((1,), 1, 1), ((0,), 5, 7), ((3, 5), 4, 16), ((257,), 3, 33), ((4099,), 300, 130),
                                              ((2048,), 70000, 9), ((30011,), 8, 128), ((5000,), 5000, 1030)])
def test_embedding(gpu, dtype, shape, rows, width):
    flush(f"embedding {shape} of {rows} x {width}, {dtype}")
    import torch

    from ye3t_amd import runtime

    g = torch.Generator().manual_seed(3)
    # half of all positions share one token
    tokens = torch.where(torch.rand(shape, generator=g) < 0.5, rows // 2, torch.randint(rows, shape, generator=g))
    table = normal((rows, width), dtype, 1, gpu)
    adjoint = normal((*shape, width), dtype, 2, gpu)
    for index in (torch.int32, torch.int64):
        ids = tokens.to(index).to(gpu)
        out = runtime.embedding(ids, table, scale=1.7)
        near(out, table.double().cpu()[tokens] * 1.7, dtype, what="rows")
        grad = runtime.embedding_adjoint(adjoint, ids, rows, scale=1.7)
        want = torch.zeros((rows, width), dtype=torch.float64)
        want.index_add_(0, tokens.reshape(-1), adjoint.double().cpu().reshape(-1, width) * 1.7)
        near(grad, want, dtype, what="gradient")
        assert torch.equal(grad, runtime.embedding_adjoint(adjoint, ids, rows, scale=1.7))  # bit for bit
    leaf = table.clone().requires_grad_()
    (through,) = torch.autograd.grad(runtime.embedding(ids, leaf, scale=1.7), leaf, adjoint)
    assert torch.equal(through, grad)


def test_embedding_strides_and_tokens_outside(gpu):
    import torch

    from ye3t_amd import runtime

    flush("embedding of strided tables and unchecked tokens")
    wide = normal((50, 40), "float32", 5, gpu)
    tokens = torch.arange(49, -1, -2, device=gpu)
    for table in (wide[:, 3:20], wide.t(), wide[::2], wide.as_strided((40, 17), (1, 40)), wide[:1].expand(50, 40)):
        ids = tokens % table.shape[0]
        assert torch.equal(runtime.embedding(ids, table), table[ids])
    bad = torch.tensor([0, -1, 49, 50, 2 ** 40], device=gpu)
    with pytest.raises(RuntimeError, match="out of range"):
        runtime.embedding(bad, wide)
    out = runtime.embedding(bad, wide, validate=False)
    assert torch.equal(out[[0, 2]], wide[[0, 49]]) and not out[[1, 3, 4]].any()
    grad = runtime.embedding_adjoint(torch.ones(5, 40, device=gpu), bad, 50, validate=False)
    assert grad[0].eq(1).all() and grad[49].eq(1).all() and int(grad.count_nonzero()) == 80
    # what is not finite stays with its own token
    adjoint = torch.ones(4, 40, device=gpu)
    adjoint[1] = math.nan
    grad = runtime.embedding_adjoint(adjoint, torch.tensor([3, 4, 3, 5], device=gpu), 50)
    assert grad[4].isnan().all() and grad[3].eq(2).all() and grad[5].eq(1).all()


# ---- norm ----------------------------------------------------------------------

WIDTHS = [1, 2, 15, 16, 17, 64, 130, 161, 512, 1030, 2049, 5000, 8192, 20011]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("width", WIDTHS)
def test_rms_norm(gpu, dtype, width):
    import torch

    from ye3t_amd import runtime

    for rows in (1, 5, 1200 if width < 3000 else 70):
        flush(f"rms_norm {rows} x {width}, {dtype}")
        x, r, g, gt = (normal((rows, width), dtype, s, gpu) for s in (1, 2, 3, 4))
        w = normal((width,), dtype, 5, gpu)
        for residual in (None, r):
            leaves = [t.double().cpu().requires_grad_() for t in (x, w, r)]
            y, h = _atoms.rms_norm(leaves[0], leaves[1], None if residual is None else leaves[2], 1e-5)
            got = runtime.rms_norm(x, w, residual=residual, epsilon=1e-5)
            got_y, got_h = got if residual is not None else (got, x)
            near(got_y, y, dtype, what="y")
            near(got_h, h, dtype, what="sum")
            codes, scales, *rest = runtime.rms_norm_8bit(x, w, residual=residual, epsilon=1e-5)
            if rest:
                assert torch.equal(rest[0], got_h)
            groups = -(-width // 128)
            padded = torch.nn.functional.pad(y.detach(), (0, groups * 128 - width)).reshape(rows, groups, 128)
            want_scales = padded.abs().amax(-1) / 448.0
            near(scales, want_scales, "float32", what="scales")
            values = (padded / want_scales.clamp(min=1e-300)[..., None]).reshape(rows, -1)[:, :width]
            off = (codes.float().cpu().double() - _atoms.e4m3(values)).abs()
            # a value that lies on the border of two codes to within fp32's rounding may take either: one step
            assert bool((off <= values.abs().clamp(min=2.0 ** -6) * 0.126).all()) and float((off > 0).double().mean()) < 1e-3 + 2 / off.numel()
            total_grad = gt if residual is not None else None
            want = torch.autograd.grad((y, h), leaves[:2], (g.double().cpu(), gt.double().cpu() if residual is not None else torch.zeros_like(h)))
            dx, dw = runtime.rms_norm_adjoint(g, got_h, w, total_adjoint=total_grad, epsilon=1e-5)
            near(dx, want[0], dtype, floor=0.5, what="x gradient")
            near(dw, want[1], dtype, floor=0.5, what="weight gradient")


def test_rms_norm_rows_of_zeros_and_of_what_is_not_finite(gpu):
    import torch

    from ye3t_amd import runtime

    flush("rms_norm of rows of zeros, of the largest values, of NaN")
    x = torch.zeros(4, 300, device=gpu)
    x[1] = 1e18
    x[2, 7] = math.nan
    w = torch.ones(300, device=gpu)
    y = runtime.rms_norm(x, w, epsilon=1e-6)
    assert not y[0].any() and not y[3].any() and y[2].isnan().all()
    assert torch.allclose(y[1], torch.ones(300, device=gpu))
    codes, scales = runtime.rms_norm_8bit(x, w)
    assert not codes[0].float().any() and not scales[0].any()
    assert codes[2].float().isnan().all()
    assert (codes[1].float() == 448).all()
    dx, dw = runtime.rms_norm_adjoint(torch.ones_like(x), x, w)
    assert dx[2].isnan().all() and dx[0].isfinite().all() and dx[1].isfinite().all()
    dx, dw = runtime.rms_norm_adjoint(torch.ones(0, 300, device=gpu), x[:0], w)
    assert dx.shape == (0, 300) and not dw.any()


def test_rms_norm_autograd(gpu):
    import torch

    from ye3t_amd import runtime

    flush("rms_norm through autograd, with and without the sum")
    x, r = normal((7, 3, 50), "float32", 1, gpu).requires_grad_(), normal((7, 3, 50), "float32", 2, gpu).requires_grad_()
    w = normal((50,), "float32", 3, gpu).requires_grad_()
    for use in ("y", "sum", "both", "alone"):
        xd, rd, wd = (t.detach().double().cpu().requires_grad_() for t in (x, r, w))
        yd, hd = _atoms.rms_norm(xd, wd, None if use == "alone" else rd, 1e-6)
        if use == "alone":
            y = runtime.rms_norm(x, w)
            loss, want = y.square().sum(), yd.square().sum()
        else:
            y, h = runtime.rms_norm(x.transpose(0, 1).contiguous().transpose(0, 1), w, residual=r)
            loss = (y.pow(3).sum() if use != "sum" else 0) + (h.square().sum() if use != "y" else 0)
            want = (yd.pow(3).sum() if use != "sum" else 0) + (hd.square().sum() if use != "y" else 0)
        got = torch.autograd.grad(loss, (x, w, r), allow_unused=True)
        ref = torch.autograd.grad(want, (xd, wd, rd), allow_unused=True)
        for a, b, n in zip(got, ref, "xwr"):
            assert (a is None) == (b is None) or (a is not None and not a.any())
            if a is not None and b is not None:
                near(a, b, "float32", what=f"{use} {n}")


# ---- attention -----------------------------------------------------------------

def offsets_of(lengths, gpu):
    import torch

    o = torch.zeros(len(lengths) + 1, dtype=torch.int64)
    o[1:] = torch.tensor(lengths).cumsum(0)
    return o.to(gpu)


def problem(lengths, heads, key_heads, width, dtype, gpu, key_lengths=None, bias=False, mask=False, seed=0):
    import torch

    N = sum(lengths)
    M = N if key_lengths is None else sum(key_lengths)
    q = normal((N, heads, width), dtype, seed + 1, gpu, sd=1.5)
    k, v = (normal((M, key_heads, width), dtype, seed + s, gpu) for s in (2, 3))
    kw = {}
    if key_lengths is not None:
        kw["key_offsets"] = offsets_of(key_lengths, gpu)
    if bias:
        kw["positions"] = normal((N, 3), "float32", seed + 4, gpu, sd=3.0)
        kw["slopes"] = torch.exp2(torch.linspace(0, -3, heads)).to(gpu)
        if key_lengths is not None:
            kw["key_positions"] = normal((M, 3), "float32", seed + 5, gpu, sd=3.0)
    if mask:
        kw["key_mask"] = (torch.rand(M, generator=torch.Generator().manual_seed(seed)) < 0.8).to(gpu)
    return q, k, v, offsets_of(lengths, gpu), kw


def check(q, k, v, offsets, kw, dtype, cap=0.0, scale=None, grad=True):
    import torch

    from ye3t_amd import runtime

    names = ["slopes", "positions", "key_positions"]
    leaves = [t.detach().double().cpu().requires_grad_() for t in (q, k, v)]
    host = {n: t.cpu() for n, t in kw.items()}
    for n in names:
        if n in host:
            host[n] = host[n].double().requires_grad_()
    want, want_sums = _atoms.attention(*leaves, offsets.cpu(), scale=scale, cap=cap, **host)
    out, sums = runtime.atom_attention(q, k, v, offsets, scale=scale, cap=cap, return_log_sums=True, **kw)
    near(out, want, dtype, floor=0.1, what="out")
    seen = torch.isfinite(want_sums)
    assert torch.equal(torch.isfinite(sums).cpu(), seen) and bool((sums.cpu()[~seen] == -math.inf).all())
    near(sums[seen.to(sums.device)], want_sums[seen], "float32" if dtype == "float32" else "bfloat16", floor=1.0, what="sums")
    if not grad:
        return
    g = normal(tuple(q.shape), dtype, 77, q.device)
    bias = "slopes" in kw
    inputs = leaves + [host[n] for n in names if n in host]
    ref = torch.autograd.grad(want, inputs, g.double().cpu(), allow_unused=True)
    got = runtime.atom_attention_adjoint(g, out, sums, q, k, v, offsets, scale=scale, cap=cap, bias_gradients=bias, **kw)
    got = [t for t in got if t is not None]
    assert len(got) == len(ref)
    for a, b, n in zip(got, ref, ["q", "k", "v"] + [n for n in names if n in kw]):
        exact = n in names  # fp32 results, of bf16 calls too
        near(a, torch.zeros_like(a, dtype=torch.float64, device="cpu") if b is None else b, "float32" if exact else dtype,
             floor=0.25, what=n)
    again = runtime.atom_attention_adjoint(g, out, sums, q, k, v, offsets, scale=scale, cap=cap, bias_gradients=bias, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, [t for t in again if t is not None]))


LENGTHS = [[1], [2, 0, 1, 5], [31, 32, 33], [64, 63, 65, 1], [200, 3, 0, 129], [700]]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
@pytest.mark.parametrize("heads,key_heads,width", [(1, 1, 8), (4, 2, 32), (3, 1, 33), (2, 2, 64), (6, 3, 80), (4, 1, 128)])
def test_attention(gpu, dtype, lengths, heads, key_heads, width):
    flush(f"attention of {lengths}, {heads} heads of {key_heads}, width {width}, {dtype}")
    q, k, v, offsets, kw = problem(lengths, heads, key_heads, width, dtype, gpu)
    check(q, k, v, offsets, kw, dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("lengths", [[1, 4], [40, 33, 5], [300, 90]], ids=str)
@pytest.mark.parametrize("heads,key_heads,width", [(2, 2, 16), (4, 1, 64), (2, 1, 128)])
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("mask", [False, True])
def test_attention_bias_cap_mask(gpu, dtype, lengths, heads, key_heads, width, cap, mask):
    flush(f"attention of {lengths} with distances, {heads}/{key_heads} x {width}, cap {cap}, mask {mask}, {dtype}")
    q, k, v, offsets, kw = problem(lengths, heads, key_heads, width, dtype, gpu, bias=True, mask=mask)
    check(q, k, v, offsets, kw, dtype, cap=cap)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("lengths,keys", [([1], [5000]), ([1, 1, 0, 2], [900, 0, 7, 3000]), ([3], [1]), ([0, 7], [5, 640]),
                                          ([150], [40]), ([1] * 40, list(range(40)))], ids=str)
@pytest.mark.parametrize("heads,key_heads,width", [(4, 1, 64), (8, 8, 32), (16, 4, 128)])
@pytest.mark.parametrize("bias", [False, True])
def test_attention_to_other_atoms(gpu, dtype, lengths, keys, heads, key_heads, width, bias):
    """Few rows against long keys (split over the keys and joined), structures without rows or keys."""
    flush(f"attention of {lengths} to {keys if len(keys) < 9 else len(keys)}, {heads}/{key_heads} x {width}, bias {bias}, {dtype}")
    q, k, v, offsets, kw = problem(lengths, heads, key_heads, width, dtype, gpu, key_lengths=keys, bias=bias)
    check(q, k, v, offsets, kw, dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_attention_of_masked_structures(gpu, dtype):
    """A structure whose atoms are all masked gives zeros, and NaN, infinities and the type's lowest values in
    masked atoms reach nothing."""
    import torch

    from ye3t_amd import runtime

    flush(f"attention with everything masked, {dtype}")
    q, k, v, offsets, kw = problem([40, 70, 30], 4, 2, 64, dtype, gpu, bias=True)
    mask = torch.ones(140, dtype=torch.bool)
    mask[40:110] = False
    mask[[3, 120, 139]] = False
    kw["key_mask"] = mask.to(gpu)
    check(q, k, v, offsets, kw, dtype)
    clean = runtime.atom_attention(q, k, v, offsets, **kw)
    for value in (math.nan, math.inf, -math.inf, torch.finfo(k.dtype).min):
        k2, v2 = k.clone(), v.clone()
        k2[~kw["key_mask"]] = value
        v2[~kw["key_mask"]] = value
        out, sums = runtime.atom_attention(q, k2, v2, offsets, return_log_sums=True, **kw)
        assert torch.equal(out, clean) and not out[40:110].any()
        grads = runtime.atom_attention_adjoint(torch.ones_like(q), out, sums, q, k2, v2, offsets, bias_gradients=True, **kw)
        assert all(t is None or bool(t.isfinite().all()) for t in grads)
        assert not grads[1][~kw["key_mask"]].any() and not grads[2][~kw["key_mask"]].any()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_attention_strides(gpu, dtype):
    """Views of one projection, rows and heads in other orders, offsets of one value into an allocation."""
    import torch

    from ye3t_amd import runtime

    flush(f"attention of strided tensors, {dtype}")
    lengths, heads, width = [50, 77], 4, 40
    q, k, v, offsets, _ = problem(lengths, heads, heads, width, dtype, gpu)
    want = runtime.atom_attention(q, k, v, offsets)
    qkv = torch.stack((q, k, v), 1)
    forms = [qkv.unbind(1), torch.stack((q, k, v), 2).unbind(2), [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)],
             [t.permute(2, 1, 0).contiguous().permute(2, 1, 0) for t in (q, k, v)],
             [t.flip(0).contiguous().flip(0) for t in (q, k, v)]]
    for shift in (1, 3):
        forms.append([torch.cat((t.new_zeros(shift), t.reshape(-1)))[shift:].view(t.shape) for t in (q, k, v)])
    forms.append([torch.nn.functional.pad(t, (0, 3))[..., :width] for t in (q, k, v)])
    for a, b, c in forms:
        assert torch.equal(runtime.atom_attention(a, b, c, offsets), want)
    shared = [t[:, :1].expand(-1, heads, -1) for t in (k, v)]
    near(runtime.atom_attention(q, *shared, offsets), _atoms.attention(q.cpu(), k[:, :1].cpu(), v[:, :1].cpu(), offsets.cpu())[0], dtype,
         floor=0.1, what="broadcast keys")


def test_attention_autograd_and_differences(gpu):
    """Gradients through autograd equal the adjoint's, and differences of the 64-bit form along a direction."""
    import torch

    from ye3t_amd import runtime

    flush("attention gradients against differences")
    q, k, v, offsets, kw = problem([17, 40], 2, 1, 24, "float32", gpu, bias=True, mask=True)
    names = ("slopes", "positions")
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    bias = {n: kw[n].clone().requires_grad_() for n in names}
    out = runtime.atom_attention(*leaves, offsets, cap=4.0, key_mask=kw["key_mask"], **bias)
    g = normal(tuple(out.shape), "float32", 9, gpu)
    grads = torch.autograd.grad(out, leaves + list(bias.values()), g)
    with torch.no_grad():
        o, s = runtime.atom_attention(q, k, v, offsets, cap=4.0, return_log_sums=True, **kw)
        plain = runtime.atom_attention_adjoint(g, o, s, q, k, v, offsets, cap=4.0, bias_gradients=True, **kw)
    assert all(torch.equal(a, b) for a, b in zip(grads, plain))

    def value(step, which, direction):
        x = {"q": q, "k": k, "v": v, **{n: kw[n] for n in names}}
        x = {n: t.double().cpu() for n, t in x.items()}
        x[which] = x[which] + step * direction
        y, _ = _atoms.attention(x["q"], x["k"], x["v"], offsets.cpu(), cap=4.0, slopes=x["slopes"], positions=x["positions"],
                                key_mask=kw["key_mask"].cpu())
        return float((y * g.double().cpu()).sum())

    for which, grad in zip(("q", "k", "v", *names), grads):
        direction = normal(tuple(grad.shape), "float64", 21, "cpu")
        # a central difference: 1e-4 squared times third derivatives of order one
        slope = (value(1e-4, which, direction) - value(-1e-4, which, direction)) / 2e-4
        got = float((grad.double().cpu() * direction).sum())
        size = float(grad.double().norm().cpu() * direction.norm())
        flush(f"  {which}: {got:.6e} and {slope:.6e}")
        assert abs(got - slope) <= 2e-5 * size


def test_attention_of_atoms_at_one_place(gpu):
    """No direction between atoms that coincide: finite, and nothing added."""
    import torch

    flush("attention of coinciding atoms")
    q, k, v, offsets, kw = problem([30], 2, 2, 16, "float32", gpu, bias=True)
    kw["positions"][5:12] = kw["positions"][4].clone()
    check(q, k, v, offsets, kw, "float32")


def test_attention_large_scores(gpu):
    """Scores far outside the range of exp: the running maximum carries them."""
    import torch

    from ye3t_amd import runtime

    flush("attention with large scores")
    q, k, v, offsets, _ = problem([100], 2, 2, 32, "float32", gpu)
    for scale in (40.0, -40.0):
        out = runtime.atom_attention(q, k, v, offsets, scale=scale)
        want, _ = _atoms.attention(q.cpu(), k.cpu(), v.cpu(), offsets.cpu(), scale=scale)
        # a score of size 1000 has an error of 1e-4 in fp32, and so have its exponential and the result
        assert float((out.cpu().double() - want).abs().max()) < 2e-3


@pytest.mark.parametrize("op", ["embedding", "norm", "attention", "split attention"])
def test_streams_and_graphs(gpu, op):
    """A side stream, and a captured graph replayed between eager work: equal bits."""
    import torch

    from ye3t_amd import runtime

    flush(f"{op} on another stream and in a graph")
    if op == "embedding":
        table, ids = normal((300, 70), "float32", 1, gpu), torch.randint(300, (5000,), device=gpu)
        g = normal((5000, 70), "float32", 2, gpu)
        call = lambda: (runtime.embedding(ids, table, validate=False),  # noqa: E731
                        runtime.embedding_adjoint(g, ids, 300, validate=False))
    elif op == "norm":
        x, w, g = normal((900, 161), "float32", 1, gpu), normal((161,), "float32", 2, gpu), normal((900, 161), "float32", 3, gpu)
        call = lambda: (runtime.rms_norm(x, w), *runtime.rms_norm_8bit(x, w), *runtime.rms_norm_adjoint(g, x, w))  # noqa: E731
    else:
        lengths, keys = ([200, 60], None) if op == "attention" else ([2, 1], [4000, 900])
        q, k, v, offsets, kw = problem(lengths, 4, 2, 64, "bfloat16", gpu, key_lengths=keys, bias=True)
        g = torch.ones_like(q)

        def call():
            out, sums = runtime.atom_attention(q, k, v, offsets, return_log_sums=True, validate=False, **kw)
            grads = runtime.atom_attention_adjoint(g, out, sums, q, k, v, offsets, bias_gradients=True, validate=False, **kw)
            return (out, sums, *(t for t in grads if t is not None))

    same = lambda a, b: all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))  # noqa: E731
    want = call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    side.synchronize()
    assert same(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for _ in range(3):
        for t in held:
            t.view(torch.uint8).zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert same(held, want)
        assert same(call(), want)


def test_refusals(gpu):
    import torch

    from ye3t_amd import runtime

    flush("refusals")
    f = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device=gpu)  # noqa: E731
    ids = torch.zeros(3, dtype=torch.int64, device=gpu)
    with pytest.raises(ValueError, match="int32 or int64"):
        runtime.embedding(ids.float(), f(4, 5))
    with pytest.raises(TypeError, match="dtype"):
        runtime.embedding(ids, f(4, 5, dtype=torch.float16))
    with pytest.raises(ValueError, match="rows, width"):
        runtime.embedding(ids, f(4))
    with pytest.raises(ValueError, match="tokens.shape"):
        runtime.embedding_adjoint(f(4, 5), ids, 4)
    with pytest.raises(RuntimeError, match="out of range"):
        runtime.embedding_adjoint(f(3, 5), ids + 4, 4)
    with pytest.raises(TypeError, match="dtype"):
        runtime.rms_norm(f(3, 5, dtype=torch.float64), f(5, dtype=torch.float64))
    with pytest.raises(ValueError, match="width"):
        runtime.rms_norm(f(3, 5), f(4))
    with pytest.raises(ValueError, match="residual"):
        runtime.rms_norm(f(3, 5), f(5), residual=f(2, 5))
    with pytest.raises(RuntimeError, match="epsilon"):
        runtime.rms_norm(f(3, 5), f(5), epsilon=0.0)
    with pytest.raises(NotImplementedError, match="no gradient"):
        runtime.rms_norm_8bit(f(3, 5).requires_grad_(), f(5))
    q, offsets = f(6, 4, 8), torch.tensor([0, 2, 6], device=gpu)
    good = dict(slopes=f(4), positions=f(6, 3))
    assert runtime.atom_attention(q, q, q, offsets, **good).shape == q.shape
    for args, kw, error, match in [
            ((q, q[:, :3], q[:, :3], offsets), {}, ValueError, "multiple"),
            ((q, q[:5], q[:5], offsets), {}, ValueError, "key_offsets"),
            ((q, q, q[..., :4], offsets), {}, ValueError, "query must be"),
            ((q, q.bfloat16(), q, offsets), {}, ValueError, "one dtype"),
            ((q.double(), q.double(), q.double(), offsets), {}, TypeError, "dtype"),
            ((f(6, 4, 129), f(6, 4, 129), f(6, 4, 129), offsets), {}, ValueError, "width"),
            ((q, q, q, offsets.int()), {}, ValueError, "int64"),
            ((q, q, q, offsets - 1), {}, ValueError, "run from 0"),
            ((q, q, q, torch.tensor([0, 4, 2, 6], device=gpu)), {}, ValueError, "non-decreasing"),
            ((q, q, q, offsets[:1]), {}, ValueError, "structures"),
            ((q, q, q, offsets), dict(cap=-1.0), ValueError, "cap"),
            ((q, q, q, offsets), dict(slopes=f(4)), ValueError, "together"),
            ((q, q, q, offsets), dict(slopes=f(3), positions=f(6, 3)), ValueError, "slopes"),
            ((q, q, q, offsets), dict(good, positions=f(6, 3).double()), ValueError, "positions"),
            ((q, q, q, offsets), dict(key_mask=f(6)), ValueError, "key_mask"),
            ((q, q, q, offsets), dict(key_offsets=offsets[:2]), ValueError, "same structures"),
            ((q, q, q, offsets), dict(good, key_offsets=offsets), ValueError, "key_positions")]:
        with pytest.raises(error, match=match):
            runtime.atom_attention(*args, **kw)
    out, sums = runtime.atom_attention(q, q, q, offsets, return_log_sums=True)
    with pytest.raises(ValueError, match="bias_gradients"):
        runtime.atom_attention_adjoint(q, out, sums, q, q, q, offsets, bias_gradients=True)
    with pytest.raises(ValueError, match="log_sums"):
        runtime.atom_attention_adjoint(q, out, sums[:3], q, q, q, offsets)


def test_unchecked_offsets_stay_inside(gpu):
    """Offsets that were not checked are clamped: the call ends, whatever it gives."""
    import torch

    from ye3t_amd import runtime

    flush("attention with offsets that were not checked")
    q, k, v, offsets, kw = problem([20, 30], 2, 2, 16, "float32", gpu, bias=True)
    for values in ([0, 900, 50], [5, 2, 50], [0, -7, 50], [10, 20, 30], [2 ** 62, 0, -2 ** 62]):
        bad = torch.tensor(values, device=gpu)
        out, sums = runtime.atom_attention(q, k, v, bad, return_log_sums=True, validate=False, **kw)
        runtime.atom_attention_adjoint(q, out, torch.zeros_like(sums), q, k, v, bad, bias_gradients=True, validate=False, **kw)
    torch.cuda.synchronize()


def test_offsets_past_32_bits(gpu):
    """Tables, rows and keys of more than 2^31 values: the last ones are the last ones."""
    import torch

    from ye3t_amd import runtime

    flush("more than 2^31 values: embedding and norm")
    rows, width = 4_200_003, 512
    big = torch.zeros((rows, width), dtype=torch.bfloat16, device=gpu)
    tail = normal((3, width), "bfloat16", 1, gpu)
    big[-3:] = tail
    ids = torch.tensor([0, rows - 1, rows - 3], device=gpu)
    assert torch.equal(runtime.embedding(ids, big), big[ids])
    weight = normal((width,), "bfloat16", 2, gpu)
    y = runtime.rms_norm(big, weight)
    assert torch.equal(y[-3:], runtime.rms_norm(tail, weight)) and not y[:100].any()
    del y
    flush("  their gradients")
    dx, dw = runtime.rms_norm_adjoint(big, big, weight)
    want = runtime.rms_norm_adjoint(tail, tail, weight)
    assert torch.equal(dx[-3:], want[0]) and torch.equal(dw, want[1])
    del dx, big
    flush("  attention to the last of 17 000 000 keys")
    keys = 17_000_000
    k = torch.zeros((keys, 1, 128), dtype=torch.bfloat16, device=gpu)
    v = torch.zeros_like(k)
    mask = torch.zeros(keys, dtype=torch.bool, device=gpu)
    seen = torch.tensor([0, 1, keys - 40, keys - 2, keys - 1], device=gpu)
    mask[seen] = True
    k[seen], v[seen] = normal((5, 1, 128), "bfloat16", 3, gpu), normal((5, 1, 128), "bfloat16", 4, gpu)
    q = normal((1, 2, 128), "bfloat16", 5, gpu)
    out = runtime.atom_attention(q, k, v, torch.tensor([0, 1], device=gpu), key_offsets=torch.tensor([0, keys], device=gpu),
                                 key_mask=mask)
    want, _ = _atoms.attention(q.cpu(), k[seen].cpu(), v[seen].cpu(), torch.tensor([0, 1]), key_offsets=torch.tensor([0, 5]))
    near(out, want, "bfloat16", what="out")
