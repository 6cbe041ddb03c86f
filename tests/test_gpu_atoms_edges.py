"""Embedding, norm and attention where they can go wrong: rows and atoms that are not finite, empty batches, atoms that
nearly meet or lie far away, large caps, long inputs, and gradients of every variant held to the size of their terms
element by element."""

import math

import pytest

from tests import _atoms_sizes
from tests._util import flush
from tests.test_gpu_atoms import normal, problem

pytestmark = pytest.mark.gpu

TYPES = ["float32", "bfloat16"]


def run(q, k, v, offsets, kw, cap=0.0, forces=False, g=None):
    """{name: tensor} of the forward and its gradients, and the adjoint they were taken for."""
    from ye3t_amd import runtime

    out, sums = runtime.atom_attention(q, k, v, offsets, cap=cap, return_log_sums=True, **kw)
    g = normal(tuple(q.shape), str(q.dtype).split(".")[1], 77, q.device) if g is None else g
    grads = runtime.atom_attention_adjoint(g, out, sums, q, k, v, offsets, cap=cap, bias_gradients=forces, **kw)
    names = ("q", "k", "v", "slopes", "positions", "key_positions")
    return {"out": out, "sums": sums, **{n: t for n, t in zip(names, grads) if t is not None}}, g


# ---- rows that see nothing -------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [16, 64, 128])
@pytest.mark.parametrize("lengths", [[5, 9, 4], [40, 210, 30]], ids=str)
@pytest.mark.parametrize("cap,bias", [(0.0, False), (5.0, False), (0.0, True), (5.0, True)])
def test_rows_of_a_hidden_structure_that_are_not_finite(gpu, dtype, width, lengths, cap, bias):
    """Rows that see nothing give zeros and no gradients whatever they hold; the other structures' results keep their
    bits."""
    import torch

    flush(f"rows that are not finite and see nothing, {lengths} x {width}, cap {cap}, bias {bias}, {dtype}")
    q, k, v, offsets, kw = problem(lengths, 4, 2, width, dtype, gpu, bias=bias)
    hidden = slice(lengths[0], lengths[0] + lengths[1])
    kw["key_mask"] = torch.ones(sum(lengths), dtype=torch.bool, device=gpu)
    kw["key_mask"][hidden] = False
    clean, g = run(q, k, v, offsets, kw, cap, bias)
    assert not clean["out"][hidden].any() and bool((clean["sums"][hidden] == -math.inf).all())
    for value in (math.nan, math.inf, -math.inf):
        held = [t.clone() for t in (q, k, v)]
        for t in held:
            t[hidden] = value
        other = dict(kw)
        if bias:
            other["positions"] = kw["positions"].clone()
            other["positions"][hidden] = value
        for adjoint in (g, g.index_fill(0, torch.arange(hidden.start, hidden.stop, device=gpu), value)):
            got, _ = run(*held, offsets, other, cap, bias, adjoint)
            for n, t in got.items():
                assert torch.equal(t, clean[n]), (value, n)


@pytest.mark.parametrize("dtype", TYPES)
def test_few_rows_that_are_not_finite_against_hidden_keys(gpu, dtype):
    """The same where the keys are split among workgroups and joined."""
    import torch

    flush(f"few rows that are not finite against hidden keys, {dtype}")
    q, k, v, offsets, kw = problem([2, 1, 1], 4, 2, 64, dtype, gpu, key_lengths=[3000, 900, 0], bias=True)
    kw["key_mask"] = torch.ones(3900, dtype=torch.bool, device=gpu)
    kw["key_mask"][3000:] = False
    clean, g = run(q, k, v, offsets, kw, 0.0, True)
    q, kw["positions"] = q.clone(), kw["positions"].clone()
    q[2:], kw["positions"][2:] = math.nan, math.inf
    got, _ = run(q, k, v, offsets, kw, 0.0, True, g)
    assert not got["out"][2:].any() and bool((got["sums"][2:] == -math.inf).all())
    for n, t in got.items():
        assert torch.equal(t, clean[n]), n


# ---- empty batches ---------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,keys", [([0, 0], [3, 40]), ([5, 2], [0, 0]), ([0], [0]), ([0, 0], None), ([], None), ([], [])],
                         ids=str)
@pytest.mark.parametrize("bias", [False, True])
def test_no_rows_and_no_keys(gpu, dtype, lengths, keys, bias):
    """Rows without keys give zeros, keys without rows no gradient; autograd too."""
    import torch

    from ye3t_amd import runtime

    flush(f"attention of {lengths} to {keys}, bias {bias}, {dtype}")
    q, k, v, offsets, kw = problem(lengths, 4, 2, 32, dtype, gpu, key_lengths=keys, bias=bias)
    got, _ = run(q, k, v, offsets, kw, 0.0, bias)
    assert got["out"].shape == q.shape and bool((got["sums"] == -math.inf).all())
    for n in ("out", "q", "k", "v", "slopes", "positions", "key_positions"):
        assert n not in got or not got[n].any(), n
    leaves = [t.requires_grad_() for t in (q, k, v)] + [kw[n].requires_grad_() for n in kw if n != "key_offsets"]
    out = runtime.atom_attention(q, k, v, offsets, **kw)
    for t, grad in zip(leaves, torch.autograd.grad(out.sum(), leaves)):
        assert grad.shape == t.shape and not grad.any()


def test_layer_without_atoms(gpu):
    import torch

    from ye3t_amd.ace.atom_block import AtomBlock

    flush("the layer on structures without atoms")
    block = AtomBlock(20, 3, width=32, heads=2).to(gpu)
    for ends in ([0], [0, 0, 0]):
        energies = block(torch.zeros(0, 20, device=gpu), torch.zeros(0, dtype=torch.int32, device=gpu),
                         torch.zeros(0, 3, device=gpu), torch.tensor(ends, device=gpu))
        assert energies.shape == (len(ends) - 1,) and not energies.any()


# ---- atoms that nearly meet, and far away ones -------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", [[21], [150]], ids=str)
def test_forces_of_atoms_that_nearly_meet(gpu, dtype, lengths):
    """Atoms whose squared distance is below the smallest normal float are at one place."""
    flush(f"forces of {lengths} atoms, some nearly at one place, {dtype}")
    q, k, v, offsets, kw = problem(lengths, 2, 2, 24, dtype, gpu, bias=True)
    kw["positions"][3] = 0.0
    for atom, x in ((4, 1e-20), (5, 1e-25), (6, -3e-21), (7, 1e-30)):
        kw["positions"][atom] = 0.0
        kw["positions"][atom, atom % 3] = x
    got, g = run(q, k, v, offsets, kw, 0.0, True)
    exact = _atoms_sizes.attention(q, k, v, offsets, g, **kw)
    for n, e in exact.items():
        _atoms_sizes.check(n, got[n], e, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", [[21, 12], [150, 40]], ids=str)
@pytest.mark.parametrize("far", [1e20, 1e25, 3e38, math.inf])
def test_forces_with_hidden_atoms_put_far_away(gpu, dtype, lengths, far):
    """Hidden atoms whose squared distance overflows reach nothing, see nothing and have no forces."""
    import torch

    flush(f"forces of {lengths} atoms, hidden ones at {far}, {dtype}")
    q, k, v, offsets, kw = problem(lengths, 2, 2, 24, dtype, gpu, bias=True)
    kw["key_mask"] = torch.ones(sum(lengths), dtype=torch.bool, device=gpu)
    kw["key_mask"][2:5] = False
    kw["positions"][2:4, 0] = far
    kw["positions"][4] = -far
    got, g = run(q, k, v, offsets, kw, 0.0, True)
    visible = kw["key_mask"].nonzero()[:, 0]
    # what is left when the hidden atoms are taken out
    ends = offsets.clone()
    ends[1:] -= 3
    less = {"slopes": kw["slopes"], "positions": kw["positions"][visible]}
    exact = _atoms_sizes.attention(q[visible], k[visible], v[visible], ends, g[visible], **less)
    for n, e in exact.items():
        _atoms_sizes.check(n, got[n] if n == "slopes" else got[n][visible], e, dtype)
    for n in ("out", "q", "k", "v", "positions"):
        assert not got[n][2:5].any(), n


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", [[21, 12], [150, 40]], ids=str)
@pytest.mark.parametrize("far", [1e20, 1e25])
@pytest.mark.parametrize("forces", [False, True])
def test_gradients_with_atoms_far_away(gpu, dtype, lengths, far, forces):
    """Atoms that are seen, but so far away that their squared distance overflows: they see themselves alone."""
    flush(f"gradients of {lengths} atoms, some at {far}, forces {forces}, {dtype}")
    q, k, v, offsets, kw = problem(lengths, 2, 2, 24, dtype, gpu, bias=True)
    kw["positions"][2, 0] = far
    kw["positions"][3, 0] = -far
    kw["positions"][4] = far
    got, g = run(q, k, v, offsets, kw, 0.0, forces)
    exact = _atoms_sizes.attention(q, k, v, offsets, g, **kw)
    for n, e in exact.items():
        if n in got:
            _atoms_sizes.check(n, got[n], e, dtype)


# ---- the longest structure -----------------------------------------------------------

def test_as_many_keys_as_there_may_be(gpu):
    """2^31 - 256 keys of one structure: the last ones are found, and every one gets its gradient."""
    import torch

    from ye3t_amd import runtime

    keys = 2 ** 31 - 256
    flush(f"attention of a row to the last of {keys} keys")
    k = normal((1, 1, 1), "bfloat16", 1, gpu).expand(keys, 1, 1)
    v = torch.zeros((keys, 1, 1), dtype=torch.bfloat16, device=gpu)
    v[-3:, 0, 0] = torch.tensor([3.0, 6.0, 9.0], device=gpu)
    mask = torch.zeros(keys, dtype=torch.bool, device=gpu)
    mask[-3:] = True
    q, offsets, ends = normal((1, 1, 1), "bfloat16", 2, gpu), torch.tensor([0, 1], device=gpu), torch.tensor([0, keys], device=gpu)
    out = runtime.atom_attention(q, k, v, offsets, key_offsets=ends, key_mask=mask)
    assert abs(float(out) - 6.0) <= 6.0 * 2.0 ** -8
    flush("  the gradients of keys without rows")
    none = q[:0]
    grads = runtime.atom_attention_adjoint(none, none, torch.zeros((0, 1), device=gpu), none, k, v, torch.tensor([0, 0], device=gpu),
                                           key_offsets=ends, key_mask=mask)
    assert not grads[1].any() and not grads[2].any()


# ---- caps --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [32, 64, 128])
@pytest.mark.parametrize("cap", [0.5, 30.0, 1e3, 1e5, 1e7, 1e20])
def test_caps_of_any_size(gpu, dtype, width, cap):
    """A cap far above the scores changes nothing."""
    flush(f"attention capped at {cap}, width {width}, {dtype}")
    for lengths in ([9], [170]):
        q, k, v, offsets, kw = problem(lengths, 2, 1, width, dtype, gpu, bias=True)
        got, g = run(q, k, v, offsets, kw, cap, True)
        exact = _atoms_sizes.attention(q, k, v, offsets, g, cap=cap, **kw)
        for n, e in exact.items():
            _atoms_sizes.check(n, got[n], e, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [1e-300, 1e-44, 1e-33, 1e35, 1e300])
@pytest.mark.parametrize("scale", [0.25, -3.0])
def test_caps_outside_of_fp32(gpu, dtype, cap, scale):
    """Caps too small for fp32 leave equal scores, caps too large the scores as they are."""
    import torch

    from ye3t_amd import runtime

    flush(f"attention capped at {cap}, scale {scale}, {dtype}")
    q, k, v, offsets, kw = problem([70, 9], 2, 1, 32, dtype, gpu)
    q[3] = 0.0  # scores of zero
    out, sums = runtime.atom_attention(q, k, v, offsets, scale=scale, cap=cap, return_log_sums=True)
    exact = _atoms_sizes.attention(q, k, v, offsets, q, scale=scale, cap=cap)
    _atoms_sizes.check("out", out, exact["out"], dtype)
    grads = runtime.atom_attention_adjoint(q, out, sums, q, k, v, offsets, scale=scale, cap=cap)
    _atoms_sizes.check("v", grads[2], exact["v"], dtype)
    if cap > 1:
        _atoms_sizes.check("q", grads[0], exact["q"], dtype)
        _atoms_sizes.check("k", grads[1], exact["k"], dtype)
    assert bool(torch.isfinite(grads[0]).all()) and bool(torch.isfinite(grads[1]).all())


# ---- norm ----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [5, 300, 9000])
@pytest.mark.parametrize("epsilon", [1e-300, 1e-50, 1e-40])
def test_norm_with_an_epsilon_below_fp32(gpu, dtype, width, epsilon):
    """Rows of zeros give zeros for any positive epsilon, other rows what they give without it."""
    import torch

    from ye3t_amd import runtime

    flush(f"norm of rows of zeros with epsilon {epsilon}, width {width}, {dtype}")
    x, w = normal((4, width), dtype, 1, gpu), normal((width,), dtype, 2, gpu)
    x[1] = 0.0
    y = runtime.rms_norm(x, w, epsilon=epsilon)
    assert not y[1].any() and bool(y.isfinite().all())
    near = runtime.rms_norm(x, w, epsilon=1e-20)
    assert torch.equal(y, near)
    codes, scales = runtime.rms_norm_8bit(x, w, epsilon=epsilon)
    assert not codes[1].float().any() and not scales[1].any() and bool(codes.float().isfinite().all())
    dx, dw = runtime.rms_norm_adjoint(x, x, w, epsilon=epsilon)
    assert bool(dx.isfinite().all()) and bool(dw.isfinite().all()) and not dx[1].any()
    assert torch.equal(dw, runtime.rms_norm_adjoint(x, x, w, epsilon=1e-20)[1])


def test_last_kernel_of_the_norm_in_8_bits(gpu):
    import torch

    from ye3t_amd import runtime
    from ye3t_amd.runtime import native

    flush("the kernel that the norm in 8 bits reports")
    runtime.rms_norm_8bit(torch.ones(3, 8, device=gpu), torch.ones(8, device=gpu))
    assert native.last_kernel() == "rms_norm_kernel"


def test_refusals_of_the_norms_gradient_name_their_argument(gpu):
    import torch

    from ye3t_amd import runtime

    flush("what the norm's gradient refuses")
    x, w = torch.ones(3, 8, device=gpu), torch.ones(8, device=gpu)
    with pytest.raises(ValueError, match="^adjoint must"):
        runtime.rms_norm_adjoint(x[:2], x, w)
    with pytest.raises(ValueError, match="^total_adjoint must"):
        runtime.rms_norm_adjoint(x, x, w, total_adjoint=x.bfloat16())
    with pytest.raises(ValueError, match="^residual must"):
        runtime.rms_norm(x, w, residual=x[:2])


# ---- every gradient variant, element by element --------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", [[1, 12, 20], [70, 33, 150], [600]], ids=str)
@pytest.mark.parametrize("heads,key_heads,width", [(2, 2, 16), (4, 2, 64), (3, 1, 100), (4, 2, 128)])
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("mask", [False, True])
def test_gradients_with_distances_and_without_forces(gpu, dtype, lengths, heads, key_heads, width, cap, mask):
    """Distances that no gradient is wanted of; 600 atoms also take the key side's row axis in parts."""
    import torch

    flush(f"gradients of {lengths} with distances, {heads}/{key_heads} x {width}, cap {cap}, mask {mask}, {dtype}")
    q, k, v, offsets, kw = problem(lengths, heads, key_heads, width, dtype, gpu, bias=True, mask=mask)
    got, g = run(q, k, v, offsets, kw, cap, False)
    assert set(got) == {"out", "sums", "q", "k", "v"}
    exact = _atoms_sizes.attention(q, k, v, offsets, g, cap=cap, **kw)
    for n in ("out", "q", "k", "v"):
        _atoms_sizes.check(n, got[n], exact[n], dtype)
    again, _ = run(q, k, v, offsets, kw, cap, False)
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("dtype", TYPES)
def test_autograd_with_distances_and_without_forces(gpu, dtype):
    import torch

    from ye3t_amd import runtime

    flush(f"autograd in query, key and value beside distances, {dtype}")
    q, k, v, offsets, kw = problem([30, 90], 4, 2, 40, dtype, gpu, bias=True)
    got, g = run(q, k, v, offsets, kw, 5.0, False)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = runtime.atom_attention(*leaves, offsets, cap=5.0, **kw)
    for n, t in zip("qkv", torch.autograd.grad(out, leaves, g)):
        assert torch.equal(t, got[n])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,keys", [([1, 1, 0, 2], [900, 0, 7, 3000]), ([1], [5000]), ([3], [1]), ([150], [40]), ([400], [33])],
                         ids=str)
@pytest.mark.parametrize("heads,key_heads,width", [(8, 8, 32), (4, 1, 64), (16, 4, 128)])
@pytest.mark.parametrize("forces", [False, True])
def test_gradients_to_other_atoms_by_element(gpu, dtype, lengths, keys, heads, key_heads, width, forces):
    """Few rows give each of many keys little: the last tile's keys are held to their own size."""
    flush(f"gradients of {lengths} to {keys}, {heads}/{key_heads} x {width}, forces {forces}, {dtype}")
    q, k, v, offsets, kw = problem(lengths, heads, key_heads, width, dtype, gpu, key_lengths=keys, bias=True)
    got, g = run(q, k, v, offsets, kw, 0.0, forces)
    exact = _atoms_sizes.attention(q, k, v, offsets, g, **kw)
    for n, e in exact.items():
        if n in got:
            _atoms_sizes.check(n, got[n], e, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", [[1, 12, 20], [70, 33, 150], [700]], ids=str)
@pytest.mark.parametrize("heads,key_heads,width", [(1, 1, 8), (6, 3, 80), (4, 1, 128)])
@pytest.mark.parametrize("mask", [False, True])
def test_gradients_without_distances_by_element(gpu, dtype, lengths, heads, key_heads, width, mask):
    flush(f"gradients of {lengths}, {heads}/{key_heads} x {width}, mask {mask}, {dtype}")
    q, k, v, offsets, kw = problem(lengths, heads, key_heads, width, dtype, gpu, mask=mask)
    got, g = run(q, k, v, offsets, kw)
    exact = _atoms_sizes.attention(q, k, v, offsets, g, **kw)
    for n, e in exact.items():
        _atoms_sizes.check(n, got[n], e, dtype)


# ---- embedding gradients of many tokens ------------------------------------------------

@pytest.mark.parametrize("count,rows,width", [(70001, 8, 128), (70001, 40000, 128), (300001, 300, 16), (600007, 8, 4),
                                              (600007, 100003, 5), (9001, 3, 1030), (5000, 1 << 17, 3), (5000, (1 << 24) + 5, 1),
                                              (3000, (1 << 24) + 5, 1)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float64"])
def test_embedding_gradients_of_many_tokens(gpu, dtype, count, rows, width):
    """Shares of more than 16 positions, sort runs of more than 2 048, all four sort passes: each element within its
    terms' size (fp32: sums of up to 600 007 terms in shares, below 1e-4 of it; fp64 1e-12; bf16 one rounding more)."""
    import torch

    from ye3t_amd import runtime

    flush(f"embedding gradient of {count} tokens by {rows} x {width}, {dtype}")
    g = torch.Generator().manual_seed(count)
    tokens = (torch.exp(torch.rand(count, generator=g, dtype=torch.float64) * math.log(rows + 1.0)) - 1.0).long().clamp_(0, rows - 1)
    tokens[::7] = rows - 1
    adjoint = normal((count, width), dtype, 2, gpu)
    exact, size = (torch.zeros((rows, width), dtype=torch.float64).index_add_(0, tokens, t)
                   for t in (adjoint.double().cpu(), adjoint.double().cpu().abs()))
    allowed = size * {"float32": 1e-4, "float64": 1e-12, "bfloat16": 1e-4}[dtype] + exact.abs() * (2.0 ** -8 if dtype == "bfloat16" else 0)
    for index in (torch.int32, torch.int64):
        got = runtime.embedding_adjoint(adjoint, tokens.to(index).to(gpu), rows)
        assert bool(((got.double().cpu() - exact).abs() <= allowed).all())
    assert torch.equal(got, runtime.embedding_adjoint(adjoint, tokens.to(gpu), rows))


def test_embedding_gradients_past_32_bits(gpu):
    """Adjoints and tables of more than 2^31 values: the last rows are the last ones."""
    import torch

    from ye3t_amd import runtime

    flush("embedding gradients of more than 2^31 values")
    rows, width = 4_200_003, 512
    tail = normal((3, width), "bfloat16", 1, gpu)
    adjoint = torch.zeros((rows, width), dtype=torch.bfloat16, device=gpu)
    adjoint[-3:] = tail
    tokens = torch.zeros(rows, dtype=torch.int32, device=gpu)
    tokens[-3:] = torch.tensor([5, 6, 5], device=gpu)
    grad = runtime.embedding_adjoint(adjoint, tokens, 7)
    assert torch.equal(grad[6], tail[1]) and not grad[:5].any()
    assert torch.equal(grad[5], (tail[0].float() + tail[2].float()).bfloat16())
    del adjoint
    flush("  tables of more than 2^31 values")
    tokens = torch.tensor([rows - 1, 0, rows - 3], device=gpu)
    grad = runtime.embedding_adjoint(tail, tokens, rows)
    assert torch.equal(grad[tokens], tail) and int((grad != 0).any(1).sum()) == 3
