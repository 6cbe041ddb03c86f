"""Operators of a model's own layers around the ACE features: a learned vector
for each species, the root-mean-square norm of feature rows, and attention
among the atoms of each structure.

Atoms are packed one structure after the other, with the row offsets of the
density's CSR (int64, from 0 to the atom count) for the structures.  Storage is
float32 or bfloat16 (the embedding also float64, for double-precision
densities); means, softmax statistics and sums are held in 32 bits or more.
bfloat16 attention rounds the softmax weights, and in the gradient the
gradients of the scores, to bfloat16 for the matrix instructions.  The forward operators are differentiable once; each has its adjoint as a
function of its own.  No reference counterparts.
"""

import torch

from ye3t_amd.runtime import _require_device, native

__all__ = ("embedding", "embedding_adjoint", "rms_norm", "rms_norm_8bit", "rms_norm_adjoint", "atom_attention",
           "atom_attention_adjoint")


def _tracked(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _require_one_device(name, first, *rest):
    """A call's kernels run on the device of its first tensor, and read no other one's memory."""
    _require_device(first, name)
    for t in rest:
        if t is not None:
            _require_device(t, name)
            if t.device != first.device:
                raise ValueError(f"{name}: tensors on {first.device} and {t.device}")


def _unit_rows(t):
    """``t``, or a contiguous copy where the last axis is not laid out value after value."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


# ---- embedding -----------------------------------------------------------------

def _check_tokens(tokens, rows, name):
    found = native.check_indices((tokens, 0, rows, False)) if tokens.is_cuda else None
    if found is not None:
        bad = found[0][2]
    else:
        bad = bool(tokens.numel()) and (int(tokens.min()) < 0 or int(tokens.max()) >= rows)
    if bad:
        raise RuntimeError(f"{name} token out of range [0, {rows})")


def _tokens(tokens, rows, validate, name):
    if tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError("tokens must be int32 or int64")
    tokens = tokens.contiguous()
    if validate:
        _check_tokens(tokens, rows, name)
    return tokens


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, tokens, scale):
        ctx.save_for_backward(tokens)
        ctx.rows, ctx.scale = int(table.shape[0]), scale
        return native.embedding(tokens, table, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (tokens,) = ctx.saved_tensors
        return native.embedding_adjoint(grad.contiguous(), tokens, ctx.rows, ctx.scale), None, None


def embedding(tokens, table, *, scale=1.0, validate=True):
    """Rows of ``table [rows, width]`` by ``tokens`` (int32 or int64 of any
    shape), times ``scale``: ``[*tokens.shape, width]`` in the table's dtype
    (float32, float64 or bfloat16), the product rounded once.  For species
    vectors, for instance the ``node_features`` of :func:`ace_density`.

    Differentiable in ``table`` (:func:`embedding_adjoint`).  ``validate``
    range-checks the tokens first (one kernel and one wait); a caller that has
    checked them before may skip it.  A token outside the table that is not
    checked gives a row of zeros and no gradient."""
    _require_one_device("embedding", table, tokens)
    if table.ndim != 2:
        raise ValueError("table must be [rows, width]")
    tokens = _tokens(tokens, int(table.shape[0]), validate, "embedding")
    scale = float(scale)
    if _tracked(table):
        return _Embedding.apply(table, tokens, scale)
    return native.embedding(tokens, table, scale)


def embedding_adjoint(adjoint, tokens, rows, *, scale=1.0, validate=True):
    """Gradient ``[rows, width]`` of :func:`embedding` with respect to its table
    for the output's ``adjoint [*tokens.shape, width]``.

    The positions are sorted by token and summed in equal shares in a fixed
    order in float32 (float64 for float64): equal calls give equal bits, and a
    token that most rows share costs no more than any other."""
    _require_one_device("embedding_adjoint", adjoint, tokens)
    rows = int(rows)
    if rows < 0:
        raise ValueError("rows must be non-negative")
    if adjoint.ndim != tokens.ndim + 1 or tuple(adjoint.shape[:-1]) != tuple(tokens.shape):
        raise ValueError("adjoint must be [*tokens.shape, width]")
    tokens = _tokens(tokens, rows, validate, "embedding_adjoint")
    return native.embedding_adjoint(adjoint.contiguous(), tokens, rows, float(scale))


# ---- norm ----------------------------------------------------------------------

def _norm_rows(input, weight, name, **rows):
    """Checks ``input`` and ``weight``, and that the others (by their arguments' names) are like ``input``."""
    _require_one_device(name, input, weight, *rows.values())
    if input.ndim < 1 or weight.ndim != 1 or int(weight.shape[0]) != int(input.shape[-1]):
        raise ValueError("weight must be [width] with input [..., width]")
    if weight.dtype != input.dtype:
        raise ValueError(f"weight must have dtype {input.dtype}")
    for n, t in rows.items():
        if t is not None and (t.shape != input.shape or t.dtype != input.dtype):
            raise ValueError(f"{n} must have the input's shape and dtype")


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, weight, residual, epsilon):
        y, total = native.rms_norm(input, weight, residual, epsilon)
        ctx.save_for_backward(input if residual is None else total, weight)
        ctx.epsilon, ctx.added = epsilon, residual is not None
        ctx.set_materialize_grads(False)
        return (y, total) if residual is not None else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, total_grad=None):
        total, weight = ctx.saved_tensors
        if grad is None and total_grad is None:
            return None, None, None, None
        if grad is None:  # only the sum was used
            return total_grad, None, total_grad if ctx.added else None, None
        dx, dw = native.rms_norm_adjoint(grad.contiguous(), total, weight,
                                         None if total_grad is None else total_grad.contiguous(), ctx.epsilon)
        return dx, dw, dx if ctx.added else None, None


def rms_norm(input, weight, *, residual=None, epsilon=1e-6):
    """``y = h * weight / sqrt(mean(h^2) + epsilon)`` over the last axis, with
    ``h = input + residual``: returns ``y``, or ``(y, h)`` with a residual.

    float32 or bfloat16; the mean and ``y`` come from the unrounded sum in
    float32, ``y`` and ``h`` are rounded once each.  Differentiable
    (:func:`rms_norm_adjoint`); the gradient is taken at the rounded ``h``."""
    _norm_rows(input, weight, "rms_norm", residual=residual)
    epsilon = float(epsilon)
    input = input.contiguous()
    residual = None if residual is None else residual.contiguous()
    if _tracked(input, weight, residual):
        return _RMSNorm.apply(input, weight.contiguous(), residual, epsilon)
    y, total = native.rms_norm(input, weight.contiguous(), residual, epsilon)
    return y if residual is None else (y, total)


def rms_norm_adjoint(adjoint, total, weight, *, total_adjoint=None, epsilon=1e-6):
    """Gradients of :func:`rms_norm` at ``total`` (its ``h``, or its input where
    there was no residual) for the output's ``adjoint`` and the sum's
    ``total_adjoint``: ``(input_adjoint, weight_adjoint)``; the residual's is
    the input's.  The weight's sum over rows is float32 in a fixed order."""
    _norm_rows(total, weight, "rms_norm_adjoint", adjoint=adjoint, total_adjoint=total_adjoint)
    return native.rms_norm_adjoint(adjoint.contiguous(), total.contiguous(), weight.contiguous(),
                                   None if total_adjoint is None else total_adjoint.contiguous(), float(epsilon))


def rms_norm_8bit(input, weight, *, residual=None, epsilon=1e-6):
    """:func:`rms_norm` with its rows in 8 bits, for descriptors that are stored
    or handed to 8-bit products: ``(codes, scales)``, or ``(codes, scales, h)``
    with a residual.

    ``codes`` has the input's shape in ``torch.float8_e4m3fn``; ``scales
    [..., ceil(width / 128)]`` is float32, one for each 128 columns (the
    largest value over 448, 0 for columns of zeros), so that ``y`` is about
    ``codes * scales``.  Not differentiable."""
    _norm_rows(input, weight, "rms_norm_8bit", residual=residual)
    if _tracked(input, weight, residual):
        raise NotImplementedError("rms_norm_8bit: no gradient (use rms_norm)")
    codes, scales, total = native.rms_norm_8bit(input.contiguous(), weight.contiguous(),
                                                None if residual is None else residual.contiguous(), float(epsilon))
    return (codes, scales) if residual is None else (codes, scales, total)


# ---- attention -----------------------------------------------------------------

def _check_offsets(offsets, count, name):
    if offsets.dtype != torch.int64 or offsets.ndim != 1 or offsets.numel() < 1:
        raise ValueError(f"{name} must be int64 [structures + 1]")


def _validate_offsets(pairs):
    """The values of row offsets: one kernel and one wait, or reductions that name the fault."""
    found = native.check_indices(*((t, native.INT64_MIN, native.INT64_MAX, True) for t, _, _ in pairs))
    if found is not None and all(f[:2] == (0, n) and not f[3] for f, (_, n, _) in zip(found, pairs)):
        return
    for t, n, name in pairs:
        first, last = int(t[0]), int(t[-1])
        if first != 0 or last != n:
            raise ValueError(f"{name} must run from 0 to the atom count {n} (got {first} .. {last})")
        if bool((t[1:] < t[:-1]).any()):
            raise ValueError(f"{name} must be non-decreasing")


def _attention_problem(query, key, value, offsets, key_offsets, scale, cap, slopes, positions, key_positions,
                       key_mask, validate, name):
    """The checked arguments as ``native.Attention``."""
    _require_one_device(name, query, key, value, offsets, key_offsets, slopes, positions, key_positions, key_mask)
    if query.ndim != 3 or key.ndim != 3 or value.shape != key.shape or query.shape[2] != key.shape[2]:
        raise ValueError("query must be [atoms, heads, width], key and value [atoms, key_heads, width]")
    if query.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"unsupported dtype {query.dtype}; expected float32 or bfloat16")
    if key.dtype != query.dtype or value.dtype != query.dtype:
        raise ValueError("query, key and value must share one dtype")
    N, H, D = (int(x) for x in query.shape)
    M, HK = int(key.shape[0]), int(key.shape[1])
    if HK < 1 or H < 1 or H % HK:
        raise ValueError("heads must be a positive multiple of the key heads")
    if not 1 <= D <= 128:
        raise ValueError(f"head width {D} is outside 1 .. 128")
    _check_offsets(offsets, N, "offsets")
    if key_offsets is None:
        if M != N:
            raise ValueError("keys of other atoms than the queries' need key_offsets")
    else:
        _check_offsets(key_offsets, M, "key_offsets")
        if key_offsets.shape != offsets.shape:
            raise ValueError("offsets and key_offsets must name the same structures")
    if offsets.numel() < 2 and (N or M):
        raise ValueError("offsets must name the atoms' structures")
    cap = float(cap)
    if not 0.0 <= cap < float("inf"):
        raise ValueError("cap must be non-negative")
    if (slopes is None) != (positions is None):
        raise ValueError("slopes and positions come together")
    if slopes is None and key_positions is not None:
        raise ValueError("key_positions need slopes")
    if slopes is not None:
        if key_offsets is not None and key_positions is None:
            raise ValueError("keys of other atoms than the queries' need key_positions")
        for t, shape, n in ((slopes, (H,), "slopes"), (positions, (N, 3), "positions"),
                            (key_positions, (M, 3), "key_positions")):
            if t is not None and (tuple(t.shape) != shape or t.dtype != torch.float32):
                raise ValueError(f"{n} must be float32 {list(shape)}")
    if key_mask is not None and (key_mask.dtype != torch.bool or tuple(key_mask.shape) != (M,)):
        raise ValueError(f"key_mask must be bool [{M}]")
    offsets = offsets.contiguous()
    key_offsets = None if key_offsets is None else key_offsets.contiguous()
    if validate:
        pairs = [(offsets, N, "offsets")]
        if key_offsets is not None:
            pairs.append((key_offsets, M, "key_offsets"))
        _validate_offsets(pairs)
    whole = lambda t: None if t is None else t.contiguous()  # noqa: E731
    return native.Attention(_unit_rows(query), _unit_rows(key), _unit_rows(value), offsets, key_offsets,
                            float(D ** -0.5 if scale is None else scale), cap, whole(slopes), whole(positions),
                            whole(key_positions), whole(key_mask))


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, slopes, positions, key_positions, problem):
        # the problem holds these themselves, or contiguous copies where they were needed
        out, sums = problem.forward(True)
        ctx.save_for_backward(out, sums, *problem.tensors())
        ctx.problem = problem.rest()
        ctx.mark_non_differentiable(sums)
        return out, sums

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _):
        out, sums, *tensors = ctx.saved_tensors
        problem = native.Attention.of(tensors, ctx.problem)
        need = any(ctx.needs_input_grad[3:6])
        dq, dk, dv, ds, dp, dkp = problem.adjoint(grad.contiguous(), out, sums, need)
        return dq, dk, dv, ds, dp, dkp, None


def atom_attention(query, key, value, offsets, *, key_offsets=None, scale=None, cap=0.0, slopes=None, positions=None,
                   key_positions=None, key_mask=None, return_log_sums=False, validate=True):
    """Softmax attention of the atoms of each structure over that structure's atoms.

    ``query [N, H, D]``, ``key`` and ``value [M, HK, D]`` (float32 or bfloat16,
    any strides, D at most 128, HK a divisor of H: query head h reads key head
    ``h // (H // HK)``); ``offsets`` int64 ``[S + 1]``, the structures' row
    offsets.  Returns ``[N, H, D]``.

    * ``key_offsets``: the keys are other atoms than the queries, with row
      offsets of their own over the same structures (a few moved atoms against
      whole structures, for instance).
    * ``scale``: of the scores, ``D ** -0.5`` by default.
    * ``cap``: scores become ``cap * tanh(score / cap)``; 0: they stay as they are.
    * ``slopes [H]`` and ``positions [N, 3]`` (float32; ``key_positions [M, 3]``
      with ``key_offsets``): scores are lowered by ``slopes[h]`` times the
      distance of the two atoms, after the cap.  Atoms more than 1.8e19 apart do
      not see each other; atoms less than 1.1e-19 apart have no direction.
    * ``key_mask`` bool ``[M]``: False for atoms that no row sees (ghosts,
      padding); what they hold is not used for other atoms' rows.  A row that
      sees nothing gives zeros and has no gradient, whatever it holds.
    * ``return_log_sums``: also ``[N, H]`` float32, the logarithm of each row's
      sum of exponentials (-infinity for a row that sees nothing), which
      :func:`atom_attention_adjoint` takes.

    Differentiable in query, key, value, slopes and the positions.  ``validate``
    checks the offsets' values first (one kernel and one wait); with offsets
    that were not checked and do not run from 0 to the atom count without
    falling, no access leaves the arrays but the results are undefined."""
    problem = _attention_problem(query, key, value, offsets, key_offsets, scale, cap, slopes, positions,
                                 key_positions, key_mask, validate, "atom_attention")
    if _tracked(query, key, value, slopes, positions, key_positions):
        out, sums = _Attention.apply(query, key, value, slopes, positions, key_positions, problem)
    else:
        out, sums = problem.forward(return_log_sums)
    return (out, sums) if return_log_sums else out


def atom_attention_adjoint(adjoint, out, log_sums, query, key, value, offsets, *, key_offsets=None, scale=None,
                           cap=0.0, slopes=None, positions=None, key_positions=None, key_mask=None,
                           bias_gradients=False, validate=True):
    """Gradients of :func:`atom_attention` for the output's ``adjoint [N, H, D]``,
    from its output, its ``log_sums`` and the same arguments: ``(query, key,
    value, slopes, positions, key_positions)``.  The last three are None
    without ``bias_gradients``; without ``key_positions`` the gradient to
    positions holds both of an atom's parts and the last is None."""
    problem = _attention_problem(query, key, value, offsets, key_offsets, scale, cap, slopes, positions,
                                 key_positions, key_mask, validate, "atom_attention_adjoint")
    _require_one_device("atom_attention_adjoint", query, adjoint, out, log_sums)
    for t, n in ((adjoint, "adjoint"), (out, "out")):
        if t.shape != query.shape or t.dtype != query.dtype:
            raise ValueError(f"{n} must have the query's shape and dtype")
    if log_sums.dtype != torch.float32 or tuple(log_sums.shape) != tuple(query.shape[:2]):
        raise ValueError("log_sums must be float32 [atoms, heads]")
    if bias_gradients and slopes is None:
        raise ValueError("bias_gradients need slopes and positions")
    return problem.adjoint(adjoint.contiguous(), out.contiguous(), log_sums.contiguous(), bool(bias_gradients))
