"""Attention and its gradients from the formulas in 64 bits, with the size of the terms of every sum (not collected).

A result that is a sum of terms t is held to an error of tolerance x sum |t|, element by element, so that nothing is
hidden where the terms cancel or where all of a result is small.  Two sizes: ``near`` takes the sums over the width
(go . v and D) at their values, ``wide`` at the sums of their terms' magnitudes.

float32 calls are held to 2e-5 of ``wide``: sums of at most a few thousand terms, exponentials of scores below 60
(60 x 2^-24) and logarithms of the same size.  bfloat16 calls round the weights p, or the gradients ds of the scores,
once for the matrix instruction and the result once, at most 2^-8 relative each (eight bits): 2 x 2^-8 of ``near``, and
float32's part.  Gradients to slopes and positions are sums in float32 in both types.
"""

import torch

FLOAT32, BFLOAT16 = 2e-5, 2 * 2.0 ** -8


def tolerance(dtype, near, wide):
    return FLOAT32 * wide + (BFLOAT16 * near if dtype == "bfloat16" else 0.0)


def attention(q, k, v, offsets, g, key_offsets=None, scale=None, cap=0.0, slopes=None, positions=None,
              key_positions=None, key_mask=None):
    """name: (value, near, wide) of out, q, k, v, slopes, positions and key_positions (gradients for the adjoint g)."""
    d = lambda t: None if t is None else t.detach().double().cpu()  # noqa: E731
    q, k, v, g, slopes, positions, key_positions = (d(t) for t in (q, k, v, g, slopes, positions, key_positions))
    H, D = q.shape[1:]
    group = H // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    first = offsets.tolist()
    key_first = first if key_offsets is None else key_offsets.tolist()
    seen = torch.ones(len(k), dtype=torch.bool) if key_mask is None else key_mask.cpu()
    at = positions if key_positions is None else key_positions
    result = {n: [torch.zeros_like(t) for _ in range(3)] for n, t in
              (("out", q), ("q", q), ("k", k), ("v", v), ("slopes", slopes), ("positions", positions),
               ("key_positions", key_positions)) if t is not None}
    heads_first = lambda t: t.transpose(0, 1)  # noqa: E731
    groups = lambda t: t.reshape(-1, group, *t.shape[1:]).sum(1).transpose(0, 1)  # noqa: E731
    for b in range(len(first) - 1):
        i, j = slice(first[b], first[b + 1]), slice(key_first[b], key_first[b + 1])
        if not bool(seen[j].any()):
            continue  # zeros
        live = seen[j].double()
        # what hidden keys hold is not used
        kk, vv = (torch.where(seen[j][:, None, None], t[j], torch.zeros_like(t[j])) for t in (k, v))
        kk, vv = (heads_first(t).repeat_interleave(group, 0) for t in (kk, vv))
        a, go = heads_first(q[i]), heads_first(g[i])
        raw = scale * (a @ kk.mT)
        bend = torch.tanh(raw / cap) if cap > 0 else torch.zeros_like(raw)
        z = cap * bend if cap > 0 else raw
        if slopes is not None:
            apart = positions[i, None] - torch.where(seen[j][:, None], at[j], torch.zeros_like(at[j]))[None]
            square = apart.square().sum(-1)
            square = torch.where(square < 2.0 ** -126, torch.zeros_like(square), square)  # one place
            far = square.sqrt()
            unit = torch.where(far[..., None] > 0, apart / far.clamp(min=1e-300)[..., None], torch.zeros_like(apart))
            z = z - slopes[:, None, None] * far
        p = torch.softmax(z.masked_fill(~seen[j], -torch.inf), -1)
        dp = (go @ vv.mT) * live
        wide_dp = (go.abs() @ vv.abs().mT) * live
        drawn = (p * dp).sum(-1, keepdim=True)
        dz = p * (dp - drawn)
        near = p * (dp.abs() + drawn.abs())
        wide = p * (wide_dp + (p * wide_dp).sum(-1, keepdim=True))
        ds = scale * dz * (1 - bend.square())
        for n, x, y in (("out", p @ vv, p @ vv.abs()),):
            for slot, t in zip(result[n], (x, y, y)):
                slot[i] = heads_first(t)
        for slot, t, m in zip(result["q"], (ds, abs(scale) * near, abs(scale) * wide), (kk, kk.abs(), kk.abs())):
            slot[i] = heads_first(t @ m)
        for slot, t, m in zip(result["k"], (ds, abs(scale) * near, abs(scale) * wide), (a, a.abs(), a.abs())):
            slot[j] = groups(t.mT @ m)
        for slot, m in zip(result["v"], (go, go.abs(), go.abs())):
            slot[j] = groups(p.mT @ m)
        if slopes is None:
            continue
        for slot, t in zip(result["slopes"], (-dz, near, wide)):
            slot += (t * far).sum((1, 2))
        for n, t, u in ((0, -dz, unit), (1, near, unit.abs()), (2, wide, unit.abs())):
            pull = torch.einsum("hij,h->ij", t, slopes if n == 0 else slopes.abs())[..., None] * u
            result["positions"][n][i] += pull.sum(1)
            keys = result["positions" if key_positions is None else "key_positions"][n]
            keys[j] += -pull.sum(0) if n == 0 else pull.sum(0)
    return result


def check(name, got, exact, dtype):
    """``got`` against (value, near, wide) of :func:`attention`; True-valued where a sum has no terms at all."""
    want, near, wide = exact
    got = got.detach().double().cpu()
    assert got.shape == want.shape, name
    if not got.numel():
        return
    assert torch.isfinite(got).all(), name
    low = name not in ("slopes", "positions", "key_positions")
    allowed = tolerance(dtype if low else "float32", near, wide)
    off = (got - want).abs()
    worst = float((off / allowed.clamp(min=1e-30)).max())
    print(f"  {name}: error {worst:.3f} of what is allowed", flush=True)
    assert bool((off <= allowed + 1e-30).all()), f"{name}: {worst:.3f} times what is allowed"
