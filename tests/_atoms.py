"""Plain 64-bit forms of the operators around the features (not collected)."""

import math

import torch


def rms_norm(x, weight, residual, epsilon):
    h = x.double() + (0 if residual is None else residual.double())
    return h * weight.double() / (h.square().mean(-1, keepdim=True) + epsilon).sqrt(), h


def e4m3(v):
    """Nearest value of the 8-bit format with four exponent and three mantissa bits, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def attention(q, k, v, offsets, key_offsets=None, scale=None, cap=0.0, slopes=None, positions=None,
              key_positions=None, key_mask=None):
    """Structure by structure; differentiable, so that autograd gives the gradients of the formula."""
    q, k, v = q.double(), k.double(), v.double()
    N, H, D = q.shape
    group = H // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    o = offsets.tolist()
    ko = o if key_offsets is None else key_offsets.tolist()
    kp = positions if key_positions is None else key_positions
    out, sums = [], []
    for b in range(len(o) - 1):
        i, j = slice(o[b], o[b + 1]), slice(ko[b], ko[b + 1])
        visible = torch.ones(ko[b + 1] - ko[b], dtype=torch.bool) if key_mask is None else key_mask[j]
        kk, vv = (t[j][visible].repeat_interleave(group, 1).transpose(0, 1) for t in (k, v))
        s = scale * (q[i].transpose(0, 1) @ kk.transpose(1, 2))
        if cap > 0:
            s = cap * torch.tanh(s / cap)
        if slopes is not None:
            apart = positions.double()[i, None] - kp.double()[j][visible][None]
            square = apart.square().sum(-1)
            # no gradient where two atoms meet
            far = torch.where(square > 0, square, torch.ones_like(square)).sqrt() * (square > 0)
            s = s - slopes.double()[:, None, None] * far
        if s.shape[-1] == 0:
            out.append(torch.zeros(s.shape[1], H, D, dtype=torch.float64))
            sums.append(torch.full((s.shape[1], H), -math.inf, dtype=torch.float64))
            continue
        out.append((torch.softmax(s, -1) @ vv).transpose(0, 1))
        sums.append(torch.logsumexp(s, -1).transpose(0, 1))
    return torch.cat(out) if out else torch.zeros(0, H, D, dtype=torch.float64), torch.cat(sums) if sums else None
