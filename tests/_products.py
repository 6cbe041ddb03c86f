"""Products with learned weights and dropout in 64 bits, with the size of the terms of every sum (not collected).

A result that is a sum of products is held to an error of tolerance x (sum of the products' magnitudes), value by value,
so that nothing is hidden where the terms cancel.  Each name maps to (value, rounded, wide):

* ``wide``: the magnitudes of what float32 sums up.  Sums of at most a few thousand products in float32, whose factors
  are good to 2^-24 (three parts of eight bits and more, terms below 2^-26 left out), exponentials good to a few 2^-22 and the
  normal integral to 2e-7: 2e-5 of ``wide``, what this package holds float32 to.  An activation's slope is at most 1.13
  (gelu at sqrt 2), so a sum's error reaches its output at most 1.13 times.
* ``rounded``: the magnitudes that are rounded to bfloat16 on the way, 2^-8 of each: the result once, and the gradient
  behind the product before it is multiplied.  In float32 the same roundings are 2^-24 and covered by ``wide``.
"""

import math

import numpy as np
import torch

FLOAT32, BFLOAT16 = 2e-5, 2.0 ** -8


def philox(counter, key):
    """Philox 4x32-10 of uint64 arrays holding 32-bit words: four arrays of words."""
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k = [int(v) for v in key]
    low = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), q & low, (p >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return c


def kept(rows, columns, probability, seed, layer, first=0):
    """[rows, columns]: 0 for dropped values, 1 / (1 - p) for the others, p in steps of 2^-16; rows from ``first`` on."""
    below = int(math.floor(probability * 65536 + 0.5))
    chunks = -(-columns // 8)
    row, chunk = (a.reshape(-1).astype(np.uint64) for a in np.meshgrid(np.arange(first, first + rows), np.arange(chunks), indexing="ij"))
    words = philox((chunk, np.full_like(chunk, layer), row & np.uint64(0xFFFFFFFF), row >> np.uint64(32)),
                   (seed % 2 ** 32, seed % 2 ** 64 >> 32))
    halves = np.stack([h for w in words for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], -1)
    halves = halves.reshape(rows, chunks * 8)[:, :columns].astype(np.int64)
    scale = 65536.0 / (65536 - below) if below < 65536 else 0.0
    return torch.from_numpy(np.where(halves < below, 0.0, scale)).reshape(rows, columns)


def phi(z):
    return 0.5 * torch.erfc(-z * math.sqrt(0.5))


def activated(name, z):
    return {None: lambda: z, "relu": lambda: z.clamp(min=0.0), "silu": lambda: z / (1.0 + torch.exp(-z)),
            "gelu": lambda: z * phi(z)}[name]()


def slope(name, z):
    s = 1.0 / (1.0 + torch.exp(-z))
    return {None: lambda: torch.ones_like(z), "relu": lambda: (z > 0).double(), "silu": lambda: s + z * s * (1.0 - s),
            "gelu": lambda: phi(z) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)}[name]()


def slope_size(name, z):
    """The magnitudes of a slope's terms.  silu's s + z s (1 - s) vanishes at z = -1.28 and gelu's phi + z bell at -0.75,
    where the terms cancel: each is good to a few 2^-24 of itself, so the slope is good to that share of their
    sum and not of its own value.  The gradient behind the product is so too, and what is summed of it."""
    s = 1.0 / (1.0 + torch.exp(-z))
    return {None: lambda: torch.ones_like(z), "relu": lambda: (z > 0).double(), "silu": lambda: s + z.abs() * s * (1.0 - s),
            "gelu": lambda: phi(z) + z.abs() * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)}[name]()


def d(t):
    return None if t is None else t.detach().double().cpu()


def members(species, count, rows):
    """The rows of each weight; species None: one weight for all."""
    if species is None:
        return [torch.arange(rows)]
    return [torch.nonzero(species.cpu().long() == k)[:, 0] for k in range(count)]


def forward(x, weight, bias, residual, species=None, activation=None, keep=None):
    """out and preactivation."""
    x, w, bias, residual = d(x), d(weight), d(bias), d(residual)
    w = w if species is not None else w[None]
    bias = None if bias is None else bias.reshape(len(w), w.shape[-1])
    z = torch.zeros(len(x), w.shape[-1], dtype=torch.float64)
    wide = torch.zeros_like(z)
    for k, rows in enumerate(members(species, len(w), len(x))):
        z[rows], wide[rows] = x[rows] @ w[k], x[rows].abs() @ w[k].abs()
        if bias is not None:
            z[rows] += bias[k]
            wide[rows] += bias[k].abs()
    y = activated(activation, z)
    far = 1.13 * wide + y.abs()
    if keep is not None:
        y, far = y * keep, far * keep
    if residual is not None:
        y, far = y + residual, far + residual.abs()
    return {"out": (y, y.abs(), far), "preactivation": (z, z.abs(), wide)}


def backward(g, x, weight, preactivation, species=None, activation=None, keep=None):
    """input, weight and bias gradients at the given (rounded) preactivation."""
    g, x, w, z = d(g), d(x), d(weight), d(preactivation)
    shape = w.shape
    w = w if species is not None else w[None]
    dz = g if keep is None else g * keep
    size = dz.abs()
    if activation is not None:
        dz, size = dz * slope(activation, z), size * slope_size(activation, z)
    shaped = activation is not None or keep is not None
    out = {n: [torch.zeros(s, dtype=torch.float64) for _ in range(3)]
           for n, s in (("input", x.shape), ("weight", w.shape), ("bias", (len(w), w.shape[-1])))}
    for k, rows in enumerate(members(species, len(w), len(x))):
        a, b = x[rows], dz[rows]
        for n, at, value in (("input", rows, lambda v, m: v @ m(w[k]).T), ("weight", k, lambda v, m: m(a).T @ v),
                             ("bias", k, lambda v, m: v.sum(0))):
            exact, near, wide = value(b, lambda t: t), value(b.abs(), torch.abs), value(size[rows], torch.abs)
            for slot, t in zip(out[n], (exact, exact.abs() + (near if shaped else 0.0), wide)):
                slot[at] = t
    lead = shape[:-2]
    return {"input": tuple(out["input"]), "weight": tuple(t.reshape(shape) for t in out["weight"]),
            "bias": tuple(t.reshape(*lead, shape[-1]) for t in out["bias"])}


def check(name, got, exact, dtype):
    want, rounded, wide = exact
    got = d(got)
    assert got.shape == want.shape, name
    if not got.numel():
        return
    assert torch.isfinite(got).all(), name
    allowed = FLOAT32 * wide + (BFLOAT16 * rounded if dtype == "bfloat16" else 0.0) + 1e-37
    off = (got - want).abs()
    worst = float((off / allowed).max())
    print(f"  {name}: error {worst:.3f} of what is allowed", flush=True)
    assert worst <= 1.0, f"{name}: {worst:.3f} times what is allowed"
