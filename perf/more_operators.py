"""Performance cases of the products with learned weights on atoms' rows and of
dropout.

  linear         residual + dropout(activation(x W + b))
  linear_train   the same and the gradients of x, W and b
  species        the same with the weights of each atom's species
  species_train  and the gradients
  dropout        residual + dropout(x)
  dropout_train  and the gradient of x

Where ``own`` is false ``run`` computes the operators from elementary Torch
operations in 32 bits, rounded once at the end; where it is true it calls
``ye3t_amd.runtime``.  ``listed()`` holds the sizes that are tracked,
``draw(rng)`` gives more of the same ranges, ``prepare``/``run`` make and run
one, ``work`` counts what a pass cannot do without, and ``exact`` computes the
outputs in 64 bits.

A value in column c of row r is dropped where sixteen bits of Philox 4x32-10
(key: the seed; counter: c / 8, the layer, r; halves in ascending order) are
below the probability times 65536.
"""

import math

import torch

own = False

REAL = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
LAYER = 3  # number of the layer that a mask belongs to: any


def listed():
    return [
        # one moved atom through a wide layer: every weight is read for one row
        {"name": "linear-one-atom", "kind": "linear", "dtype": "bf16", "rows": 1, "inputs": 1024, "outputs": 4096,
         "activation": "silu", "bias": True, "residual": False, "drop": 0.0, "turned": False},
        # a small structure's atoms in single precision, weights kept as [out, in]
        {"name": "linear-few-atoms", "kind": "linear", "dtype": "f32", "rows": 37, "inputs": 2048, "outputs": 1024,
         "activation": "none", "bias": True, "residual": True, "drop": 0.0, "turned": True},
        # the message couplings' 161 columns to a layer of 96: no multiple of anything, many rows
        {"name": "linear-features", "kind": "linear", "dtype": "f32", "rows": 200003, "inputs": 161, "outputs": 96,
         "activation": "gelu", "bias": True, "residual": False, "drop": 0.0, "turned": False},
        # a wide layer over a large batch, its output dropped and added to the rows
        {"name": "linear-batch", "kind": "linear", "dtype": "bf16", "rows": 65536, "inputs": 2048, "outputs": 2048,
         "activation": "none", "bias": True, "residual": True, "drop": 0.1, "turned": False},
        # the widening half of a feed-forward layer in mixed-precision training
        {"name": "linear-train", "kind": "linear_train", "dtype": "bf16", "rows": 16384, "inputs": 1024,
         "outputs": 4096, "activation": "gelu", "bias": True, "residual": False, "drop": 0.0, "turned": False},
        # the first product after the features, training in single precision: 1449 columns, two of three dimensions odd
        {"name": "linear-train-features", "kind": "linear_train", "dtype": "f32", "rows": 20001, "inputs": 1449,
         "outputs": 256, "activation": "silu", "bias": True, "residual": False, "drop": 0.1, "turned": False},
        # a molecule's atoms by the weights of their species: latency
        {"name": "species-molecule", "kind": "species", "dtype": "f32", "rows": 21, "species": 4, "inputs": 128,
         "outputs": 128, "activation": "none", "bias": True, "residual": True, "drop": 0.0, "turned": False},
        # a batch of structures of eight species, evaluation
        {"name": "species-batch", "kind": "species", "dtype": "bf16", "rows": 40000, "species": 8, "inputs": 512,
         "outputs": 1024, "activation": "silu", "bias": True, "residual": False, "drop": 0.0, "turned": False},
        # a universal potential: 89 species, most of them rare, trained in single precision
        {"name": "species-train-89", "kind": "species_train", "dtype": "f32", "rows": 30011, "species": 89,
         "inputs": 128, "outputs": 128, "activation": "silu", "bias": True, "residual": True, "drop": 0.0,
         "turned": False},
        # the narrowing half of a feed-forward layer by species, mixed precision, dropped and added to the rows
        {"name": "species-train", "kind": "species_train", "dtype": "bf16", "rows": 16384, "species": 8,
         "inputs": 2048, "outputs": 1024, "activation": "none", "bias": True, "residual": True, "drop": 0.1,
         "turned": False},
        # one small structure's rows: launch latency
        {"name": "dropout-structure", "kind": "dropout", "dtype": "f32", "rows": 64, "width": 256, "residual": True,
         "drop": 0.1},
        # a training step's rows, odd width: the mask is made twice and never stored
        {"name": "dropout-train", "kind": "dropout_train", "dtype": "bf16", "rows": 200000, "width": 513,
         "residual": True, "drop": 0.2},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _drawn(rng):
    kind = rng.choice(["linear", "linear_train", "species", "species_train", "dropout", "dropout_train"])
    c = {"kind": kind, "dtype": rng.choice(["f32", "bf16"]), "rows": _log(rng, 1, 200000)}
    if kind.startswith("dropout"):
        return c | {"width": _log(rng, 1, 4096), "residual": rng.random() < 0.5, "drop": rng.choice([0.05, 0.1, 0.3, 0.5])}
    if kind.startswith("species"):
        c["species"] = _log(rng, 1, 100)
    return c | {"inputs": _log(rng, 1, 4096), "outputs": _log(rng, 1, 4096),
                "activation": rng.choice(["none", "relu", "silu", "gelu"]), "bias": rng.random() < 0.7,
                "residual": rng.random() < 0.4, "drop": rng.choice([0.0, 0.0, 0.1, 0.4]), "turned": rng.random() < 0.3}


def draw(rng):
    """A case of the ranges above that costs no more than the largest listed one, in traffic and in operations."""
    while True:
        c = _drawn(rng)
        w = work(c)
        if w["bytes"] <= 1e9 and w["flops"] <= (1.2e11 if c["dtype"] == "f32" else 5.4e11):
            return c


# ---- what a case needs -------------------------------------------------------

def work(case):
    """Bytes and operations of one pass, each input read once and each output written once."""
    s, n, train = SIZE[case["dtype"]], case["rows"], case["kind"].endswith("_train")
    if case["kind"].startswith("dropout"):
        w = case["width"]
        return {"bytes": n * w * s * (2 + case["residual"] + 2 * train), "flops": n * w * (2 + train)}
    a, b, groups = case["inputs"], case["outputs"], case.get("species", 1)
    used = min(groups, n)
    parameters = a * b + b * case["bias"]
    read = n * a * s + used * parameters * s + n * b * s * case["residual"] + (4 * n if "species" in case else 0)
    if not train:
        return {"bytes": read + n * b * s, "flops": 2 * n * a * b}
    held = n * b * s * (case["activation"] != "none")  # written by the forward and read by the gradient
    back = n * a * s + n * b * s + used * a * b * s + n * a * s + groups * parameters * s
    return {"bytes": read + n * b * s + 2 * held + back, "flops": 6 * n * a * b}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype, n = REAL[case["dtype"]], case["rows"]

    def normal(*shape, sd=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * sd).to(dtype)

    state = dict(case) | {"seed": int(seed) * 7919 + 11, "layer": LAYER}
    if case["kind"].startswith("dropout"):
        w = case["width"]
        return state | {"x": normal(n, w), "rows_before": normal(n, w, sd=2.0) if case["residual"] else None,
                        "adjoint": normal(n, w) if case["kind"] == "dropout_train" else None}
    a, b, groups = case["inputs"], case["outputs"], case.get("species", 0)
    lead = (groups,) if groups else ()
    if case["turned"]:
        weight = normal(*lead, b, a, sd=1.0 / math.sqrt(a)).transpose(-1, -2)
    else:
        weight = normal(*lead, a, b, sd=1.0 / math.sqrt(a))
    state |= {"x": normal(n, a), "weight": weight, "offset": normal(*lead, b, sd=0.3) if case["bias"] else None,
              "rows_before": normal(n, b, sd=2.0) if case["residual"] else None,
              "adjoint": normal(n, b) if case["kind"].endswith("_train") else None}
    if groups:
        # frequencies fall with the species' number; atoms come in the structures' order, not the species'
        u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
        state["ids"] = (torch.exp(u * math.log(groups + 1.0)) - 1.0).to(torch.int32).clamp_(0, groups - 1)
    return state


# ---- the plain forms ---------------------------------------------------------

def _plain_kept(s, columns):
    """[rows, columns]: what values are multiplied by, 0 where they are dropped."""
    n, low = s["rows"], 0xFFFFFFFF
    below = int(math.floor(s["drop"] * 65536.0 + 0.5))
    row = torch.arange(n, device="cuda")[:, None]
    chunk = torch.arange(-(-columns // 8), device="cuda")[None]
    c0, c1, c2, c3 = torch.broadcast_tensors(chunk, torch.full_like(row, s["layer"]), row & low, row >> 32)
    k0, k1 = s["seed"] & low, s["seed"] >> 32 & low
    for _ in range(10):
        p, q = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (q >> 32 & low) ^ c1 ^ k0, q & low, (p >> 32 & low) ^ c3 ^ k1, p & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack((c0, c1, c2, c3), -1)
    halves = torch.stack((words & 0xFFFF, words >> 16), -1).reshape(n, -1)[:, :columns]
    return (halves >= below).float() * (65536.0 / (65536.0 - below))


def _plain_activation(name, z):
    if name == "relu":
        return z.clamp(min=0.0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z


def _plain_slope(name, z):
    if name == "relu":
        return (z > 0).float()
    if name == "silu":
        e = torch.sigmoid(z)
        return e * (1.0 + z * (1.0 - e))
    return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * math.sqrt(0.5 / math.pi)


def _plain_order(s):
    """Rows in their species' order, and where each species begins."""
    ids = s["ids"].long()
    order = torch.argsort(ids, stable=True)
    return order, [0] + torch.bincount(ids, minlength=s["species"]).cumsum(0).tolist()


def _plain_product(s, x, weight, order, ends):
    """x times the weight of each row's species: one product for each species that occurs."""
    if order is None:
        return x @ weight
    out = torch.empty((x.shape[0], weight.shape[-1]), device="cuda")
    for k in range(s["species"]):
        if ends[k] < ends[k + 1]:
            rows = order[ends[k]:ends[k + 1]]
            out[rows] = x[rows] @ weight[k]
    return out


def _plain_linear(s):
    dtype, x, weight = s["x"].dtype, s["x"].float(), s["weight"].float()
    order, ends = _plain_order(s) if "species" in s else (None, None)
    z = _plain_product(s, x, weight, order, ends)
    if s["offset"] is not None:
        z = z + (s["offset"].float()[s["ids"].long()] if "species" in s else s["offset"].float())
    y = _plain_activation(s["activation"], z)
    kept = _plain_kept(s, s["outputs"]) if s["drop"] > 0 else None
    if kept is not None:
        y = y * kept
    if s["rows_before"] is not None:
        y = y + s["rows_before"].float()
    out = {"y": y.to(dtype)}
    if s["adjoint"] is None:
        return out
    dz = s["adjoint"].float()
    if kept is not None:
        dz = dz * kept
    if s["activation"] != "none":
        out["z"] = z.to(dtype)
        dz = dz * _plain_slope(s["activation"], out["z"].float())  # the gradient at what the program keeps
    out["x_adjoint"] = _plain_product(s, dz, weight.transpose(-1, -2), order, ends).to(dtype)
    if order is None:
        out["weight_adjoint"] = (x.transpose(0, 1) @ dz).to(dtype)
        if s["offset"] is not None:
            out["offset_adjoint"] = dz.sum(0).to(dtype)
        return out
    dw = torch.zeros(weight.shape, device="cuda")
    for k in range(s["species"]):
        rows = order[ends[k]:ends[k + 1]]
        dw[k] = x[rows].transpose(0, 1) @ dz[rows]
    out["weight_adjoint"] = dw.to(dtype)
    if s["offset"] is not None:
        out["offset_adjoint"] = torch.zeros_like(s["offset"], dtype=torch.float32).index_add_(0, s["ids"].long(), dz).to(dtype)
    return out


def _plain_dropout(s):
    dtype, kept = s["x"].dtype, _plain_kept(s, s["width"])
    y = s["x"].float() * kept
    if s["rows_before"] is not None:
        y = y + s["rows_before"].float()
    out = {"y": y.to(dtype)}
    if s["adjoint"] is not None:
        out["x_adjoint"] = (s["adjoint"].float() * kept).to(dtype)
    return out


# ---- this framework's operators ----------------------------------------------

def _own(s):
    from ye3t_amd import runtime

    if s["kind"].startswith("dropout"):
        out = {"y": runtime.dropout(s["x"], s["drop"], s["seed"], layer=s["layer"], residual=s["rows_before"])}
        if s["adjoint"] is not None:
            out["x_adjoint"] = runtime.dropout_adjoint(s["adjoint"], s["drop"], s["seed"], layer=s["layer"])
        return out
    shape = {"activation": None if s["activation"] == "none" else s["activation"]}
    if s["drop"] > 0:
        shape |= {"dropout": s["drop"], "seed": s["seed"], "layer": s["layer"]}
    if "species" in s:
        # the species of a program's data are checked once, where the data is loaded
        groups = (runtime.species_groups(s["ids"], s["species"], validate=False),)
        forward, backward = runtime.species_linear, runtime.species_linear_adjoint
    else:
        groups, forward, backward = (), runtime.linear, runtime.linear_adjoint
    keep = s["adjoint"] is not None and s["activation"] != "none"
    y = forward(s["x"], s["weight"], *groups, s["offset"], residual=s["rows_before"], return_preactivation=keep, **shape)
    if s["adjoint"] is None:
        return {"y": y}
    y, z = y if keep else (y, None)
    dx, dw, db = backward(s["adjoint"], s["x"], s["weight"], *groups, preactivation=z, bias=s["offset"] is not None, **shape)
    out = {"y": y} | ({"z": z} if keep else {}) | {"x_adjoint": dx, "weight_adjoint": dw}
    return out | ({"offset_adjoint": db} if db is not None else {})


def run(state):
    if own:
        return _own(state)
    return _plain_dropout(state) if state["kind"].startswith("dropout") else _plain_linear(state)


# ---- in 64 bits --------------------------------------------------------------

def _exact_kept(s, columns):
    """The generator with its 32-bit products in halves of sixteen bits."""
    def both(a, m):  # high and low word of a m
        cross = [(a & 0xFFFF) * (m & 0xFFFF), (a >> 16) * (m & 0xFFFF), (a & 0xFFFF) * (m >> 16), (a >> 16) * (m >> 16)]
        middle = (cross[0] >> 16) + (cross[1] & 0xFFFF) + (cross[2] & 0xFFFF)
        high = cross[3] + (cross[1] >> 16) + (cross[2] >> 16) + (middle >> 16)
        return high, (middle & 0xFFFF) << 16 | cross[0] & 0xFFFF

    chunks = -(-columns // 8)
    at = torch.arange(s["rows"] * chunks, device="cuda")
    row = torch.div(at, chunks, rounding_mode="floor")
    c = [at - row * chunks, torch.full_like(at, s["layer"]), row % 2 ** 32, torch.div(row, 2 ** 32, rounding_mode="floor")]
    key = [s["seed"] % 2 ** 32, s["seed"] // 2 ** 32 % 2 ** 32]
    for k in range(10):
        h0, l0 = both(c[0], 0xD2511F53)
        h1, l1 = both(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ (key[0] + k * 0x9E3779B9) % 2 ** 32, l1, h0 ^ c[3] ^ (key[1] + k * 0xBB67AE85) % 2 ** 32, l0]
    bits = torch.empty((s["rows"], chunks, 8), dtype=torch.int64, device="cuda")
    for k, word in enumerate(c):
        bits[..., 2 * k] = (word % 65536).reshape(s["rows"], chunks)
        bits[..., 2 * k + 1] = torch.div(word, 65536, rounding_mode="floor").reshape(s["rows"], chunks)
    below = round(s["drop"] * 65536)
    keep = bits.reshape(s["rows"], 8 * chunks)[:, :columns] >= below
    return torch.where(keep, 65536.0 / (65536 - below), 0.0).double()


def exact(case, seed):
    s = prepare(case, seed)
    x, g = s["x"].double(), None if s["adjoint"] is None else s["adjoint"].double()
    before = 0.0 if s["rows_before"] is None else s["rows_before"].double()
    columns = s["width"] if case["kind"].startswith("dropout") else s["outputs"]
    kept = _exact_kept(s, columns) if s["drop"] > 0 else torch.ones((), dtype=torch.float64, device="cuda")
    if case["kind"].startswith("dropout"):
        return {"y": before + x * kept} | ({} if g is None else {"x_adjoint": g * kept})
    w = s["weight"].double()
    w = w if w.ndim == 3 else w[None]
    groups = w.shape[0]
    ids = s["ids"].long() if "ids" in s else torch.zeros(s["rows"], dtype=torch.int64, device="cuda")
    members = [torch.nonzero(ids == k)[:, 0] for k in range(groups)]
    z = torch.zeros((s["rows"], columns), dtype=torch.float64, device="cuda")
    for k, rows in enumerate(members):
        z[rows] = torch.mm(x[rows], w[k])
    if s["offset"] is not None:
        z += s["offset"].double().reshape(groups, columns).index_select(0, ids)
    normal = lambda v: torch.special.ndtr(v)  # noqa: E731
    value = {"none": lambda v: v, "relu": lambda v: torch.where(v > 0, v, torch.zeros_like(v)),
             "silu": lambda v: v / (1.0 + torch.exp(-v)), "gelu": lambda v: v * normal(v)}[s["activation"]]
    result = {"y": before + kept * value(z)}
    if g is None:
        return result
    dz = g * kept
    if s["activation"] != "none":
        result["z"] = z
        logistic = 1.0 / (1.0 + torch.exp(-z))
        dz = dz * {"relu": lambda: torch.heaviside(z, torch.zeros_like(z)),
                   "silu": lambda: logistic + z * logistic * (1.0 - logistic),
                   "gelu": lambda: normal(z) + z * torch.exp(-z.square() / 2.0) / math.sqrt(2.0 * math.pi)}[s["activation"]]()
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros((groups, columns), dtype=torch.float64, device="cuda")
    for k, rows in enumerate(members):
        dx[rows] = torch.mm(dz[rows], w[k].t())
        dw[k] = torch.mm(x[rows].t(), dz[rows])
        db[k] = dz[rows].sum(0)
    result |= {"x_adjoint": dx, "weight_adjoint": dw.reshape(s["weight"].shape)}
    return result | ({} if s["offset"] is None else {"offset_adjoint": db.reshape(s["offset"].shape)})
