"""Performance cases of the operators around the ACE features: the species
embedding, the root-mean-square norm of feature rows, and attention among the
atoms of a structure.

  embed        rows of a table by token (species), scaled
  embed_train  the same and the table's gradient
  norm8        a residual's addition, the norm, and its rows in 8 bits with
               one scale for each 128 columns
  norm_train   the addition and the norm, forward and gradient
  attend       attention of the atoms of each structure, forward
  attend_train the same, forward and gradients

Where ``own`` is false ``run`` computes the operators from elementary Torch
operations in 32 bits, rounded once at the end; where it is true it calls
``ye3t_amd.runtime``.  ``listed()`` holds the sizes that are tracked,
``draw(rng)`` gives more of the same ranges, ``prepare``/``run`` make and run
one, ``work`` counts what a pass cannot do without, and ``exact`` computes the
outputs in 64 bits.
"""

import math

import torch

own = False

REAL = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
EPSILON = 1e-6
GROUP = 128          # columns that share a scale of the 8-bit rows
LARGEST_8BIT = 448.0  # of the 8-bit format with four exponent and three mantissa bits


def listed():
    return [
        # the species vectors of one small structure: launch latency
        {"name": "embed-128", "kind": "embed", "dtype": "f32", "tokens": 128, "vocabulary": 8, "width": 16},
        # a training step's species vectors: every atom of a large batch, eight species, so one row of the table
        # gets the sum of tens of thousands of rows
        {"name": "embed-train-200000", "kind": "embed_train", "dtype": "f32", "tokens": 200000, "vocabulary": 8,
         "width": 128},
        # a large vocabulary (species with their environments' classes): most rows are met a few times or never
        {"name": "embed-train-vocabulary", "kind": "embed_train", "dtype": "bf16", "tokens": 16384,
         "vocabulary": 50021, "width": 1024},
        # the feature rows of every node and channel of the message couplings: 161 columns, no multiple of anything
        {"name": "norm-train-800000x161", "kind": "norm_train", "dtype": "f32", "rows": 800000, "width": 161},
        # wide rows in 16 bits, as between the layers of a model in training
        {"name": "norm-train-16384x2048", "kind": "norm_train", "dtype": "bf16", "rows": 16384, "width": 2048},
        # evaluation of few atoms, rows handed on in 8 bits: latency
        {"name": "norm8-37x4096", "kind": "norm8", "dtype": "bf16", "rows": 37, "width": 4096},
        # descriptors of a structure in 8 bits, for a store of descriptors
        {"name": "norm8-50000x1449", "kind": "norm8", "dtype": "f32", "rows": 50000, "width": 1449},
        # molecules: many short structures, forces wanted (gradients to slopes and positions)
        {"name": "attend-molecules", "kind": "attend_train", "dtype": "f32", "structures": 2000, "atoms": 21,
         "heads": 8, "key_heads": 8, "head_width": 32, "cap": 0.0, "bias": True, "mask": False, "forces": True},
        # crystals and cells of a few hundred atoms in mixed precision, scores capped, ghost atoms masked
        {"name": "attend-cells", "kind": "attend_train", "dtype": "bf16", "structures": 96, "atoms": 480,
         "heads": 8, "key_heads": 8, "head_width": 64, "cap": 30.0, "bias": True, "mask": True, "forces": False},
        # one large structure, key heads shared by four
        {"name": "attend-large", "kind": "attend_train", "dtype": "bf16", "structures": 1, "atoms": 8192,
         "heads": 16, "key_heads": 4, "head_width": 128, "cap": 0.0, "bias": False, "mask": False, "forces": False},
        # one moved atom in each of many structures against all their atoms
        {"name": "attend-one-atom", "kind": "attend", "dtype": "bf16", "structures": 24, "atoms": 9000,
         "queries": 1, "heads": 16, "key_heads": 4, "head_width": 128, "cap": 0.0, "bias": True, "mask": False},
        # structures of a thousand atoms in single precision, distance bias, evaluation
        {"name": "attend-structures", "kind": "attend", "dtype": "f32", "structures": 40, "atoms": 1000,
         "queries": 0, "heads": 8, "key_heads": 8, "head_width": 64, "cap": 0.0, "bias": True, "mask": True},
    ]


def _log(rng, low, high):
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return n - (n == 3072)


def _drawn(rng):
    kind = rng.choice(["embed", "embed_train", "norm8", "norm_train", "attend", "attend_train"])
    dtype = rng.choice(["f32", "bf16"])
    if kind.startswith("embed"):
        return {"kind": kind, "dtype": dtype, "tokens": _log(rng, 1, 400000), "vocabulary": _log(rng, 1, 100000),
                "width": _log(rng, 1, 2048)}
    if kind.startswith("norm"):
        return {"kind": kind, "dtype": dtype, "rows": _log(rng, 1, 400000), "width": _log(rng, 1, 8192)}
    heads = rng.choice([1, 2, 4, 8, 12, 16])
    # an atom alone has no gradient but that of its value, and rounding would be all there is to compare
    c = {"kind": kind, "dtype": dtype, "structures": _log(rng, 1, 2000), "heads": heads,
         "atoms": _log(rng, 8 if kind == "attend_train" else 1, 6000),
         "key_heads": rng.choice([k for k in (1, 2, 4, 8, 12, 16) if heads % k == 0]),
         "head_width": rng.choice([8, 16, 20, 32, 33, 40, 64, 80, 96, 128]), "cap": rng.choice([0.0, 0.0, 20.0, 50.0]),
         "bias": rng.random() < 0.6, "mask": rng.random() < 0.4}
    if kind == "attend":
        c["queries"] = rng.choice([0, 0, 1, 3])
    else:
        c["forces"] = bool(c["bias"] and dtype == "f32" and rng.random() < 0.7)
    return c


def draw(rng):
    """A case of the ranges above that costs no more than the largest listed one, in traffic, in operations and in
    the memory its plain form takes."""
    while True:
        c = _drawn(rng)
        w = work(c)
        if w["bytes"] > 3e9 or w["flops"] > 1e12:
            continue
        if "heads" in c:
            longest = 2 * c["atoms"]
            queries = c.get("queries") or longest
            rows = c["structures"] * longest
            if c["structures"] * c["heads"] * queries * longest > 1.2e9 or rows * c["heads"] * c["head_width"] > 4e8:
                continue
        return c


# ---- what a case needs -------------------------------------------------------

def _lengths(case):
    """Atoms of each structure: from half to one and a half times the mean."""
    n, mean = case["structures"], case["atoms"]
    if n == 1:
        return [mean]
    return [max(1, int(mean * (0.5 + ((k * 0.6180339887) % 1.0)))) for k in range(n)]


def work(case):
    """Bytes and operations of one pass, each input read once and each output written once."""
    kind, s = case["kind"], SIZE[case["dtype"]]
    if kind.startswith("embed"):
        n, v, w = case["tokens"], case["vocabulary"], case["width"]
        touched, ids = min(n, v), (4 if v <= 128 else 8) * n
        if kind == "embed":
            return {"bytes": ids + touched * w * s + n * w * s, "flops": n * w}
        return {"bytes": ids + touched * w * s + 2 * n * w * s + v * w * s, "flops": 2 * n * w}
    if kind.startswith("norm"):
        n, w = case["rows"], case["width"]
        if kind == "norm8":
            return {"bytes": n * w * (3 * s + 1) + n * -(-w // GROUP) * 4 + w * s, "flops": 5 * n * w}
        # x, r in, y, h out; h, both adjoints in, one adjoint out
        return {"bytes": 8 * n * w * s + 3 * w * s, "flops": 12 * n * w}
    lengths = _lengths(case)
    keys = sum(lengths)
    queries = case.get("queries", 0)
    rows = queries * len(lengths) if queries else keys
    pairs = sum((queries or n) * n for n in lengths)
    h, hk, d = case["heads"], case["key_heads"], case["head_width"]
    io = (2 * rows * h + 2 * keys * hk) * d * s + 8 * (len(lengths) + 1) + (12 * keys if case["bias"] else 0)
    if kind == "attend":
        return {"bytes": io, "flops": 4 * pairs * h * d}
    # the backward reads q, k, v, o and o's adjoint and writes three adjoints
    return {"bytes": io + (3 * rows * h + 2 * keys * hk) * d * s + (rows * h + 2 * keys * hk) * d * s,
            "flops": 14 * pairs * h * d}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def prepare(case, seed):
    g = _generator(seed)
    kind, dtype = case["kind"], REAL[case["dtype"]]

    def normal(*shape, sd=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * sd).to(dtype)

    state = dict(case)
    if kind.startswith("embed"):
        n, v, w = case["tokens"], case["vocabulary"], case["width"]
        # frequencies fall with the token's number, as those of species and of words do
        u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
        tokens = (torch.exp(u * math.log(v + 1.0)) - 1.0).to(torch.int64).clamp_(0, v - 1)
        state |= {"ids": tokens.to(torch.int32) if v <= 128 else tokens, "table": normal(v, w), "scale": math.sqrt(w),
                  "adjoint": normal(n, w) if kind == "embed_train" else None}
        return state
    if kind.startswith("norm"):
        n, w = case["rows"], case["width"]
        state |= {"x": normal(n, w), "residual": normal(n, w, sd=2.0), "weight": 1.0 + normal(w, sd=0.1)}
        if kind == "norm_train":
            state |= {"adjoint": normal(n, w), "total_adjoint": normal(n, w)}
        return state

    lengths = _lengths(case)
    b, keys, queries = len(lengths), sum(lengths), case.get("queries", 0)
    h, hk, d = case["heads"], case["key_heads"], case["head_width"]
    lens = torch.tensor(lengths, dtype=torch.int64)
    offsets = torch.zeros(b + 1, dtype=torch.int64)
    offsets[1:] = lens.cumsum(0)
    state |= {"offsets": offsets.cuda(), "longest": max(lengths), "scale": 1.0 / math.sqrt(d), "key_offsets": None,
              "key_positions": None, "key_mask": None, "slopes": None, "positions": None, "longest_query": max(lengths)}
    if queries:
        state["key_offsets"] = state["offsets"]
        state["offsets"] = (torch.arange(b + 1) * queries).cuda()
        state["longest_query"] = queries
        state["q"], state["k"], state["v"] = normal(b * queries, h, d, sd=1.5), normal(keys, hk, d), normal(keys, hk, d)
    elif h == hk:  # one projection gives all three: views of it
        qkv = normal(keys, 3, h, d, sd=1.2)
        state["q"], state["k"], state["v"] = qkv.unbind(1)
    else:
        state["q"], kv = normal(keys, h, d, sd=1.5), normal(keys, 2, hk, d)
        state["k"], state["v"] = kv.unbind(1)
    if case["bias"]:
        # atoms of a cell of about 20 cubic Angstrom each
        side = (20.0 * lens.double()).pow(1.0 / 3.0).float().cuda()
        owner = torch.repeat_interleave(torch.arange(b, device="cuda"), lens.cuda(), output_size=keys)
        at = torch.rand((keys, 3), generator=g, device="cuda") * side[owner, None]
        state["slopes"] = torch.exp2(torch.linspace(0.0, -5.0, h)).cuda()
        if queries:
            state["key_positions"] = at
            first = state["key_offsets"][:-1].repeat_interleave(queries)
            state["positions"] = at[first] + torch.randn((b * queries, 3), generator=g, device="cuda") * 0.3
        else:
            state["positions"] = at
    if case["mask"]:
        mask = torch.rand(keys, generator=g, device="cuda") < 0.9
        if b > 1:
            mask[int(offsets[-2]):] = False  # a structure of ghost atoms: its rows see nothing
        state["key_mask"] = mask
    if kind == "attend_train":
        state["adjoint"] = normal(keys, h, d)
    return state


# ---- the plain forms ---------------------------------------------------------

def _plain_embed(s):
    return {"rows": (s["table"].float()[s["ids"].long()] * s["scale"]).to(s["table"].dtype)}


def _plain_embed_train(s):
    out = _plain_embed(s)
    grad = torch.zeros(s["table"].shape, device="cuda")
    grad.index_add_(0, s["ids"].long(), s["adjoint"].float())
    return out | {"table_adjoint": (grad * s["scale"]).to(s["table"].dtype)}


def _plain_norm(s):
    total = s["x"].float() + s["residual"].float()
    inverse = torch.rsqrt(total.square().mean(-1, keepdim=True) + EPSILON)
    return total, total * inverse * s["weight"].float()


def _plain_norm8(s):
    total, y = _plain_norm(s)
    n, w = y.shape
    groups = -(-w // GROUP)
    padded = torch.nn.functional.pad(y, (0, groups * GROUP - w)).reshape(n, groups, GROUP)
    scales = padded.abs().amax(-1) / LARGEST_8BIT
    divisor = torch.where(scales > 0, scales, torch.ones_like(scales))
    codes = (padded / divisor[..., None]).clamp(-LARGEST_8BIT, LARGEST_8BIT).reshape(n, -1)[:, :w]
    return {"codes": codes.to(torch.float8_e4m3fn), "scales": scales, "total": total.to(s["x"].dtype)}


def _plain_norm_train(s):
    dtype = s["x"].dtype
    total, y = _plain_norm(s)
    out = {"y": y.to(dtype), "total": total.to(dtype)}
    h, g = out["total"].float(), s["adjoint"].float()  # the gradient at the sum that the program keeps
    inverse = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPSILON)
    u = g * s["weight"].float()
    dx = inverse * (u - h * inverse.square() * (u * h).mean(-1, keepdim=True)) + s["total_adjoint"].float()
    return out | {"x_adjoint": dx.to(dtype), "weight_adjoint": (g * h * inverse).sum(0).to(dtype)}


def _places(offsets, longest, count):
    """For packed rows: their numbers as [structure, place], which places exist, and each row's structure and place."""
    lens = offsets[1:] - offsets[:-1]
    place = torch.arange(longest, device="cuda")
    index = (offsets[:-1, None] + place).clamp_(max=max(count - 1, 0))
    row = torch.arange(count, device="cuda")
    owner = torch.searchsorted(offsets, row, right=True) - 1
    return index, place < lens[:, None], owner, row - offsets[owner]


def _plain_attend(s, train):
    q, k, v = s["q"], s["k"], s["v"]
    n, h, d = q.shape
    hk, group = k.shape[1], h // k.shape[1]
    b, lq, lk = s["offsets"].numel() - 1, s["longest_query"], s["longest"]
    q_index, _, owner, place = _places(s["offsets"], lq, n)
    if s["key_offsets"] is None:
        k_index, live, k_owner, k_place = _places(s["offsets"], lk, k.shape[0])
    else:
        k_index, live, k_owner, k_place = _places(s["key_offsets"], lk, k.shape[0])
    if s["key_mask"] is not None:
        live = live & s["key_mask"][k_index]
    live = live[:, None, None, None, :]

    def rows(x):  # [rows, heads, d] to [structure, key head, group x place, d]
        return x.float()[q_index].reshape(b, lq, hk, group, d).permute(0, 2, 3, 1, 4).reshape(b, hk, group * lq, d)

    def cols(x):  # [keys, key heads, d] to [structure, key head, place, d]
        return x.float()[k_index].permute(0, 2, 1, 3).contiguous()

    def back(x, where):  # and back to packed rows
        x = x.reshape(b, hk, group, lq, d).permute(0, 3, 1, 2, 4).reshape(b, lq, h, d)
        return x[where].to(q.dtype)

    qp, kp, vp = rows(q), cols(k), cols(v)
    score = (qp @ kp.transpose(-1, -2)).reshape(b, hk, group, lq, lk) * s["scale"]
    bend = None
    if s["cap"] > 0:
        bend = torch.tanh(score / s["cap"])
        score = s["cap"] * bend
    if s["bias"]:
        slope = s["slopes"].reshape(1, hk, group, 1, 1)
        kpos = s["positions"] if s["key_positions"] is None else s["key_positions"]
        apart = s["positions"][q_index][:, :, None, :] - kpos[k_index][:, None, :, :]
        far = apart.square().sum(-1).sqrt()
        score = score - slope * far[:, None, None]
    score = torch.where(live, score, torch.full((), -math.inf, device="cuda"))
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    del score
    out = p.reshape(b, hk, group * lq, lk) @ vp
    result = {"out": back(out, (owner, place))}
    if not train:
        return result
    gp = rows(s["adjoint"])
    lost = gp @ vp.transpose(-1, -2)
    # rows past a structure's end repeat another atom's: nothing of theirs counts
    exists = (torch.arange(lq, device="cuda") < (s["offsets"][1:] - s["offsets"][:-1])[:, None])[:, None, None, :, None]
    p = torch.where(exists, p, torch.zeros((), device="cuda"))
    slant = p * (lost.reshape(p.shape) - (gp * out).sum(-1).reshape(b, hk, group, lq, 1))
    del lost
    result["v_adjoint"] = (p.reshape(b, hk, group * lq, lk).transpose(-1, -2) @ gp).permute(0, 2, 1, 3)[k_owner, k_place].to(q.dtype)
    if s["forces"]:
        result["slopes_adjoint"] = -(slant * far[:, None, None]).sum((0, 3, 4)).reshape(h)
        pull = -(slant * slope).sum((1, 2)) / torch.where(far > 0, far, torch.ones_like(far))
        pair = pull[..., None] * apart
        result["positions_adjoint"] = pair.sum(2)[owner, place] - pair.sum(1)[k_owner, k_place]
    del p
    if bend is not None:
        slant = slant * (1.0 - bend.square())
    slant = (slant * s["scale"]).reshape(b, hk, group * lq, lk)
    result["q_adjoint"] = back(slant @ kp, (owner, place))
    result["k_adjoint"] = (slant.transpose(-1, -2) @ qp).permute(0, 2, 1, 3)[k_owner, k_place].to(q.dtype)
    return result


# ---- this framework's operators ----------------------------------------------

def _own(s):
    from ye3t_amd import runtime

    kind = s["kind"]
    if kind.startswith("embed"):
        # the tokens of a program's data are checked once, where the data is loaded
        out = {"rows": runtime.embedding(s["ids"], s["table"], scale=s["scale"], validate=False)}
        if kind == "embed_train":
            out["table_adjoint"] = runtime.embedding_adjoint(s["adjoint"], s["ids"], s["vocabulary"], scale=s["scale"],
                                                             validate=False)
        return out
    if kind == "norm8":
        codes, scales, total = runtime.rms_norm_8bit(s["x"], s["weight"], residual=s["residual"], epsilon=EPSILON)
        return {"codes": codes, "scales": scales, "total": total}
    if kind == "norm_train":
        y, total = runtime.rms_norm(s["x"], s["weight"], residual=s["residual"], epsilon=EPSILON)
        dx, dw = runtime.rms_norm_adjoint(s["adjoint"], total, s["weight"], total_adjoint=s["total_adjoint"],
                                          epsilon=EPSILON)
        return {"y": y, "total": total, "x_adjoint": dx, "weight_adjoint": dw}
    kw = dict(key_offsets=s["key_offsets"], scale=s["scale"], cap=s["cap"], slopes=s["slopes"], positions=s["positions"],
              key_positions=s["key_positions"], key_mask=s["key_mask"], validate=False)
    if kind == "attend":
        return {"out": runtime.atom_attention(s["q"], s["k"], s["v"], s["offsets"], **kw)}
    out, sums = runtime.atom_attention(s["q"], s["k"], s["v"], s["offsets"], return_log_sums=True, **kw)
    grads = runtime.atom_attention_adjoint(s["adjoint"], out, sums, s["q"], s["k"], s["v"], s["offsets"],
                                           bias_gradients=s["forces"], **kw)
    result = {"out": out, "q_adjoint": grads[0], "k_adjoint": grads[1], "v_adjoint": grads[2]}
    if s["forces"]:
        result |= {"slopes_adjoint": grads[3], "positions_adjoint": grads[4]}
    return result


def run(state):
    if own:
        return _own(state)
    kind = state["kind"]
    if kind.startswith("attend"):
        return _plain_attend(state, kind == "attend_train")
    return {"embed": _plain_embed, "embed_train": _plain_embed_train, "norm8": _plain_norm8,
            "norm_train": _plain_norm_train}[kind](state)


# ---- in 64 bits --------------------------------------------------------------

def _exact_embed(s):
    t = s["table"].double()
    out = {"rows": t.index_select(0, s["ids"].long()) * s["scale"]}
    if s["kind"] == "embed_train":
        order = torch.argsort(s["ids"].long())
        counts = torch.bincount(s["ids"].long(), minlength=t.shape[0])
        sums = torch.segment_reduce(s["adjoint"].double()[order], "sum", lengths=counts, axis=0, unsafe=True)
        out["table_adjoint"] = s["scale"] * sums
    return out


def _exact_norm(s):
    h = s["x"].double() + s["residual"].double()
    w = s["weight"].double()
    rho = 1.0 / ((h * h).sum(1, keepdim=True) / h.shape[1] + EPSILON).sqrt()
    y = rho * w * h
    if s["kind"] == "norm_train":
        g = s["adjoint"].double()
        along = (g * w * h).sum(1, keepdim=True) * rho ** 3 / h.shape[1]
        return {"y": y, "total": h, "x_adjoint": rho * g * w - along * h + s["total_adjoint"].double(),
                "weight_adjoint": torch.einsum("nw,nw,n->w", g, h, rho[:, 0])}
    n, width = y.shape
    codes, scales = torch.empty_like(y), torch.empty((n, -(-width // GROUP)), dtype=torch.float64, device="cuda")
    for k, c in enumerate(range(0, width, GROUP)):
        part = y[:, c:c + GROUP]
        scale = part.abs().max(dim=1, keepdim=True).values / LARGEST_8BIT
        x = part / scale.clamp(min=1e-300)
        # three mantissa bits above 2^-6, steps of 2^-9 below; ties to even
        step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3.0)
        codes[:, c:c + GROUP] = (torch.round(x / step) * step).clamp(-LARGEST_8BIT, LARGEST_8BIT)
        scales[:, k] = scale[:, 0]
    return {"codes": codes, "scales": scales, "total": h}


def _exact_attend(s):
    train = s["kind"] == "attend_train"
    q, k, v = s["q"], s["k"], s["v"]
    group = q.shape[1] // k.shape[1]
    zero = lambda x: torch.zeros(x.shape, dtype=torch.float64, device="cuda")  # noqa: E731
    out, dq, dk, dv = zero(q), zero(q), zero(k), zero(v)
    forces = train and s["forces"]
    dslope = zero(s["slopes"]) if forces else None
    dpos = zero(s["positions"]) if forces else None
    first = s["offsets"].tolist()
    key_first = first if s["key_offsets"] is None else s["key_offsets"].tolist()
    kpos = s["positions"] if s["key_positions"] is None else s["key_positions"]
    # all heads of a structure together, or one key head after the other where that would be large
    for b in range(len(first) - 1):
        i, j = slice(first[b], first[b + 1]), slice(key_first[b], key_first[b + 1])
        nq, nk = i.stop - i.start, j.stop - j.start
        at_once = max(1, min(k.shape[1], int(3e8 // max(1, nq * nk * group))))
        if s["bias"]:
            apart = s["positions"][i, None].double() - kpos[None, j].double()
            far = torch.linalg.vector_norm(apart, dim=-1)
            unit = torch.where(far[..., None] > 0, apart / far[..., None], torch.zeros_like(apart)) if forces else None
        for c in range(0, k.shape[1], at_once):
            kh = slice(c, min(k.shape[1], c + at_once))
            qh = slice(kh.start * group, kh.stop * group)
            spread = lambda x: x[j, kh].double().transpose(0, 1).repeat_interleave(group, 0).contiguous()  # noqa: E731
            gather = lambda x: x.reshape(-1, group, *x.shape[1:]).sum(1).transpose(0, 1)  # noqa: E731
            a, kk, vv = q[i, qh].double().transpose(0, 1).contiguous(), spread(k), spread(v)
            raw = s["scale"] * torch.bmm(a, kk.transpose(1, 2))
            z = s["cap"] * torch.tanh(raw / s["cap"]) if s["cap"] > 0 else raw
            if s["bias"]:
                z = z - s["slopes"][qh].double()[:, None, None] * far
            if s["key_mask"] is not None:
                z = z.masked_fill(~s["key_mask"][j], -math.inf)
            p = torch.softmax(z, -1).nan_to_num(0.0)
            o = torch.bmm(p, vv)
            out[i, qh] = o.transpose(0, 1)
            if not train:
                continue
            g = s["adjoint"][i, qh].double().transpose(0, 1).contiguous()
            dp = torch.bmm(g, vv.transpose(1, 2))
            dz = p * (dp - (p * dp).sum(-1, keepdim=True))
            dv[j, kh] = gather(torch.bmm(p.transpose(1, 2), g))
            if forces:
                dslope[qh] -= (dz * far).sum((1, 2))
                pull = -torch.einsum("hij,h->ij", dz, s["slopes"][qh].double())[..., None] * unit
                dpos[i] += pull.sum(1)
                dpos[j] -= pull.sum(0)
            draw_ = dz * s["scale"]
            if s["cap"] > 0:
                draw_ = draw_ / torch.cosh(raw / s["cap"]).square()
            dq[i, qh] = torch.bmm(draw_, kk).transpose(0, 1)
            dk[j, kh] = gather(torch.bmm(draw_.transpose(1, 2), a))
    result = {"out": out}
    if train:
        result |= {"q_adjoint": dq, "k_adjoint": dk, "v_adjoint": dv}
    if forces:
        result |= {"slopes_adjoint": dslope, "positions_adjoint": dpos}
    return result


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"].startswith("attend"):
        return _exact_attend(s)
    return _exact_embed(s) if case["kind"].startswith("embed") else _exact_norm(s)
