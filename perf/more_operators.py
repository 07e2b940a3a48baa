"""Workloads of the operators around a transformer block over sparse-voxel features: the norm at a
block's border with gate, residual scale, modulation and dropout; dropout by itself; the router of a
mixture of experts, and the products of its feed-forward, grouped by expert.

Where ``own`` is false ``run`` computes an operator in plain torch operations, where it is true
with the calls of ``mlx_diffuser_b200``. The largest sizes are those of the package's residual
stack: two surfaces at 64^3, 40,662 voxels, 1024 channels.
"""

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
EPS = 1e-6


# ---- cases ------------------------------------------------------------------------------------


def listed():
    return [
        # a training step at a modulated block's border: two surfaces, one modulation each
        {"name": "block_train", "op": "block", "rows": 20331, "channels": 1024, "batch": 2,
         "dtype": "bf16", "norm": "layer", "branch_norm": False, "gate": True, "modulated": True,
         "affine": False, "alpha": 1.0, "dropout": 0.1, "train": True},
        # norms on both sides of a block with a residual scale, every voxel, serving
        {"name": "block_both_norms", "op": "block", "rows": 40662, "channels": 1024, "batch": 2,
         "dtype": "bf16", "norm": "rms", "branch_norm": True, "gate": True, "modulated": False,
         "affine": True, "alpha": 0.5, "dropout": 0.0, "train": False},
        # the smallest call: a handful of conditioning rows in fp32
        {"name": "block_few_rows", "op": "block", "rows": 8, "channels": 256, "batch": 1,
         "dtype": "fp32", "norm": "layer", "branch_norm": False, "gate": True, "modulated": True,
         "affine": True, "alpha": 1.0, "dropout": 0.0, "train": False},
        # dropout of a whole feature map in training
        {"name": "dropout_train", "op": "dropout", "rows": 40662, "channels": 1024,
         "dtype": "bf16", "residual": False, "p": 0.1, "train": True},
        # an odd feature map, added to the residual stream
        {"name": "dropout_odd", "op": "dropout", "rows": 5041, "channels": 331, "dtype": "fp16",
         "residual": True, "p": 0.25, "train": False},
        # the router's step of training, many experts
        {"name": "route_train", "op": "route", "rows": 40662, "experts": 64, "k": 4,
         "dtype": "fp32", "normalize": True, "masked": False, "train": True},
        # the router for a handful of rows
        {"name": "route_few_rows", "op": "route", "rows": 8, "experts": 16, "k": 2,
         "dtype": "bf16", "normalize": True, "masked": False, "train": False},
        # the widening products of a mixture of experts, every voxel, serving
        {"name": "expert_up", "op": "expert", "rows": 40662, "experts": 8, "k": 2, "inputs": 1024,
         "outputs": 4096, "dtype": "bf16", "activation": "gelu_tanh", "gather": True,
         "combine": False, "bias": True, "masked": False, "train": False},
        # one training step of the narrowing products and the weighted sum behind them
        {"name": "expert_down_train", "op": "expert", "rows": 12001, "experts": 16, "k": 2,
         "inputs": 2048, "outputs": 1024, "dtype": "bf16", "activation": "none", "gather": False,
         "combine": True, "bias": True, "masked": False, "train": True},
        # a lone row: two experts' weights are read once
        {"name": "expert_one_row", "op": "expert", "rows": 1, "experts": 16, "k": 2,
         "inputs": 1024, "outputs": 4096, "dtype": "bf16", "activation": "silu", "gather": True,
         "combine": False, "bias": True, "masked": False, "train": False},
        # odd channel counts on both sides, single-layer experts, a training step
        {"name": "expert_odd", "op": "expert", "rows": 5041, "experts": 5, "k": 1, "inputs": 331,
         "outputs": 517, "dtype": "fp16", "activation": "gelu", "gather": True, "combine": True,
         "bias": False, "masked": True, "train": True},
        # a small scene in fp32, training
        {"name": "expert_fp32", "op": "expert", "rows": 2001, "experts": 4, "k": 2, "inputs": 256,
         "outputs": 512, "dtype": "fp32", "activation": "silu", "gather": True, "combine": False,
         "bias": True, "masked": False, "train": True},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _channels(rng, low, high):
    """Channel counts: multiples of 64 half of the time, anything otherwise."""
    c = _log(rng, low, high)
    return max(64, c // 64 * 64) if rng.random() < 0.5 else c


def draw(rng: random.Random):
    op = rng.choice(["block", "dropout", "route", "expert", "expert"])
    if op == "block":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        rows = _log(rng, 1, 20331 if dtype == "fp32" else 40662)
        return {"op": op, "rows": rows, "channels": _channels(rng, 8, 1024),
                "batch": rng.randint(1, min(4, rows)), "dtype": dtype,
                "norm": rng.choice(["layer", "rms"]), "branch_norm": rng.random() < 0.4,
                "gate": rng.random() < 0.7, "modulated": rng.random() < 0.6,
                "affine": rng.random() < 0.5, "alpha": rng.choice([1.0, 0.5, 0.125]),
                "dropout": rng.choice([0.0, 0.0, 0.1, 0.5]), "train": rng.random() < 0.5}
    if op == "dropout":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        return {"op": op, "rows": _log(rng, 1, 20331 if dtype == "fp32" else 40662),
                "channels": _channels(rng, 8, 1024), "dtype": dtype,
                "residual": rng.random() < 0.5, "p": rng.choice([0.05, 0.1, 0.3, 0.5]),
                "train": rng.random() < 0.5}
    if op == "route":
        experts = _log(rng, 2, 256)
        return {"op": op, "rows": _log(rng, 1, 40662), "experts": experts,
                "k": rng.randint(1, min(8, experts)),
                "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"]),
                "normalize": rng.random() < 0.6, "masked": rng.random() < 0.4,
                "train": rng.random() < 0.5}
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    train = rng.random() < 0.5
    experts = _log(rng, 2, 32)
    acts = ["none", "silu", "gelu", "gelu_tanh"]
    gather, combine = rng.choice([(True, False), (True, False), (False, True), (True, True)])
    return {"op": op, "rows": _log(rng, 1, 12001 if train or dtype == "fp32" else 40662),
            "experts": experts, "k": rng.randint(1, min(4, experts)) if rng.random() < 0.5
            else min(2, experts), "inputs": _channels(rng, 8, 1024),
            "outputs": _channels(rng, 8, 1024), "dtype": dtype,
            "activation": "none" if combine and not gather else rng.choice(acts),
            "gather": gather, "combine": combine, "bias": rng.random() < 0.7,
            "masked": rng.random() < 0.3, "train": train}


# ---- inputs -----------------------------------------------------------------------------------


def _normal(shape, dtype, gen, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)


def _mask(logits, gen):
    """Masks experts here and there, and every expert of one row in sixteen (padding)."""
    n, e = logits.shape
    logits[torch.rand((n, e), device="cuda", generator=gen) < 0.2] = float("-inf")
    logits[torch.rand((n,), device="cuda", generator=gen) < 1 / 16] = float("-inf")
    return logits


def _router_logits(case, dtype, gen):
    """Some experts are asked for more than others."""
    e = case["experts"]
    logits = torch.randn((case["rows"], e), device="cuda", generator=gen)
    logits += 0.7 * torch.randn((e,), device="cuda", generator=gen)
    if case["masked"]:
        _mask(logits, gen)
    return logits.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case)
    s["seed"] = random.Random(int(seed)).getrandbits(63)
    n, train = case["rows"], case["train"]
    dt = DTYPES[case["dtype"]]
    leaves = []
    if case["op"] == "block":
        c, b = case["channels"], case["batch"]
        s["x"], s["branch"] = _normal((n, c), dt, gen, 2.0), _normal((n, c), dt, gen)
        for name, there, shape, mean, scale in (
            ("g", case["gate"], (b, c), 0.3, 0.5), ("s", case["modulated"], (b, c), 0.0, 0.3),
            ("t", case["modulated"], (b, c), 0.0, 0.3), ("w", case["affine"], (c,), 1.0, 0.2),
            ("beta", case["affine"] and case["norm"] == "layer", (c,), 0.0, 0.2),
            ("wb", case["branch_norm"], (c,), 1.0, 0.2),
        ):
            kind = dt if name in "gst" else torch.float32
            r = torch.randn(shape, device="cuda", generator=gen)
            s[name] = (mean + scale * r).to(kind) if there else None
        # rows (batch, x, y, z), batch elements in turn
        coords = np.zeros((n, 4), np.int32)
        coords[:, 0] = np.arange(n) * b // n
        coords[:, 1:] = np.random.default_rng(seed).integers(0, 64, (n, 3))
        s["coords"] = torch.from_numpy(coords).cuda()
        s["index"] = s["coords"][:, 0].long()
        # a row of ones and zeros a voxel: the modulations' rows as a product, with a quick gradient
        s["hot"] = torch.nn.functional.one_hot(s["index"], b).float()
        leaves = ["x", "branch", "g", "s", "t", "w", "beta", "wb"]
        if train:
            s["dy"], s["dh"] = _normal((n, c), dt, gen), _normal((n, c), dt, gen)
    elif case["op"] == "dropout":
        c = case["channels"]
        s["x"] = _normal((n, c), dt, gen)
        s["res"] = _normal((n, c), dt, gen, 2.0) if case["residual"] else None
        leaves = ["x", "res"]
        if train:
            s["dy"] = _normal((n, c), dt, gen)
    elif case["op"] == "route":
        s["logits"] = _router_logits(case, dt, gen)
        leaves = ["logits"]
        if train:
            s["dw"] = _normal((n, case["k"]), torch.float32, gen)
    else:
        e, k, i, o = (case[name] for name in ("experts", "k", "inputs", "outputs"))
        logits = _router_logits(case, torch.float32, gen)
        chosen, weights, order, offsets, place = _plain_route(logits, k, True)
        slots = n * k
        s["x"] = _normal((n if case["gather"] else slots, i), dt, gen)
        s["w"] = _normal((e, o, i), dt, gen, 1 / math.sqrt(i))
        s["b"] = _normal((e, o), dt, gen, 0.5) if case["bias"] else None
        leaves = ["x", "w", "b"]
        if own:
            from mlx_diffuser_b200 import route

            # the routing that a program holds for both products of the block
            s["routes"] = route(logits, k)
            s["p"] = s["routes"].weights
        else:
            bounds = offsets.tolist()
            s["p"] = weights
            s["order"], s["place"] = order.long(), place.long()
            s["spans"] = list(zip(bounds[:-1], bounds[1:]))
        if case["combine"]:
            leaves.append("p")
        if train:
            s["dy"] = _normal((n if case["combine"] else slots, o), dt, gen)
    if train:
        s["leaves"] = [s[name].requires_grad_(True) for name in leaves if s[name] is not None]
    return s


# ---- one pass ---------------------------------------------------------------------------------


def _philox(count, seed, subsequence):
    """Philox4x32 with ten rounds: the eight 16-bit numbers of each of ``count`` counters, in a row.
    32-bit words held in 64 bits; a product's upper word is right although its 64 bits wrap."""
    low = 0xFFFFFFFF
    i = torch.arange(count, device="cuda")
    c0, c1 = i & low, i >> 32
    c2, c3 = (torch.full_like(i, v) for v in (subsequence & low, subsequence >> 32))
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low)
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack((c0, c1, c2, c3), 1)
    return torch.stack((words & 0xFFFF, words >> 16), 2).flatten()


def _threshold(p):
    return int(p * 65536 + 0.5)


def _plain_drop(x, p, seed):
    """x in 32 bits: what is kept over its share, zeros elsewhere."""
    cut = _threshold(p)
    numbers = _philox((x.numel() + 7) // 8, seed, 0)[: x.numel()].view(x.shape)
    return torch.where(numbers >= cut, x * (65536 / (65536 - cut)), torch.zeros_like(x))


def _act(z, name):
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _plain_norm(x, kind):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _plain_block(s):
    x, u = s["x"].float(), s["branch"].float()
    if s["dropout"]:
        u = _plain_drop(u, s["dropout"], s["seed"])
    if s["branch_norm"]:
        u = _plain_norm(u, s["norm"]) * s["wb"]
    u = u * s["alpha"]
    if s["gate"]:
        u = u * (s["hot"] @ s["g"].float())
    h = x + u
    # the residual stream is held in the features' type; its gradient stays in 32 bits
    h = h + (h.to(s["x"].dtype).float() - h).detach()
    y = _plain_norm(h, s["norm"])
    if s["w"] is not None:
        y = y * s["w"]
    if s["beta"] is not None:
        y = y + s["beta"]
    if s["modulated"]:
        y = y * (1 + s["hot"] @ s["s"].float()) + s["hot"] @ s["t"].float()
    return y.to(s["x"].dtype), h.to(s["x"].dtype)


def _plain_dropout(s):
    y = _plain_drop(s["x"].float(), s["p"], s["seed"])
    if s["res"] is not None:
        y = y + s["res"].float()
    return y.to(s["x"].dtype)


def _plain_route(logits, k, normalize):
    """Experts by falling logit, the lowest index first among equals, none where the logit is -inf;
    their weights; and the slots (row * k + choice) in the order of their experts."""
    n, e = logits.shape
    x = logits.float()
    index = torch.arange(e, device=x.device)
    left, picked = x.detach().clone(), []
    for _ in range(k):
        top = left.amax(1, keepdim=True)
        best = torch.where(left == top, index, e).amin(1)
        best = torch.where(top[:, 0] == float("-inf"), -1, best)
        picked.append(best)
        left.scatter_(1, best.clamp(min=0)[:, None], float("-inf"))
    chosen = torch.stack(picked, 1)
    there = chosen >= 0
    at = torch.gather(x, 1, chosen.clamp(min=0)).masked_fill(~there, float("-inf"))
    top = x.detach().amax(1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    total = torch.exp((at if normalize else x) - top).sum(1, keepdim=True)
    total = torch.where(total == 0, torch.ones_like(total), total)
    weights = torch.exp(at - top) / total
    flat = torch.where(there, chosen, e).flatten()
    order = torch.sort(flat, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(n * k, device=x.device)
    place = torch.where(there, place.view(n, k), -1)
    counts = (flat[:, None] == index).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    return chosen.int(), weights, order.int(), offsets.int(), place.int()


def _plain_expert(s):
    x, w = s["x"].float(), s["w"].float()
    k = s["k"]
    parts = []
    for e, (first, last) in enumerate(s["spans"]):
        rows = x.index_select(0, s["order"][first:last] // k) if s["gather"] else x[first:last]
        z = rows @ w[e].t()
        if s["bias"]:
            z = z + s["b"].float()[e]
        parts.append(_act(z, s["activation"]))
    behind = s["order"].numel() - s["spans"][-1][1]  # slots that no expert has
    parts.append(x.new_zeros((behind, w.shape[1])))
    out = torch.cat(parts)
    if s["combine"]:
        at = s["place"]
        taken = out.index_select(0, at.clamp(min=0).flatten()).view(*at.shape, -1)
        out = (taken * torch.where(at >= 0, s["p"], 0.0)[..., None]).sum(1)
    return out.to(s["x"].dtype)


def _own_block(s):
    from mlx_diffuser_b200 import block_norm

    drop = {"dropout": s["dropout"], "seed": s["seed"]} if s["dropout"] else {}
    return block_norm(s["x"], s["branch"], norm=s["norm"], branch_norm=s["branch_norm"],
                      branch_weight=s["wb"], gate=s["g"], residual_scale=s["alpha"],
                      weight=s["w"], bias=s["beta"], scale=s["s"], shift=s["t"],
                      coords=s["coords"], batch_size=s["batch"], eps=EPS, **drop)


def _own_dropout(s):
    from mlx_diffuser_b200 import dropout

    return dropout(s["x"], s["p"], s["seed"], residual=s["res"])


def _own_route(s):
    from mlx_diffuser_b200 import route

    r = route(s["logits"], s["k"], normalize=s["normalize"])
    return r.experts, r.weights, r.order, r.offsets, r.place


def _own_expert(s):
    from mlx_diffuser_b200 import expert_linear

    return expert_linear(s["x"], s["w"], s["routes"], s["b"], activation=s["activation"],
                         gather=s["gather"], combine=s["combine"])


def run(state):
    s = state
    if s["op"] == "block":
        step = _own_block if own else _plain_block
    elif s["op"] == "dropout":
        step = _own_dropout if own else _plain_dropout
    elif s["op"] == "expert":
        step = _own_expert if own else _plain_expert
    elif own:
        step = _own_route
    else:
        def step(s):
            return _plain_route(s["logits"], s["k"], s["normalize"])
    if not s["train"]:
        with torch.no_grad():
            return step(s)
    out = step(s)
    if s["op"] == "block":
        return (*out, *torch.autograd.grad(out, s["leaves"], (s["dy"], s["dh"])))
    if s["op"] == "route":
        return (*out, *torch.autograd.grad(out[1], s["leaves"], s["dw"]))
    return (out, *torch.autograd.grad(out, s["leaves"], s["dy"]))


# ---- what a pass cannot do without --------------------------------------------------------------


def work(case):
    n, train, e = case["rows"], case["train"], BYTES[case["dtype"]]
    if case["op"] == "block":
        c, b = case["channels"], case["batch"]
        small = e * b * c * (case["gate"] + 2 * case["modulated"])
        small += 4 * c * (case["affine"] * (1 + (case["norm"] == "layer")) + case["branch_norm"])
        # x, branch, h, y; backwards dy, dh, h, branch, dx, dbranch, of which h and branch are there
        return {"bytes": n * c * e * (8 if train else 4) + small * (2 if train else 1) + 16 * n,
                "flops": n * c * (40 if train else 14)}
    if case["op"] == "dropout":
        cells = n * case["channels"]
        return {"bytes": cells * e * (2 + case["residual"] + 2 * train), "flops": cells * 2}
    if case["op"] == "route":
        m, k = case["experts"], case["k"]
        # logits; experts, weights, order, place, offsets; backwards the weights' gradient
        b = n * m * e * (1 + train) + n * k * 4 * (4 + train) + 4 * (m + 1)
        return {"bytes": b, "flops": n * m * (k + 4)}
    m, k, i, o = (case[name] for name in ("experts", "k", "inputs", "outputs"))
    slots = n * k
    held = min(m, slots)  # experts whose weights are read
    ins = (n if case["gather"] else slots) * i
    outs = (n if case["combine"] else slots) * o
    params = held * o * (i + case["bias"])
    b = e * (ins + outs + params) + 4 * slots * (1 + case["combine"])
    if train:  # dy; the gradients of x, weights and bias
        b += e * (outs + ins + m * o * (i + case["bias"])) + 4 * slots * case["combine"]
    return {"bytes": b, "flops": 2 * slots * i * o * (3 if train else 1)}


# ---- the definition in 64 bits ------------------------------------------------------------------


def _numbers64(cells, seed):
    """The generator's 16-bit numbers by numpy's unsigned words."""
    u64, low = np.uint64, np.uint64(0xFFFFFFFF)
    ctr = np.arange((cells + 7) // 8, dtype=u64)
    x = [ctr & low, ctr >> u64(32), np.zeros_like(ctr), np.zeros_like(ctr)]
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        p, q = x[0] * u64(0xD2511F53), x[2] * u64(0xCD9E8D57)
        x = [(q >> u64(32)) ^ x[1] ^ u64(key[0]), q & low, (p >> u64(32)) ^ x[3] ^ u64(key[1]),
             p & low]
        key = [(key[0] + 0x9E3779B9) % 2**32, (key[1] + 0xBB67AE85) % 2**32]
    words = np.stack(x, 1).astype("<u4")
    return torch.from_numpy(words.view("<u2").reshape(-1)[:cells].astype(np.int32)).cuda()


def _kept64(shape, p, seed):
    """What each element is multiplied by."""
    cut = _threshold(p)
    kept = _numbers64(math.prod(shape), seed).view(shape) >= cut
    return kept.to(torch.float64) * (65536.0 / (65536 - cut))


def _norm64(x, kind):
    """The normed rows and the factor that the gradient is multiplied by."""
    if kind == "layer":
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        r = (var + EPS) ** -0.5
        return (x - mean) * r, r
    r = (torch.linalg.vector_norm(x, dim=1, keepdim=True) ** 2 / x.shape[1] + EPS) ** -0.5
    return x * r, r


def _norm_grad64(g, unit, r, kind):
    d = g - unit * (g * unit).mean(1, keepdim=True)
    if kind == "layer":
        d = d - g.mean(1, keepdim=True)
    return d * r


def _exact_block(s):
    f = torch.float64
    n, c = s["x"].shape
    batch = s["batch"]

    def rows(name, missing):
        t = s[name]
        return torch.full((1, 1), missing, dtype=f, device="cuda") if t is None else t.to(f)

    def spread(t):
        return t[s["index"]] if t.shape[1] == c else t

    def per_batch(t):
        return torch.stack([t[s["index"] == i].sum(0) for i in range(batch)])

    keep = _kept64((n, c), s["dropout"], s["seed"]) if s["dropout"] else 1.0
    d = s["branch"].to(f) * keep
    wb = s["wb"].to(f) if s["branch_norm"] else torch.ones(c, dtype=f, device="cuda")
    unit_d, r_d = _norm64(d, s["norm"]) if s["branch_norm"] else (d, None)
    gate = spread(rows("g", 1.0)) * s["alpha"]
    h = (s["x"].to(f) + gate * wb * unit_d).to(s["x"].dtype).to(f)
    unit, r = _norm64(h, s["norm"])
    w = torch.ones(c, dtype=f, device="cuda") if s["w"] is None else s["w"].to(f)
    beta = torch.zeros(c, dtype=f, device="cuda") if s["beta"] is None else s["beta"].to(f)
    sc, sh = spread(rows("s", 0.0)), spread(rows("t", 0.0))
    y = (unit * w + beta) * (1 + sc) + sh
    if not s["train"]:
        return y, h
    dy = s["dy"].to(f)
    dt = dy * (1 + sc)
    dh = s["dh"].to(f) + _norm_grad64(dt * w, unit, r, s["norm"])
    du = gate * dh
    db = du * wb
    if s["branch_norm"]:
        db = _norm_grad64(db, unit_d, r_d, s["norm"])
    out = [y, h, dh, db * keep]
    if s["g"] is not None:
        out.append(per_batch(dh * wb * unit_d) * s["alpha"])
    if s["s"] is not None:
        out += [per_batch(dy * (unit * w + beta)), per_batch(dy)]
    if s["w"] is not None:
        out.append((dt * unit).sum(0))
    if s["beta"] is not None:
        out.append(dt.sum(0))
    if s["wb"] is not None:
        out.append((du * unit_d).sum(0))
    return tuple(out)


def _exact_dropout(s):
    f = torch.float64
    keep = _kept64(tuple(s["x"].shape), s["p"], s["seed"])
    y = s["x"].to(f) * keep
    if s["res"] is not None:
        y = y + s["res"].to(f)
    if not s["train"]:
        return y
    dy = s["dy"].to(f)
    return (y, dy * keep) if s["res"] is None else (y, dy * keep, dy)


def _exact_route(s):
    f = torch.float64
    x = s["logits"].detach()
    n, m = x.shape
    k = s["k"]
    v = x.double().cpu().numpy()
    best = np.argsort(-v, axis=1, kind="stable")[:, :k]
    picked = np.take_along_axis(v, best, 1)
    none = np.isneginf(picked)
    experts = np.where(none, -1, best)
    keys = np.where(none, m, best).reshape(-1)
    order = np.argsort(keys, kind="stable")
    place = np.empty(n * k, np.int64)
    place[order] = np.arange(n * k)
    place = np.where(none, -1, place.reshape(n, k))
    offsets = np.concatenate([[0], np.cumsum(np.bincount(keys, minlength=m + 1)[:m])])
    scores = torch.from_numpy(np.where(none, -np.inf, picked) if s["normalize"] else v).cuda()
    at = torch.from_numpy(np.where(none, -np.inf, picked)).cuda()
    total = torch.logsumexp(scores, 1, keepdim=True)
    total = torch.where(total == float("-inf"), 0.0, total)
    weights = torch.exp(at - total)
    ints = [torch.from_numpy(a.astype(np.int32)).cuda() for a in (experts, order, offsets, place)]
    out = (ints[0], weights, *ints[1:])
    if not s["train"]:
        return out
    dw = s["dw"].to(f)
    dot = (dw * weights).sum(1, keepdim=True)
    grad = torch.zeros((n, m), dtype=f, device="cuda")
    if not s["normalize"]:
        grad -= torch.exp(x.to(f) - total) * dot
        dot = 0.0
    grad.scatter_add_(1, torch.from_numpy(best).cuda(), weights * (dw - dot))
    return (*out, grad)


def _act64(z, name):
    """The activation and its derivative."""
    if name == "silu":
        g = torch.sigmoid(z)
        return z * g, g * (1 + z * (1 - g))
    if name == "gelu":
        p = torch.special.ndtr(z)
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(8 / math.pi)
        g = torch.sigmoid(c * (z + 0.044715 * z**3))
        return z * g, g + z * g * (1 - g) * c * (1 + 3 * 0.044715 * z * z)
    return z, None


def _exact_expert(s, logits):
    f = torch.float64
    n, m, k = s["rows"], s["experts"], s["k"]
    experts, p, order, offsets, place = _exact_route(
        {"logits": logits, "k": k, "normalize": True, "train": False})
    x, w = s["x"].detach().to(f), s["w"].detach().to(f)
    bias = s["b"].detach().to(f) if s["bias"] else None
    token = order.long() // k
    rows = torch.zeros((n * k, s["outputs"]), dtype=f, device="cuda")
    slopes = [None] * m
    bounds = offsets.tolist()

    def inputs(a, b):
        return x[token[a:b]] if s["gather"] else x[a:b]

    for i in range(m):
        a, b = bounds[i], bounds[i + 1]
        z = torch.einsum("nk,ok->no", inputs(a, b), w[i])
        rows[a:b], slopes[i] = _act64(z if bias is None else z + bias[i], s["activation"])
    out = rows
    if s["combine"]:
        out = torch.zeros((n, s["outputs"]), dtype=f, device="cuda")
        for j in range(k):
            out += p[:, j, None] * rows[place[:, j].long().clamp(min=0)]
    if not s["train"]:
        return out
    dy = s["dy"].to(f)
    share = p.reshape(-1)[order.long()]
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    db = None if bias is None else torch.zeros_like(bias)
    for i in range(m):
        a, b = bounds[i], bounds[i + 1]
        dz = dy[token[a:b]] * share[a:b, None] if s["combine"] else dy[a:b].clone()
        if slopes[i] is not None:
            dz *= slopes[i]
        dw[i] = dz.T @ inputs(a, b)
        if db is not None:
            db[i] = dz.sum(0)
        if s["gather"]:
            dx.index_add_(0, token[a:b], dz @ w[i])
        else:
            dx[a:b] = dz @ w[i]
    grads = [dx, dw] + ([] if db is None else [db])
    if s["combine"]:
        dp = [(dy * rows[place[:, j].long().clamp(min=0)]).sum(1) for j in range(k)]
        grads.append(torch.stack(dp, 1) * (place >= 0))
    return (out, *grads)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "expert":
            gen = torch.Generator(device="cuda").manual_seed(int(seed))
            return _exact_expert(s, _router_logits(case, torch.float32, gen))
        return {"block": _exact_block, "dropout": _exact_dropout,
                "route": _exact_route}[case["op"]](s)
