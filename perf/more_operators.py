"""Performance cases of the products with affine weights, of a routed layer for a
few tokens and of the router's choice of experts.

Each case is one call that a serving program or a fine-tuning step makes:
``linear.affine_linear`` (packed 2-, 4- or 8-bit codes with a scale and a bias for
each group of a row), ``experts.ExpertMLP.decode`` (all of a routed layer's
experts for a few rows) and ``experts.top_k_softmax`` with its gradient. Sizes are
those of the benchmark layers (``bench.py``) or generic.

``listed()`` are the fixed cases, ``draw()`` gives others over the same ranges,
``prepare()`` builds what the program holds before the call, ``run()`` is one
pass: in plain torch operations in 32 bits, or, with ``own``, through the
framework. ``exact()`` is the same result from the definition in 64 bits.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _package():
    # the package lives in a directory whose name is no Python identifier
    path = os.path.join(os.getcwd(), "mlx-gptq-mxfp_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from mlx_gptq import experts, linear

    return experts, linear


# --------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------
#
# kind     affine: a product with affine weights; decode: a routed layer for a few
#          tokens; router: the choice of experts (train: with its gradient)
# groups   experts (0: one dense weight, no offsets)
# rows     affine: out features; decode: the experts' inner size
# cols     affine: in features; decode: the hidden size
# tokens   rows of x; affine with top_k > 0: every row is routed to top_k experts
#          and the product gathers its rows
# group    values that share a scale and a bias; params: the type of these


def _affine(name, **kw):
    c = {"name": name, "kind": "affine", "dtype": "bf16", "params": "bf16", "bits": 4, "group": 64,
         "groups": 0, "top_k": 0, "empty": 0}
    c.update(kw)
    return c


def _decode(name, fmt, **kw):
    c = {"name": name, "kind": "decode", "format": fmt, "dtype": "bf16", "groups": 128, "rows": 768,
         "cols": 2048, "top_k": 8}
    if fmt == "affine":
        c.update(params="bf16", bits=4, group=64)
    c.update(kw)
    return c


def listed():
    return [
        # a dense MLP matrix in the solver's default grid, one token
        _affine("affine_token", rows=14336, cols=4096, tokens=1),
        # odd sizes in half precision, 8-bit codes in short groups, a small batch
        _affine("affine_odd", dtype="f16", params="f16", bits=8, group=32, rows=1001, cols=736,
                tokens=37),
        # gate/up products of a routed layer, 64 sequences decoding together
        _affine("affine_experts", groups=128, rows=1536, cols=2048, tokens=64, top_k=8),
        # 8-bit experts whose rows are in the experts' order already, fp32 scales
        _affine("affine_ragged", params="f32", bits=8, group=128, groups=60, rows=1408, cols=1024,
                tokens=4099, empty=3),
        # the dense matrix again, a prompt
        _affine("affine_prompt", rows=14336, cols=4096, tokens=8191),
        # a whole routed layer for one token: 16-bit weights
        _decode("decode_dense", "dense", tokens=1),
        # the same with the solver's MXFP4 codes
        _decode("decode_mxfp4", "mxfp4", tokens=1),
        # affine codes, a small batch of sequences
        _decode("decode_affine", "affine", tokens=16),
        # MXFP8 codes, the largest batch of the call
        _decode("decode_mxfp8", "mxfp8", tokens=64),
        # a small layer of odd sizes in half precision
        _decode("decode_odd", "dense", dtype="f16", groups=8, rows=333, cols=737, tokens=5, top_k=2),
        # the router of one token
        {"name": "router_token", "kind": "router", "dtype": "f32", "groups": 128, "tokens": 1,
         "top_k": 8, "renormalize": True, "masked": 0, "train": False},
        # the router of a calibration batch in training, with the experts' groups that
        # a row may not use masked out
        {"name": "router_train", "kind": "router", "dtype": "bf16", "groups": 128, "tokens": 65536,
         "top_k": 8, "renormalize": False, "masked": 4, "train": True},
    ]


def _log_int(rng, lo, hi, multiple=1):
    """An integer in [lo, hi], even over the logarithm, a multiple of `multiple`."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(multiple, min(hi // multiple, max(1, round(v / multiple))) * multiple)


def draw(rng):
    kind = rng.choice(("affine", "affine", "decode", "decode", "router"))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    if kind == "router":
        groups = rng.choice((8, 60, 64, 100, 128, 256, 512))
        top_k = rng.choice([k for k in (1, 2, 4, 6, 8) if k <= groups // 2])
        return {"kind": kind, "dtype": rng.choice(("bf16", "f16", "f32")), "groups": groups,
                "tokens": _log_int(rng, 1, 65536), "top_k": top_k,
                "renormalize": rng.random() < 0.5, "masked": rng.choice((0, 0, 4)),
                "train": rng.random() < 0.5}
    group = rng.choice((32, 64, 64, 128))
    bits = rng.choice((4, 4, 4, 8, 2))
    params = rng.choice((dtype, dtype, "f32"))
    if kind == "affine":
        groups = rng.choice((0, 0, 0, 8, 60, 128))
        rows = _log_int(rng, 256, 14336 if groups < 9 else 2048, rng.choice((1, 16, 128)))
        cols = _log_int(rng, 256, 8192 if groups < 9 else 2048, group)
        # at most as many products as the largest listed case has
        entries = _log_int(rng, 1, max(1, min(16384, 8191 * 14336 * 4096 // (rows * cols))))
        top_k = rng.choice((0, 2, 8)) if groups else 0
        return {"kind": kind, "dtype": dtype, "params": params, "bits": bits, "group": group,
                "groups": groups, "rows": rows, "cols": cols,
                "tokens": max(1, entries // max(top_k, 1)), "top_k": top_k,
                "empty": groups // 16 if groups >= 60 else 0}
    fmt = rng.choice(("dense", "mxfp4", "mxfp8", "affine", "affine"))
    groups = rng.choice((8, 16, 60, 128))
    if fmt in ("mxfp4", "mxfp8"):
        dtype = "bf16"
    multiple = {"dense": rng.choice((1, 8, 64)), "affine": group}.get(fmt, 32)
    case = {"kind": kind, "format": fmt, "dtype": dtype, "groups": groups,
            "rows": _log_int(rng, 128, 1536, multiple),
            "cols": _log_int(rng, 256, 4096 if groups < 60 else 2048, multiple),
            "tokens": _log_int(rng, 1, 64), "top_k": rng.choice((1, 2, 4, 8))}
    if fmt == "affine":
        case.update(params=params, bits=bits, group=group)
    return case


def _routing(case):
    """(counts, entries): list entries of each expert, heaviest first, and
    their sum. The counts follow the case alone; a seed only says which expert
    has which. They fall off as 1 / rank^0.8, as a router without a balancing
    loss leaves them; an expert gets a token at most once."""
    groups, tokens, top_k = case["groups"], case["tokens"], case["top_k"]
    entries = tokens * max(top_k, 1)
    if groups <= 1:
        return [entries], entries
    active = groups - case.get("empty", 0)
    if top_k:
        active = max(active, top_k)
    rng = random.Random(entries * 31 + groups)
    weight = [(r + 1) ** -0.8 * rng.uniform(0.8, 1.25) for r in range(active)]
    cap = tokens if top_k else entries
    counts = [0] * active
    left = entries
    while left > 0:  # shares of what is left, none above the cap
        free = [r for r in range(active) if counts[r] < cap]
        total = sum(weight[r] for r in free)
        before = left
        for r in free:
            take = min(cap - counts[r], int(before * weight[r] / total), left)
            counts[r] += take
            left -= take
        if left == before:  # less than one each: the heaviest take it
            for r in free[:left]:
                counts[r] += 1
            left -= min(left, len(free))
    return counts + [0] * (groups - active), entries


def _row_bytes(case, fmt, cols):
    """Bytes of one weight row of `cols` values with its scales."""
    if fmt == "dense":
        return 2 * cols
    if fmt == "affine":
        return cols * case["bits"] // 8 + cols // case["group"] * 2 * _DTYPES[case["params"]].itemsize
    return (cols // 2 if fmt == "mxfp4" else cols) + cols // 32


def work(case):
    tokens, rows, cols, kind = case["tokens"], case.get("rows"), case.get("cols"), case["kind"]
    if kind == "router":
        experts, k, size = case["groups"], case["top_k"], _DTYPES[case["dtype"]].itemsize
        out = tokens * k * 12
        if case["train"]:  # dw read, the logits' gradient written
            out += tokens * (4 * k + size * experts)
        return {"bytes": tokens * experts * size + out, "flops": tokens * experts * 4}
    counts, entries = _routing(case)
    active = sum(1 for c in counts if c)
    if kind == "decode":
        weight = active * (2 * rows * _row_bytes(case, case["format"], cols) +
                           cols * _row_bytes(case, case["format"], rows))
        return {"bytes": weight + 4 * tokens * cols + 12 * entries,
                "flops": 6 * entries * rows * cols}
    size = 2 * tokens * cols + active * rows * _row_bytes(case, "affine", cols) + 2 * entries * rows
    index = 4 * entries if case["top_k"] else 0
    offsets = 4 * (case["groups"] + 1) if case["groups"] else 0
    return {"bytes": size + index + offsets, "flops": 2 * entries * rows * cols}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------


def _rows(tokens, cols, g):
    """Hidden states: normal, each channel with a scale of its own."""
    scale = torch.exp(0.5 * torch.randn(cols, generator=g, device=DEV))
    x = torch.empty(tokens, cols, device=DEV)
    x.normal_(generator=g)
    return x.mul_(scale)


def _words(q, bits):
    """uint8 codes, `bits` each, low bits first, as int32 words."""
    per = 8 // bits
    out = q[..., 0::per].clone()
    for i in range(1, per):
        out |= q[..., i::per] << (bits * i)
    return out.view(torch.int32)


def _weight(case, fmt, shape, g):
    """A weight [G, N, K] of standard deviation about K^-0.5 in its format."""
    groups, rows, cols = shape
    dev = cols**-0.5
    if fmt == "dense":
        w = torch.empty(shape, dtype=_DTYPES[case["dtype"]], device=DEV)
        for part in w:
            part.copy_(torch.randn(rows, cols, generator=g, device=DEV) * dev)
        return w
    if fmt == "affine":
        bits, span = case["bits"], cols // case["group"]
        top = 2**bits - 1
        packed = torch.empty(groups, rows, cols * bits // 32, dtype=torch.int32, device=DEV)
        for part in packed:
            q = torch.randn(rows, cols, generator=g, device=DEV) * (top / 5) + top / 2
            part.copy_(_words(q.round_().clamp_(0, top).to(torch.uint8), bits))
        s = (torch.rand(groups, rows, span, generator=g, device=DEV) + 0.5) * (5 * dev / top)
        b = -s * (top / 2) * (1 + 0.1 * torch.randn(groups, rows, span, generator=g, device=DEV))
        dt = _DTYPES[case["params"]]
        return packed, s.to(dt), b.to(dt)
    bits = 4 if fmt == "mxfp4" else 8
    packed = torch.empty(groups, rows, cols * bits // 32, dtype=torch.int32, device=DEV)
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV)
    for part in packed:
        w = torch.randn(rows, cols, generator=g, device=DEV)
        if bits == 8:
            q = (w * 96).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        else:
            q = torch.bucketize(w.abs() * 1.7, edges).to(torch.uint8) + (w < 0).to(torch.uint8) * 8
        part.copy_(_words(q, bits))
    mid = 127 + round(math.log2(dev / (1.7 if bits == 4 else 96)))
    scales = torch.randint(mid - 1, mid + 2, (groups, rows, cols // 32), generator=g, device=DEV,
                           dtype=torch.uint8)
    return packed, scales


def _pick(weight, e):
    return weight[e] if isinstance(weight, torch.Tensor) else tuple(t[e] for t in weight)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 1000003 + 17)
    kind, tokens, cols, rows = case["kind"], case["tokens"], case.get("cols"), case.get("rows")
    top_k, dtype = case["top_k"], _DTYPES[case["dtype"]]
    if kind == "router":
        experts = case["groups"]
        logits = torch.randn(tokens, experts, generator=g, device=DEV) * 2
        if case["masked"]:  # each row may use half of `masked` groups of experts
            keep = torch.rand(tokens, case["masked"], generator=g, device=DEV)
            keep = keep <= keep.sort(dim=1).values[:, case["masked"] // 2 - 1:case["masked"] // 2]
            group = torch.arange(experts, device=DEV) * case["masked"] // experts
            logits.masked_fill_(~keep[:, group], -math.inf)
        st = {"case": case, "logits": logits.to(dtype)}
        if case["train"]:
            st["dw"] = torch.randn(tokens, top_k, generator=g, device=DEV)
        return st
    st = {"case": case, "x": _rows(tokens, cols, g).to(dtype)}
    counts, entries = _routing(case)
    groups = max(case["groups"], 1)
    order = random.Random(seed).sample(range(groups), groups)
    per_expert = [0] * groups
    for r, e in enumerate(order):
        per_expert[e] = counts[r]
    bounds = [0]
    for c in per_expert:
        bounds.append(bounds[-1] + c)
    st["bounds"] = bounds  # the same offsets on the host, for the plain form's loop
    st["offsets"] = torch.tensor(bounds, dtype=torch.int32, device=DEV) if case["groups"] else None
    st["row_index"] = None
    if top_k:
        # expert e takes a run of its count from one endless list of the tokens
        # (in an order of the seed's): no expert gets a token twice. A stable
        # sort by expert leaves an expert's rows in the tokens' order.
        perm = torch.randperm(tokens, generator=g, device=DEV)
        at = torch.arange(entries, device=DEV)
        expert = torch.bucketize(at, torch.tensor(bounds[1:], device=DEV), right=True)
        key = torch.sort(expert * tokens + perm[at % tokens]).values
        st["row_index"] = (key % tokens).to(torch.int32)
    if kind == "affine":
        w = _weight(case, "affine", (groups, rows, cols), g)
        st["weight"] = w if case["groups"] else tuple(t[0] for t in w)
        return st
    # every row's experts, in an order of their own, with the router's weights
    key = (key % tokens) * groups + key // tokens
    index = (key.sort().values % groups).view(tokens, top_k)
    mix = torch.rand(tokens, top_k, generator=g, device=DEV).argsort(dim=1)
    st["index"] = index.gather(1, mix)
    st["weights"] = torch.softmax(torch.randn(tokens, top_k, generator=g, device=DEV), dim=1)
    st["gate_up"] = _weight(case, case["format"], (groups, 2 * rows, cols), g)
    st["down"] = _weight(case, case["format"], (groups, cols, rows), g)
    if own:
        st["layer"] = _layer(st)
    return st


def _layer(st):
    return _package()[0].ExpertMLP(st["gate_up"], st["down"], st["case"]["format"])


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------


def run(st):
    case = st["case"]
    return (_run_own if own else _run_plain)(st, case, case["kind"])


def _run_own(st, case, kind):
    experts, lin = _package()
    if kind == "affine":
        return lin.affine_linear(st["x"], *st["weight"], case["bits"], st["offsets"],
                                 st["row_index"], validate=False)
    if kind == "decode":
        layer = st["layer"] if "layer" in st else _layer(st)
        return layer.decode(st["x"], st["index"], st["weights"])
    index, weights = experts.top_k_softmax(st["logits"], case["top_k"], case["renormalize"])
    if not case["train"]:
        return index, weights
    return index, weights, experts.top_k_softmax_grad(st["dw"], st["logits"], index,
                                                      case["renormalize"])


def _run_plain(st, case, kind):
    if kind == "router":
        return _plain_router(st, case)
    x = st["x"]
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=x.device)
    b = st["bounds"]
    spans = [(e, b[e], b[e + 1]) for e in range(len(b) - 1) if b[e + 1] > b[e]]
    if kind == "affine":
        xs = x if st["row_index"] is None else x[st["row_index"].long()]
        y = torch.empty(xs.shape[0], case["rows"], dtype=x.dtype, device=x.device)
        for e, lo, hi in spans:
            w = _pick(st["weight"], e) if case["groups"] else st["weight"]
            y[lo:hi] = (xs[lo:hi].float() @ _plain_decode(case, "affine", w, table).t()).to(x.dtype)
        return y
    fmt, inner = case["format"], case["rows"]
    out = torch.zeros(x.shape, device=x.device)
    for e, lo, hi in spans:
        rows = st["row_index"][lo:hi].long()
        h = x[rows].float() @ _plain_decode(case, fmt, _pick(st["gate_up"], e), table).t()
        gate, up = h[:, :inner], h[:, inner:]
        act = gate / (1 + torch.exp(-gate)) * up
        y = act @ _plain_decode(case, fmt, _pick(st["down"], e), table).t()
        weight = (st["weights"][rows] * (st["index"][rows] == e)).sum(1, keepdim=True)
        out[rows] += y * weight
    return out.to(x.dtype)


def _plain_decode(case, fmt, w, table):
    """One expert's weight in 32 bits."""
    if fmt == "dense":
        return w.float()
    codes = w[0].view(torch.uint8)
    if fmt == "affine":
        bits = case["bits"]
        q = torch.stack([(codes >> (bits * i)) & (2**bits - 1) for i in range(8 // bits)], dim=-1)
        q = q.view(*w[1].shape, case["group"]).float()
        return (q * w[1].float().unsqueeze(-1) + w[2].float().unsqueeze(-1)).view(w[1].shape[0], -1)
    if fmt == "mxfp8":
        v = codes.view(torch.float8_e4m3fn).float()
    else:
        v = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), dim=-1)
    v = v.view(*w[1].shape, 32) * torch.pow(2.0, w[1].float() - 127.0).unsqueeze(-1)
    return v.view(w[1].shape[0], -1)


def _plain_router(st, case):
    f = st["logits"].float()
    k = case["top_k"]
    s = torch.sort(f, dim=1, descending=True, stable=True)
    values, index = s.values[:, :k], s.indices[:, :k]
    chosen = values > -math.inf
    top = torch.where(chosen[:, :1], values[:, :1], 0.0)
    ex = torch.exp(values - top)
    every = ex if case["renormalize"] else torch.exp(f - top)
    total = every.sum(1, keepdim=True)
    total = torch.where(total > 0, total, 1.0)
    weights = ex / total
    out = torch.where(chosen, index, -1), weights
    if not case["train"]:
        return out
    dot = (weights * st["dw"]).sum(1, keepdim=True)
    grad = torch.zeros_like(f) if case["renormalize"] else -(every / total) * dot
    add = weights * (st["dw"] - dot if case["renormalize"] else st["dw"])
    return *out, grad.scatter_add(1, index, add).to(st["logits"].dtype)


# --------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "router":
        return _exact_router(st, case)
    x, bounds = st["x"].double(), st["bounds"]
    decode = case["kind"] == "decode"
    out = torch.zeros(*x.shape, dtype=torch.float64, device=DEV) if decode else \
        torch.empty(bounds[-1], case["rows"], dtype=torch.float64, device=DEV)
    for e in range(len(bounds) - 1):
        lo, hi = bounds[e], bounds[e + 1]
        if lo == hi:
            continue
        if not decode:
            idx = torch.arange(lo, hi, device=DEV)
            if st["row_index"] is not None:
                idx = st["row_index"][lo:hi].long()
            w = st["weight"] if not case["groups"] else _pick(st["weight"], e)
            torch.mm(x[idx], _exact_weight(case, "affine", w).t(), out=out[lo:hi])
            continue
        t, j = torch.nonzero(st["index"] == e, as_tuple=True)
        h = torch.mm(x[t], _exact_weight(case, case["format"], _pick(st["gate_up"], e)).t())
        gate, up = h.split(case["rows"], dim=1)
        h = torch.mm(gate * torch.sigmoid(gate) * up,
                     _exact_weight(case, case["format"], _pick(st["down"], e)).t())
        out[t] += h * st["weights"].double()[t, j][:, None]  # an expert has a row once
    return out


def _exact_weight(case, fmt, w):
    if fmt == "dense":
        return w.double()
    words = w[0].long() & 0xFFFFFFFF
    bits = case["bits"] if fmt == "affine" else 4 if fmt == "mxfp4" else 8
    shift = torch.arange(0, 32, bits, device=DEV)
    code = ((words[..., None] >> shift) & (2**bits - 1)).flatten(1)
    if fmt == "affine":
        s, b = (p.double().repeat_interleave(case["group"], dim=1) for p in w[1:])
        return torch.addcmul(b, code.double(), s)
    # sign, exponent, mantissa: (-1)^s 2^(max(e, 1) - bias) ([e > 0] + m / 2^man)
    man, bias = (1, 1) if bits == 4 else (3, 7)
    sign = 1.0 - 2.0 * (code >> (bits - 1)).double()
    exp = (code >> man) & (2 ** (bits - 1 - man) - 1)
    frac = (code & (2**man - 1)).double() / 2**man + (exp > 0).double()
    value = sign * frac * torch.exp2((exp.clamp(min=1) - bias).double())
    return value * torch.exp2(w[1].double() - 127).repeat_interleave(32, dim=1)


def _exact_router(st, case):
    left = st["logits"].double()
    prob = torch.softmax(left, dim=1)
    if not case["renormalize"]:
        prob = torch.where(left.amax(1, keepdim=True) > -math.inf, prob, 0.0)
    left = left.clone()
    ids = torch.arange(case["groups"], device=DEV)
    index, weights = [], []
    for _ in range(case["top_k"]):  # the largest that is left, the first of equal ones
        best = left.amax(1, keepdim=True)
        e = torch.where(left == best, ids, case["groups"]).amin(1, keepdim=True)
        some = best > -math.inf
        index.append(torch.where(some, e, -1))
        weights.append(torch.where(some, prob.gather(1, e), 0.0))
        left.scatter_(1, e, -math.inf)
    index, weights = torch.cat(index, 1), torch.cat(weights, 1)
    if case["renormalize"]:
        total = weights.sum(1, keepdim=True)
        weights = torch.where(total > 0, weights / total, 0.0)
    if not case["train"]:
        return index, weights
    # d w_j / d l_e = w_j ([e = j] - p_e), p the softmax that the weights come from
    grads = []
    for a in range(0, st["logits"].shape[0], 4096):
        sl = slice(a, a + 4096)
        hit = (index[sl, :, None] == ids).double()
        wd = weights[sl] * st["dw"][sl].double()
        p = (weights[sl][..., None] * hit).sum(1) if case["renormalize"] else prob[sl]
        grads.append((wd[..., None] * hit).sum(1) - p * wd.sum(1)[:, None])
    return index, weights, torch.cat(grads)
