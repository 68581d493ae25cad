"""What the operators of the rest of a decoder block around 4-bit weights are measured on: the root-mean-square norm with the
residual's addition, the routing of tokens to experts, and the experts' two products.

``listed()`` names twelve cases, ``draw(rng)`` gives more of the same ranges; ``prepare`` makes what a serving program holds before
the call, ``run`` is one pass through one operator: with ``own`` through the package's kernel objects, else in plain torch in 32 bits
(64 where experts are told apart by scores).  ``exact`` is the definition in 64 bits.

A weight is what the package's dense layers multiply with: ``(q - 8) * s`` or ``(q - z) * s`` rounded to fp16, or an e2m1 code times a
power of two.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
EPS = 1e-6
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TINY = 1e-5  # an int8 row's largest magnitude counts as this much at least


def _norm(name, rows, dim, dtype, residual=True, int8=False, wider=0):
    return {"name": name, "kind": "norm", "rows": rows, "dim": dim, "dtype": dtype, "residual": residual, "int8": int8, "wider": wider}


def _route(name, tokens, experts, top_k, dtype, scores="softmax", bias=False, groups=1, top_groups=1, group_score="max", renormalize=True, factor=1.0):
    return {"name": name, "kind": "route", "tokens": tokens, "experts": experts, "top_k": top_k, "dtype": dtype, "scores": scores, "bias": bias,
            "groups": groups, "top_groups": top_groups, "group_score": group_score, "renormalize": renormalize, "factor": factor}


def _up(name, tokens, experts, top_k, N, K, weights, group=128, zeros=False, activation="silu", bias=False):
    return {"name": name, "kind": "up", "tokens": tokens, "experts": experts, "top_k": top_k, "N": N, "K": K, "weights": weights, "group": group,
            "zeros": zeros, "activation": activation, "bias": bias}


def _down(name, tokens, experts, top_k, N, K, weights, group=128, zeros=False, bias=False, residual=False):
    return {"name": name, "kind": "down", "tokens": tokens, "experts": experts, "top_k": top_k, "N": N, "K": K, "weights": weights, "group": group,
            "zeros": zeros, "bias": bias, "residual": residual}


def listed():
    return [
        # the norm in front of one new token's projections, with the residual's addition: the smallest call, latency counts
        _norm("norm one token", 1, 4096, "float16"),
        # a batch of prompts in front of an int8 x 2-bit projection: int8 codes, a scale a row
        _norm("norm int8", 2048, 8192, "float16", int8=True),
        # a long prompt of odd length
        _norm("norm prompt", 7999, 5120, "bfloat16"),
        # one new token chooses eight of 128 experts: latency counts
        _route("route one token", 1, 128, 8, "float32"),
        # a chunk of prompts: sigmoid scores, a bias for balance, four of eight groups, eight of 256 experts
        _route("route groups", 8192, 256, 8, "float32", "sigmoid", True, 8, 4, "sum2", True, 2.5),
        # an odd number of tokens and of experts, logits in 16 bits, weights as the softmax has them
        _route("route odd", 1021, 60, 4, "bfloat16", renormalize=False),
        # one new token through the gate and up projections of its eight experts: latency and the weights' bytes count
        _up("up one token", 1, 128, 8, 1024, 4096, "uint4"),
        # a serving batch, some tokens an expert: rows of weights that are no multiple of a cache line, biases
        _up("up batch mxfp4", 64, 32, 4, 2880, 2880, "mxfp4", bias=True),
        # a chunk of prompts over a few large experts
        _up("up prompt", 4096, 8, 2, 14336, 4096, "uint4"),
        # one new token back from its experts, weighted and summed
        _down("down one token", 1, 128, 8, 4096, 1024, "uint4", residual=True),
        # the serving batch's way back, onto the residual
        _down("down batch mxfp4", 64, 32, 4, 2880, 2880, "mxfp4", bias=True, residual=True),
        # the chunk's way back, zero points
        _down("down prompt", 4096, 8, 2, 4096, 14336, "uint4", zeros=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(lo * ((hi + 1) / lo) ** rng.random())))


def _drawn_norm(rng):
    dim = rng.choice((64, 128, 1024, 2048, 2880, 4096, 5120, 8192, 11008, 13824, 14336, 16384, 8 * rng.randint(8, 2048)))
    rows = _log(rng, 1, min(16384, 7999 * 5120 // dim))
    int8 = rng.random() < 0.3 and rows * dim <= 2048 * 8192
    return _norm("", rows, dim, rng.choice(("float16", "bfloat16")), rng.random() < 0.6, int8, rng.choice((0, 0, 0, 64)))


def _drawn_route(rng):
    experts = rng.choice((8, 16, 60, 64, 128, 160, 256, 384, rng.randint(4, 512)))
    top_k = rng.choice((1, 2, 4, 6, 8, 8))
    groups, top_groups, score = 1, 1, "max"
    if experts % 8 == 0 and experts >= 64 and rng.random() < 0.4:
        groups = rng.choice((4, 8))
        top_groups, score = rng.randint(2, groups), rng.choice(("max", "sum2"))
    tokens = _log(rng, 1, min(8192, 8192 * 256 // experts))
    return _route("", tokens, experts, min(top_k, experts), rng.choice(("float32", "float32", "float16", "bfloat16")), rng.choice(("softmax", "sigmoid")),
                  rng.random() < 0.4, groups, top_groups, score, rng.random() < 0.7, rng.choice((1.0, 2.5)))


def _drawn_product(rng):
    weights = rng.choice(("uint4", "mxfp4"))
    up = rng.random() < 0.5
    unit = 128 if weights == "uint4" else 64
    wide, narrow = (rng.choice((1024, 2048, 2880, 4096, 5120, 8192, unit * rng.randint(4, 64))) // unit * unit for _ in range(2))
    experts = rng.choice((4, 8, 16, 32, 64, 128, rng.randint(3, 160)))
    top_k = min(rng.choice((1, 2, 4, 6, 8)), experts)
    while experts * wide * narrow * (2 if up else 1) > 8 * 28672 * 4096:
        experts = (experts + 1) // 2
        top_k = min(top_k, experts)
    # nothing costs more than the largest listed case of its kind
    tokens = _log(rng, 1, max(1, min(4096, 4096 * 2 * 14336 * 4096 // (wide * narrow * top_k))))
    zeros = weights == "uint4" and rng.random() < 0.4
    group = rng.choice((32, 64, 128, 128)) if weights == "uint4" else 32
    if up:
        return _up("", tokens, experts, top_k, narrow, wide, weights, group, zeros, rng.choice(("silu", "silu", "gelu")), rng.random() < 0.3)
    return _down("", tokens, experts, top_k, wide, narrow, weights, group, zeros, rng.random() < 0.3, rng.random() < 0.5)


def draw(rng):
    case = rng.choice((_drawn_norm, _drawn_route, _drawn_product, _drawn_product))(rng)
    del case["name"]
    return case


# ---- inputs --------------------------------------------------------------------------------------------------------------


class _Inputs:
    """Random inputs on the GPU, from the seed alone."""

    def __init__(self, seed):
        self.dev = torch.device("cuda")
        self.gen = torch.Generator(device=self.dev)
        self.gen.manual_seed(seed)

    def normal(self, *shape, dtype=torch.float32):
        return torch.randn(shape, dtype=torch.float32, device=self.dev, generator=self.gen).to(dtype)

    def uniform(self, *shape):
        return torch.rand(shape, dtype=torch.float32, device=self.dev, generator=self.gen)

    def ints(self, lo, hi, *shape, dtype=torch.int32):
        return torch.randint(lo, hi, shape, device=self.dev, generator=self.gen, dtype=dtype)

    def weights(self, case, rows):
        """Every expert's packed weights [experts, rows, K / 2], their scales and, with zeros, zero points."""
        experts, K, groups = case["experts"], case["K"], case["K"] // case["group"]
        packed = self.ints(0, 256, experts, rows, K // 2, dtype=torch.uint8)
        if case["weights"] == "mxfp4":  # weights of about K ** -0.5, a few powers of two either way
            middle = 127 - round(math.log2(2.7 * math.sqrt(K)))
            return packed, self.ints(middle - 1, middle + 2, experts, rows, K // 32, dtype=torch.uint8), None
        scale = ((0.5 + self.uniform(experts, rows, groups)) * (K**-0.5 / 4.6)).half()
        return packed.view(torch.int8), scale, self.ints(5, 11, experts, rows, groups).half() if case["zeros"] else None


def prepare(case, seed):
    x = _Inputs(seed)
    state = {"case": dict(case)}
    if case["kind"] == "norm":
        dtype, rows, dim = DTYPES[case["dtype"]], case["rows"], case["dim"]
        # a stream as it is some blocks deep: rows of unlike size, some channels far ahead of the others
        channels = torch.where(x.uniform(dim) < 0.01, 20.0, 1.0)
        wide = (x.normal(rows, dim + case["wider"]) * torch.cat([channels, channels.new_ones(case["wider"])])).to(dtype)
        state["x"] = wide[:, :dim]
        state["residual"] = (x.normal(rows, dim) * channels * (0.5 + 4 * x.uniform(rows, 1))).to(dtype) if case["residual"] else None
        state["weight"] = (1 + 0.2 * x.normal(dim)).to(dtype)
        return state
    if case["kind"] == "route":
        state["logits"] = (1.5 * x.normal(case["tokens"], case["experts"])).to(DTYPES[case["dtype"]])
        state["bias"] = 0.1 * x.normal(case["experts"]) if case["bias"] else None
        return state
    tokens, experts, k = case["tokens"], case["experts"], case["top_k"]
    dtype = torch.float16 if case["weights"] == "uint4" else torch.bfloat16
    up = case["kind"] == "up"
    # some experts are asked for more than others
    wish = x.normal(tokens, experts) + 0.7 * x.normal(experts)
    ids = wish.argsort(dim=1, descending=True)[:, :k].int().contiguous()
    weights = torch.softmax(wish.gather(1, ids.long()), dim=1)
    flat = ids.flatten().long()
    order = flat.argsort(stable=True)
    count = torch.bincount(flat, minlength=experts)
    state["ids"], state["weights"] = ids, weights
    state["order"], state["starts"] = order.int(), torch.cat([count.new_zeros(1), count.cumsum(0)]).int()
    rows = (2 if up else 1) * case["N"]
    state["packed"], state["scale"], state["zeros"] = x.weights(case, rows)
    state["bias"] = x.normal(experts, rows, dtype=dtype) * 0.1 if case["bias"] else None
    if up:
        state["x"] = x.normal(tokens, case["K"], dtype=dtype)
    else:  # products of two projections, one of them activated
        h = x.normal(tokens * k, case["K"])
        state["h"] = (h * torch.sigmoid(h) * x.normal(tokens * k, case["K"])).to(dtype)
        state["residual"] = x.normal(tokens, case["N"], dtype=dtype) if case["residual"] else None
    # the plain form's: the experts that have rows, and where each row of the sorted order lies among theirs
    live = count.nonzero()[:, 0]
    state["live"], most = live, int(count.max())
    place = torch.arange(tokens * k, device=x.dev) - state["starts"].long()[flat[order]]
    lane = torch.full((experts,), -1, device=x.dev, dtype=torch.long)
    lane[live] = torch.arange(len(live), device=x.dev)
    state["place"], state["most"] = lane[flat[order]] * most + place, most
    return state


# ---- the plain forms: torch in 32 bits -----------------------------------------------------------------------------------


def _plain_norm(state):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    h = state["x"].float()
    if case["residual"]:
        h = h + state["residual"].float()
    y = h * torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS) * state["weight"].float()
    out = {}
    if case["int8"]:
        s = 127.0 / y.abs().amax(dim=1, keepdim=True).clamp(min=TINY)
        out["y"], out["scale"] = ((y * s).round().clamp(-127, 127) / s).to(dtype), s[:, 0]
    else:
        out["y"] = y.to(dtype)
    if case["residual"]:
        out["sum"] = h.to(dtype)
    return out


def _order(ids, experts):
    flat = ids.flatten().long()
    count = (flat[:, None] == torch.arange(experts, device=flat.device)).sum(dim=0)
    return flat.argsort(stable=True).int(), torch.cat([count.new_zeros(1), count.cumsum(0)]).int()


def _plain_route(state):
    case = state["case"]
    logits = state["logits"].float()
    # scores that choose, in 64 bits: two of them may be closer than 32 tell
    wide = logits.double()
    score = torch.sigmoid(wide) if case["scores"] == "sigmoid" else torch.softmax(wide, dim=1)
    key = wide if state["bias"] is None else score + state["bias"].double()
    if case["groups"] > 1:
        by = key if case["group_score"] == "max" else score if state["bias"] is None else key
        members = by.view(by.shape[0], case["groups"], -1).sort(dim=2, descending=True).values
        group = members[..., 0] if case["group_score"] == "max" else members[..., :2].sum(dim=2)
        rank = group.argsort(dim=1, descending=True, stable=True).argsort(dim=1)
        chosen = (rank < case["top_groups"]).repeat_interleave(case["experts"] // case["groups"], dim=1)
        key = key.masked_fill(~chosen, -math.inf)
    ids = key.argsort(dim=1, descending=True, stable=True)[:, : case["top_k"]]
    if case["scores"] == "sigmoid":
        weights = torch.sigmoid(logits).gather(1, ids)
    else:
        weights = torch.softmax(logits, dim=1).gather(1, ids)
    if case["renormalize"]:
        weights = weights / weights.sum(dim=1, keepdim=True)
    order, starts = _order(ids, case["experts"])
    return {"weights": weights * case["factor"], "ids": ids.int(), "order": order, "starts": starts}


def _plain_weights(state):
    """The weights of the experts that have rows, [experts, rows, K], in 32 bits."""
    case = state["case"]
    packed = state["packed"][state["live"]].view(torch.uint8)
    codes = torch.stack([packed & 15, packed >> 4], dim=-1).flatten(-2)
    scale = state["scale"][state["live"]]
    if case["weights"] == "mxfp4":
        table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float32, device=codes.device)
        value = table[codes.int()]
        return (value.unflatten(-1, (-1, 32)) * torch.exp2(scale.float() - 127)[..., None]).flatten(-2)
    value = codes.float().unflatten(-1, (-1, case["group"]))
    zero = 8.0 if state["zeros"] is None else state["zeros"][state["live"]].float()[..., None]
    return ((value - zero) * scale.float()[..., None]).flatten(-2).half().float()


def _plain_product(state, rows):
    """Every row of the sorted order times its expert's weights, in 32 bits."""
    w = _plain_weights(state)
    padded = rows.new_zeros((len(state["live"]) * state["most"], rows.shape[1]))
    padded[state["place"]] = rows
    y = torch.matmul(w, padded.view(len(state["live"]), state["most"], -1).transpose(1, 2).contiguous()).transpose(1, 2).contiguous()
    if state["bias"] is not None:
        y = y + state["bias"][state["live"]].float()[:, None]
    return y.flatten(0, 1)[state["place"]]


def _plain_up(state):
    case = state["case"]
    token = (state["order"] // case["top_k"]).long()
    gate, up = _plain_product(state, state["x"].float()[token]).split(case["N"], dim=1)
    if case["activation"] == "silu":
        gate = gate * torch.sigmoid(gate)
    else:
        gate = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate * gate * gate)))
    return (gate * up).to(state["x"].dtype)


def _plain_down(state):
    case = state["case"]
    pairs = _plain_product(state, state["h"].float())
    back = torch.empty_like(pairs)
    back[state["order"].long()] = pairs
    y = (back.view(case["tokens"], case["top_k"], -1) * state["weights"][..., None]).sum(dim=1)
    if state["residual"] is not None:
        y = y + state["residual"].float()
    return y.to(state["h"].dtype)


# ---- the package's kernel objects ----------------------------------------------------------------------------------------


def _kernel(state):
    """The kernel object of a case, which a program makes once and keeps."""
    import tilelang_amd as tl

    case = state["case"]
    if case["kind"] == "norm":
        return tl.rms_norm(case["rows"], case["dim"], eps=EPS, dtype=case["dtype"], residual=case["residual"], int8=case["int8"],
                           row_stride=case["dim"] + case["wider"])
    if case["kind"] == "route":
        return tl.route_experts(case["tokens"], case["experts"], case["top_k"], scores=case["scores"], bias=case["bias"], groups=case["groups"],
                                top_groups=case["top_groups"], group_score=case["group_score"], renormalize=case["renormalize"],
                                factor=case["factor"], dtype=case["dtype"])
    sizes = dict(weight_format=case["weights"], group_size=case["group"] if case["weights"] == "uint4" else None, with_zeros=case["zeros"], with_bias=case["bias"])
    if case["kind"] == "up":
        return tl.experts_up(case["tokens"], case["experts"], case["top_k"], case["N"], case["K"], activation=case["activation"], **sizes)
    return tl.experts_down(case["tokens"], case["experts"], case["top_k"], case["N"], case["K"], residual=case["residual"], **sizes)


def _own(state):
    case, kernel = state["case"], state.get("kernel")
    if kernel is None:
        kernel = state["kernel"] = _kernel(state)
    if case["kind"] == "norm":
        got = kernel(state["x"], *(() if state["residual"] is None else (state["residual"],)), state["weight"])
        got = [got] if isinstance(got, torch.Tensor) else list(got)
        out = {"y": got[0]}
        if case["int8"]:
            # (what the codes stand for, in one pass)
            out = {"y": torch.div(got[0], got[1][:, None], out=torch.empty_like(got[0], dtype=DTYPES[case["dtype"]])), "scale": got[1]}
        return out | ({"sum": got[-1]} if case["residual"] else {})
    if case["kind"] == "route":
        got = kernel(state["logits"], *(() if state["bias"] is None else (state["bias"],)))
        return dict(zip(("weights", "ids", "order", "starts"), got))
    operands = [t for t in (state["packed"], state["scale"], state["zeros"], state["bias"]) if t is not None]
    if case["kind"] == "up":
        return kernel(state["x"], *operands, state["order"], state["starts"])
    return kernel(state["h"], *operands, state["order"], state["starts"], state["ids"], state["weights"],
                  *(() if state["residual"] is None else (state["residual"],)))


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "route": _plain_route, "up": _plain_up, "down": _plain_down}[state["case"]["kind"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------


def _experts_with_rows(case):
    """How many experts some token chooses, where all are chosen alike."""
    E, pairs = case["experts"], case["tokens"] * case["top_k"]
    return min(pairs, round(E * (1 - (1 - case["top_k"] / E) ** case["tokens"])))


def work(case):
    if case["kind"] == "norm":
        values, rows = case["rows"] * case["dim"], case["rows"]
        moved = values * (2 + (4 if case["residual"] else 0) + (1 if case["int8"] else 2)) + case["dim"] * 2 + (4 * rows if case["int8"] else 0)
        return {"bytes": moved, "flops": 5 * values}
    if case["kind"] == "route":
        logits, pairs = case["tokens"] * case["experts"], case["tokens"] * case["top_k"]
        return {"bytes": logits * DTYPES[case["dtype"]].itemsize + pairs * 12 + (case["experts"] + 1) * 4 + (case["experts"] * 4 if case["bias"] else 0),
                "flops": 4 * logits}
    pairs, up = case["tokens"] * case["top_k"], case["kind"] == "up"
    rows = case["N"] * (2 if up else 1)
    scale = 1 / 32 if case["weights"] == "mxfp4" else (4 if case["zeros"] else 2) / case["group"]
    moved = _experts_with_rows(case) * rows * (case["K"] * (0.5 + scale) + (2 if case["bias"] else 0))
    if up:
        moved += 2 * case["tokens"] * case["K"] + 2 * pairs * case["N"] + 4 * pairs
    else:
        moved += 2 * pairs * case["K"] + 2 * case["tokens"] * case["N"] * (2 if case["residual"] else 1) + 12 * pairs
    return {"bytes": int(moved) + 4 * (case["experts"] + 1), "flops": 2 * pairs * rows * case["K"]}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------


def _exact_norm(state):
    case = state["case"]
    out, parts = {}, []
    for lo in range(0, case["rows"], 2048):
        x = state["x"][lo : lo + 2048].double()
        if case["residual"]:
            x = x + state["residual"][lo : lo + 2048].double()
        length = torch.sqrt(torch.linalg.vector_norm(x, dim=1) ** 2 / case["dim"] + EPS)
        y = x / length[:, None] * state["weight"].double()
        s = None
        if case["int8"]:
            s = 127 / torch.linalg.vector_norm(y, ord=math.inf, dim=1).clamp(min=TINY)
            y = torch.round(y * s[:, None]) / s[:, None]
        parts.append((y, s, x))
    out["y"] = torch.cat([p[0] for p in parts])
    if case["int8"]:
        out["scale"] = torch.cat([p[1] for p in parts])
    if case["residual"]:
        out["sum"] = torch.cat([p[2] for p in parts])
    return out


def _ranks(key):
    """How many of a row come before each: the larger ones, and of its equals those of a lower index."""
    n = key.shape[1]
    earlier = torch.arange(n, device=key.device)[None, :] < torch.arange(n, device=key.device)[:, None]
    parts = []
    for lo in range(0, key.shape[0], 256):
        a, b = key[lo : lo + 256, None, :], key[lo : lo + 256, :, None]
        parts.append(((a > b) | ((a == b) & earlier)).sum(dim=2))
    return torch.cat(parts)


def _exact_route(state):
    case = state["case"]
    x = state["logits"].double()
    if case["scores"] == "sigmoid":
        score = 1 / (1 + torch.exp(-x))
    else:
        score = torch.exp(x - torch.logsumexp(x, dim=1, keepdim=True))
    key = x if state["bias"] is None else score + state["bias"].double()
    if case["groups"] > 1:
        by = score if state["bias"] is None and case["group_score"] == "sum2" else key
        each = by.unflatten(1, (case["groups"], -1))
        largest = torch.topk(each, 1 if case["group_score"] == "max" else 2, dim=2).values.sum(dim=2)
        allowed = (_ranks(largest) < case["top_groups"])[..., None].expand(each.shape).flatten(1)
        key = torch.where(allowed, key, -math.inf)
    rank = _ranks(key)
    token, expert = (rank < case["top_k"]).nonzero(as_tuple=True)
    ids = torch.empty((case["tokens"], case["top_k"]), dtype=torch.long, device=x.device)
    ids[token, rank[token, expert]] = expert
    weights = score.gather(1, ids)
    if case["renormalize"]:
        weights = weights / weights.sum(dim=1, keepdim=True)
    chosen = torch.arange(case["experts"], device=x.device)[:, None] == ids.flatten()[None]
    starts = torch.zeros(case["experts"] + 1, dtype=torch.int32, device=x.device)
    starts[1:] = chosen.sum(dim=1).cumsum(0).int()
    return {"weights": weights * case["factor"], "ids": ids.int(), "order": chosen.nonzero()[:, 1].int(), "starts": starts}


def _exact_weights(state, e):
    """An expert's weights, [rows, K], in 64 bits."""
    case = state["case"]
    packed = state["packed"][e].view(torch.uint8).int()
    codes = torch.empty((packed.shape[0], case["K"]), dtype=torch.int32, device=packed.device)
    codes[:, 0::2], codes[:, 1::2] = packed % 16, packed // 16
    per = 32 if case["weights"] == "mxfp4" else case["group"]
    scale = state["scale"][e].double().repeat_interleave(per, dim=1)
    if case["weights"] == "mxfp4":
        sign, exponent, half = 1.0 - 2.0 * (codes // 8), codes // 2 % 4, codes % 2
        size = torch.where(exponent == 0, 0.5 * half, 2.0 ** (exponent.double() - 1) * (1 + 0.5 * half))
        return sign.double() * size * 2.0 ** (scale - 127)
    zero = 8.0 if state["zeros"] is None else state["zeros"][e].double().repeat_interleave(per, dim=1)
    return ((codes - zero) * scale).half().double()


def _exact_up(state):
    case, N = state["case"], state["case"]["N"]
    out = torch.empty((case["tokens"] * case["top_k"], N), dtype=torch.float64, device="cuda")
    starts, token = state["starts"].tolist(), (state["order"] // case["top_k"]).long()
    for e in state["live"].tolist():
        rows = slice(starts[e], starts[e + 1])
        y = state["x"][token[rows]].double() @ _exact_weights(state, e).t()
        if state["bias"] is not None:
            y = y + state["bias"][e].double()
        gate, up = y[:, :N], y[:, N:]
        if case["activation"] == "silu":
            out[rows] = up * gate / (1 + torch.exp(-gate))
        else:  # 0.5 (1 + tanh(u)) = 1 / (1 + exp(-2 u))
            out[rows] = up * gate / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (gate + 0.044715 * gate**3)))
    return out


def _exact_down(state):
    case = state["case"]
    out = torch.zeros((case["tokens"], case["N"]), dtype=torch.float64, device="cuda")
    if state["residual"] is not None:
        out += state["residual"].double()
    starts, weight = state["starts"].tolist(), state["weights"].double().flatten()
    for e in state["live"].tolist():
        rows = slice(starts[e], starts[e + 1])
        pair = state["order"][rows].long()
        y = state["h"][rows].double() @ _exact_weights(state, e).t()
        if state["bias"] is not None:
            y = y + state["bias"][e].double()
        out[pair // case["top_k"]] += y * weight[pair][:, None]  # (an expert has a token once)
    return out


def exact(case, seed):
    return {"norm": _exact_norm, "route": _exact_route, "up": _exact_up, "down": _exact_down}[case["kind"]](prepare(case, seed))
