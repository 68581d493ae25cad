"""Plain 64-bit forms of the norm, the routing and the experts' products, and the bounds of their kernels' errors."""

import math

import torch

#: half a unit in the last place, relative; and half of the smallest step of all
HALF_ULP = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
E2M1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def rounded(want, slack, dtype):
    """How far an output of `dtype` may be from `want`, which the kernel knows to within `slack`: one rounding, of a value that is off by
    as much; 2^-25: fp16's smallest steps."""
    return HALF_ULP[dtype] * (want.abs() + slack) + slack * 1.01 + 2.0**-25


def agrees(got, want, slack, dtype):
    """Whether an output is as near to `want` as it can be.  From half a step beyond the type's largest number on, rounding gives
    infinity; where the formula gives NaN (an infinity over the root of its row's squares), so does the kernel."""
    got, want, slack = got.double().cpu(), want.cpu(), torch.as_tensor(slack, dtype=torch.float64).cpu().expand(want.shape)
    top = torch.finfo(dtype).max * (1 + HALF_ULP[dtype] / 2)  # (the last step is twice the half, relative to the next power of two)
    near = (got - want).abs() <= rounded(want, slack, dtype)
    over = (want.abs() + slack >= top) & (got == want.sign() * math.inf)
    return bool((near | over | (torch.isnan(got) & torch.isnan(want))).all())


def norm(x, residual, weight, eps):
    """y and h in 64 bits, and the bounds of y's and h's errors before they are rounded."""
    x = x.double()
    h = x if residual is None else x + residual.double()
    mean = (h * h).mean(dim=1, keepdim=True)
    y = h / torch.sqrt(mean + eps) * weight.double()
    # h one rounding; a lane adds up to 32 squares one by one and 10 levels of lanes follow: 42 roundings of the sum, half as much
    # of its root; mean, sum with eps, root, quotient, two products: 6 more
    return y, h, 30 * 2.0**-24 * y.abs(), (0 if residual is None else 2.0**-24) * h.abs()


def route(logits, bias, top_k, scores="softmax", groups=1, top_groups=1, group_score="max", renormalize=True, factor=1.0):
    """ids and weights, by the definition, a token at a time."""
    x = logits.double().cpu()
    b = None if bias is None else bias.double().cpu()
    ids, weights = [], []
    for row in x:
        if scores == "sigmoid":
            score = torch.sigmoid(row)
        else:
            most = row.max()
            score = torch.exp(row - (0.0 if most == -math.inf else most))
            total = score.sum()
            score = score / total if total != 0 else score
        key = (row if b is None else score + b).tolist()
        key = [math.inf if math.isnan(k) else k for k in key]
        by = key if group_score == "max" or b is not None else [math.inf if math.isnan(s) else s for s in score.tolist()]
        size, allowed = len(key) // groups, set(range(groups))
        if groups > 1:
            of = [sorted(by[g * size : (g + 1) * size], reverse=True)[: 1 if group_score == "max" else 2] for g in range(groups)]
            of = [sum(v) for v in of]
            allowed = set(sorted(range(groups), key=lambda g: (-of[g], g))[:top_groups])
        chosen = sorted((e for e in range(len(key)) if e // size in allowed), key=lambda e: (-key[e], e))[:top_k]
        w = score[chosen]
        if renormalize:
            w = w / w.sum() if w.sum() != 0 else torch.zeros_like(w)
        ids.append(chosen)
        weights.append(w * factor)
    return torch.tensor(ids, dtype=torch.int32), torch.stack(weights)


def order(ids, experts, first=0):
    """The pairs sorted by expert, and where each begins."""
    flat = ids.flatten().tolist()
    rows = [[p for p, e in enumerate(flat) if e == first + n] for n in range(experts)]
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + len(r))
    out = [p for r in rows for p in r]
    return torch.tensor(out + [-1] * (len(flat) - len(out)), dtype=torch.int32), torch.tensor(starts, dtype=torch.int32)


class Weights:
    """Random packed weights of some experts, as the kernels take them, and their values."""

    def __init__(self, gen, experts, rows, K, weight_format="uint4", group_size=None, with_zeros=False, with_bias=False, device="cpu", whole=False):
        mx = weight_format == "mxfp4"
        self.dtype = torch.bfloat16 if mx else torch.float16
        per = 32 if mx else group_size or 128
        codes = torch.randint(0, 16, (experts, rows, K), generator=gen, dtype=torch.uint8)
        packed = codes[..., 0::2] | codes[..., 1::2] << 4
        self.zeros = self.bias = None
        if mx:
            self.packed = packed
            self.scale = torch.randint(127 if whole else 119, 129 if whole else 124, (experts, rows, K // 32), generator=gen, dtype=torch.uint8)
            value = E2M1[codes.long()] * 2.0 ** (self.scale.double() - 127).repeat_interleave(32, dim=2)
        else:
            self.packed = packed.view(torch.int8)
            shape = (experts, rows, K // per)
            self.scale = (torch.ones(shape) if whole else (torch.rand(shape, generator=gen) + 0.5) / 16).half()
            zero = 8.0
            if with_zeros:
                self.zeros = torch.randint(0, 16, shape, generator=gen).half()
                zero = self.zeros.double().repeat_interleave(per, dim=2)
            value = ((codes.double() - zero) * self.scale.double().repeat_interleave(per, dim=2)).half().double()
        if with_bias:
            self.bias = (torch.randint(-8, 9, (experts, rows), generator=gen).double() if whole else torch.randn((experts, rows), generator=gen)).to(self.dtype)
        self.value = value
        self.packed, self.scale = self.packed.to(device), self.scale.to(device)
        self.zeros = None if self.zeros is None else self.zeros.to(device)
        self.on_device = [t for t in (self.packed, self.scale, self.zeros, None if self.bias is None else self.bias.to(device)) if t is not None]

    def product(self, rows, e):
        """rows [n, K] times an expert's weights, and the bound of an fp32 sum's error: K terms, one by one, and the bias."""
        rows = rows.double()
        y, size = rows @ self.value[e].t(), rows.abs() @ self.value[e].abs().t()
        if self.bias is not None:
            y, size = y + self.bias[e].double(), size + self.bias[e].double().abs()
        return y, (rows.shape[1] + 8) * 2.0**-24 * size


def up(x, w, order, starts, top_k, N, activation):
    """h of every row, NaN behind the last one, and the bound of its error before it is rounded."""
    pairs = len(order)
    out, slack = torch.full((pairs, N), math.nan, dtype=torch.float64), torch.zeros((pairs, N), dtype=torch.float64)
    for e in range(len(starts) - 1):
        r = slice(int(starts[e]), int(starts[e + 1]))
        if r.start == r.stop:
            continue
        y, off = w.product(x.cpu()[order[r].long() // top_k], e)
        gate, u, gate_off, u_off = y[:, :N], y[:, N:], off[:, :N], off[:, N:]
        inner = gate if activation == "silu" else 2 * math.sqrt(2 / math.pi) * (gate + 0.044715 * gate**3)
        act = gate / (1 + torch.exp(-inner))
        # the activations' slopes stay below 1.13; an exponential of x is off by |x| roundings, and six follow
        act_off = 1.13 * gate_off + act.abs() * (2 * inner.abs() + 6) * 2.0**-24
        out[r] = act * u
        slack[r] = act_off * (u.abs() + u_off) + act.abs() * u_off + 2.0**-24 * out[r].abs()
    return out, slack


def down(h, w, order, starts, weights, tokens, residual):
    """y, and the bound of its error before it is rounded."""
    top_k, weights = weights.shape[1], weights.double().cpu().flatten()
    N = w.value.shape[1]
    out, size, slack = (torch.zeros((tokens, N), dtype=torch.float64) for _ in range(3))
    for e in range(len(starts) - 1):
        r = slice(int(starts[e]), int(starts[e + 1]))
        if r.start == r.stop:
            continue
        pair = order[r].long()
        y, off = w.product(h[r].cpu(), e)
        # (an expert's rows may name a token twice)
        out.index_add_(0, pair // top_k, y * weights[pair][:, None])
        size.index_add_(0, pair // top_k, y.abs() * weights[pair].abs()[:, None])
        slack.index_add_(0, pair // top_k, off * weights[pair].abs()[:, None])
    if residual is not None:
        out, size = out + residual.double().cpu(), size + residual.double().cpu().abs()
    return out, slack + (top_k + 2) * 2.0**-24 * size
