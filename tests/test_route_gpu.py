"""Routing against its definition in 64 bits: who is chosen is exact, ties and near ties too."""

import math

import pytest
import torch

import block_reference as ref
import tilelang_amd as tl

pytestmark = pytest.mark.gpu

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def _check(logits, bias, top_k, dtype="float32", groups=1, **how):
    tokens, experts = logits.shape
    logits = logits.to(DTYPES[dtype])
    kernel = tl.route_experts(tokens, experts, top_k, bias=bias is not None, dtype=dtype, groups=groups, **how)
    weights, ids, order, starts = kernel(logits.cuda(), *(() if bias is None else (bias.cuda(),)))
    want_ids, want = ref.route(logits, bias, top_k, groups=groups, top_groups=how.pop("top_groups", groups), **how)
    assert torch.equal(ids.cpu(), want_ids)
    # an exponential of x is off by |x| roundings (its argument's) and one, the sum of 1024 by as many as its 26 levels, and the quotients
    finite = logits.double()[torch.isfinite(logits)]
    spread = float(finite.max() - finite.min()) + float(finite.abs().max()) if len(finite) else 0.0
    off = (weights.double().cpu() - want).abs()
    ok = off <= (2 * spread + 60) * 2.0**-24 * want.abs() + 2.0**-126
    assert (ok | (torch.isnan(weights.cpu()) & torch.isnan(want))).all(), off.max()
    want_order, want_starts = ref.order(want_ids, experts)
    assert torch.equal(order.cpu(), want_order) and torch.equal(starts.cpu(), want_starts)
    return ids.cpu(), weights.cpu()


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("tokens,experts,top_k,dtype", [
    (1, 1, 1, "float32"), (1, 128, 8, "float32"), (2, 4, 4, "float16"), (5, 60, 4, "bfloat16"), (33, 8, 2, "float32"), (31, 64, 6, "bfloat16"),
    (64, 5, 1, "bfloat16"), (13, 9, 5, "float32"), (70, 65, 8, "float16"), (257, 160, 6, "float32"), (129, 256, 8, "bfloat16"), (64, 513, 10, "float32"), (40, 1024, 32, "float32"), (1000, 7, 3, "float16"),
])
def test_route(cuda, tokens, experts, top_k, dtype, bias, scores):
    print(f"route {tokens}x{experts} top {top_k} {dtype} bias={bias} {scores}", flush=True)
    gen = torch.Generator().manual_seed(tokens + experts)
    logits = 2 * torch.randn((tokens, experts), generator=gen)
    b = 0.1 * torch.randn(experts, generator=gen) if bias else None
    _check(logits, b, top_k, dtype, scores=scores, renormalize=tokens % 2 == 0, factor=2.5 if experts % 2 else 1.0)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("group_score", ["max", "sum2"])
@pytest.mark.parametrize("tokens,experts,top_k,groups,top_groups", [(3, 256, 8, 8, 4), (50, 16, 2, 4, 1), (20, 64, 4, 64, 5), (21, 160, 6, 8, 3), (9, 12, 12, 3, 3)])
def test_groups(cuda, tokens, experts, top_k, groups, top_groups, group_score, bias, scores):
    print(f"route groups {tokens}x{experts} top {top_k} of {top_groups}/{groups} {group_score} {bias} {scores}", flush=True)
    gen = torch.Generator().manual_seed(experts + groups)
    b = 0.3 * torch.randn(experts, generator=gen) if bias else None
    logits = torch.randn((tokens, experts), generator=gen)
    _check(logits, b, top_k, scores=scores, groups=groups, top_groups=top_groups, group_score=group_score)
    # equal keys everywhere: the lowest index
    _check(logits.round(), None if b is None else torch.zeros(experts), top_k, scores=scores, groups=groups, top_groups=top_groups, group_score=group_score)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_ties(cuda, scores, dtype):
    print(f"route ties {scores} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(4)
    logits = torch.randint(-2, 3, (150, 100), generator=gen).float()
    logits[0] = 0
    for bias in (None, torch.zeros(100), torch.full((100,), -3.0)):
        ids, _ = _check(logits, bias, 8, dtype, scores=scores)
        assert ids[0].tolist() == list(range(8))


@pytest.mark.parametrize("groups,group_score", [(1, "max"), (8, "sum2")])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_near_ties(cuda, scores, groups, group_score):
    """Biases that make up for the scores to within fp32's last bits: only wider arithmetic tells the keys apart."""
    print(f"route near ties {scores} {groups}", flush=True)
    gen = torch.Generator().manual_seed(8)
    row = torch.randn(64, generator=gen)
    score = torch.sigmoid(row.double()) if scores == "sigmoid" else torch.softmax(row.double(), 0)
    logits = row.expand(40, 64).clone()
    logits[20:] = torch.randn((20, 64), generator=gen)  # tokens that are told apart easily, in the same workgroup
    _check(logits, (1 - score).float(), 6, scores=scores, groups=groups, group_score=group_score, top_groups=max(1, groups // 2))


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("groups,group_score", [(1, "max"), (4, "max"), (4, "sum2")])
def test_masked_infinite_and_nan(cuda, scores, bias, groups, group_score):
    print(f"route masked {scores} {bias} {groups} {group_score}", flush=True)
    gen = torch.Generator().manual_seed(6)
    logits = torch.randn((12, 32), generator=gen)
    logits[0] = -math.inf
    logits[1, 3:] = -math.inf
    logits[2, :29] = -math.inf
    logits[3, 5] = math.inf
    logits[4, 30] = math.nan
    logits[5] = math.nan
    logits[6] = 3e38
    logits[7] = -3e38
    logits[8, 9], logits[8, 10] = 200.0, 300.0
    if scores == "softmax":
        logits[3, 5] = 60.0  # (an infinite one makes every score of a softmax NaN, as its token of NaN does)
    b = 0.1 * torch.randn(32, generator=gen) if bias else None
    kernel = tl.route_experts(12, 32, 4, scores=scores, bias=bias, groups=groups, top_groups=max(1, groups // 2), group_score=group_score)
    weights, ids, _, starts = kernel(logits.cuda(), *(() if b is None else (b.cuda(),)))
    want_ids, want = ref.route(logits, b, 4, scores, groups, max(1, groups // 2), group_score)
    assert torch.equal(ids.cpu(), want_ids) and int(starts[-1]) == 48
    assert torch.equal(torch.isnan(weights.cpu()), torch.isnan(want))
    seen = ~torch.isnan(want)
    assert ((weights.cpu().double() - want)[seen].abs() <= 1e-4).all()
    assert (weights[0] == 0).all() or scores == "sigmoid" and not bias and (weights[0] == 0).all() or bias


@pytest.mark.parametrize("tokens,top_k,experts,first", [
    (1, 1, 1, 0), (1, 8, 128, 0), (64, 1, 70, 2), (40, 8, 16, 16), (700, 6, 60, 3), (5000, 2, 8, 0), (4097, 3, 1024, 0), (9000, 8, 256, 100), (33, 32, 500, 0), (20000, 1, 3, 1),
])
def test_order(cuda, tokens, top_k, experts, first):
    """Ids of other experts, -1 and nonsense among them are in no expert's rows."""
    print(f"order {tokens}x{top_k} of {experts} from {first}", flush=True)
    gen = torch.Generator().manual_seed(tokens)
    ids = torch.randint(first - 2, first + experts + 2, (tokens, top_k), generator=gen, dtype=torch.int32)
    ids[torch.rand((tokens, top_k), generator=gen) < 0.05] = -1
    ids[0, 0] = -(2**31)
    ids[-1, -1] = 2**31 - 1
    flat = ids.flatten().long() - first
    inside = (flat >= 0) & (flat < experts)
    flat[~inside] = experts
    want = flat.argsort(stable=True).int()
    want[int(inside.sum()) :] = -1
    starts = torch.cat([torch.zeros(1), torch.bincount(flat, minlength=experts + 1)[:experts].cumsum(0)]).int()
    kernel = tl.experts_order(tokens, top_k, experts, first)
    order, got = kernel(ids.cuda())
    assert torch.equal(got.cpu(), starts) and torch.equal(order.cpu(), want)
    # all pairs one expert's, or nobody's
    for e in (first + experts - 1, first + experts):
        order, got = kernel(torch.full((tokens, top_k), e, dtype=torch.int32, device=cuda))
        n = tokens * top_k if e < first + experts else 0
        assert int(got[-1]) == n and int(got[-2]) == 0
        assert torch.equal(order.cpu(), torch.arange(tokens * top_k, dtype=torch.int32) if n else torch.full((tokens * top_k,), -1, dtype=torch.int32))


def test_many_tokens(cuda):
    """More chunks than one a workgroup, chunks of more than a wave's worth of tokens."""
    gen = torch.Generator().manual_seed(2)
    tokens, experts = 9001, 48
    logits = torch.randn((tokens, experts), generator=gen)
    weights, ids, order, starts = tl.route_experts(tokens, experts, 5, renormalize=False)(logits.cuda())
    want = logits.double().argsort(dim=1, descending=True, stable=True)[:, :5].int()
    assert torch.equal(ids.cpu(), want)
    soft = torch.softmax(logits.double(), dim=1).gather(1, want.long())
    assert ((weights.cpu().double() - soft).abs() <= 80 * 2.0**-24 * soft).all()
    flat = want.flatten().long()
    assert torch.equal(order.cpu(), flat.argsort(stable=True).int())
    assert torch.equal(starts.cpu()[1:], torch.bincount(flat, minlength=experts).cumsum(0).int())
