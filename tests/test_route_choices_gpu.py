"""Who is chosen where 32 bits cannot tell: groups whose biases all but cancel, more experts than a wave has in registers; and masks."""

import math

import pytest
import torch

import block_reference as ref
import tilelang_amd as tl
from test_route_gpu import _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("size", [3.0, 100.0, 1e5])
@pytest.mark.parametrize("experts,groups", [(8, 4), (64, 32), (320, 4)])
def test_groups_of_opposite_biases(cuda, experts, groups, size, scores):
    """A group's two best are large biases of either sign: their roundings are far beyond the sum's."""
    print(f"route opposite biases {experts}/{groups} {size} {scores}", flush=True)
    gen = torch.Generator().manual_seed(experts)
    per = experts // groups
    bias = torch.full((groups, per), -4 * size)
    bias[:, per - 1] = size * (1 + torch.rand(groups, generator=gen))
    bias[:, 0] = -bias[:, per - 1]
    tokens = 4000 if experts < 320 else 300
    _check(torch.randn((tokens, experts), generator=gen), bias.flatten(), 2, scores=scores, groups=groups, top_groups=groups // 2, group_score="sum2")


def test_groups_told_apart_by_64_bits(cuda):
    """fp32's sums are 1.4968338 and 1.4968414, the exact ones 1.49684026 and 1.49684014."""
    logits = torch.tensor([[0.923241138458252, 1.2723116874694824, 0.923241138458252, 1.2723109722137451]])
    ids, _ = _check(logits, torch.tensor([96.3, -96.3, 70.1, -70.1]), 2, scores="sigmoid", groups=2, top_groups=1, group_score="sum2")
    assert ids.tolist() == [[0, 1]]


MORE = [(257, 1, 1, "max"), (320, 8, 3, "sum2"), (512, 64, 5, "max"), (512, 1, 1, "max"), (1024, 4, 2, "sum2"), (1024, 1, 1, "max")]


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("experts,groups,top_groups,group_score", MORE)
def test_ties_of_many_experts(cuda, experts, groups, top_groups, group_score, dtype, scores):
    """Equal keys everywhere, which 64 bits have to look at: the lowest index."""
    print(f"route ties {experts} {groups} {group_score} {dtype} {scores}", flush=True)
    gen = torch.Generator().manual_seed(experts)
    logits = torch.randint(-2, 3, (40, experts), generator=gen).float()
    logits[0] = 0
    logits[1, : experts // 2] = -1
    for bias in (torch.zeros(experts), torch.full((experts,), -3.0), None):
        ids, _ = _check(logits, bias, 32, dtype, scores=scores, groups=groups, top_groups=top_groups, group_score=group_score)
        assert ids[0].tolist() == list(range(32))


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,top_groups,group_score", MORE)
def test_near_ties_of_many_experts(cuda, experts, groups, top_groups, group_score, scores):
    """Biases that make up for the scores to within fp32's last bits."""
    print(f"route near ties {experts} {groups} {group_score} {scores}", flush=True)
    gen = torch.Generator().manual_seed(experts + 1)
    row = torch.randn(experts, generator=gen)
    score = torch.sigmoid(row.double()) if scores == "sigmoid" else torch.softmax(row.double(), 0)
    logits = row.expand(36, experts).clone()
    logits[18:] = torch.randn((18, experts), generator=gen)
    _check(logits, (1 - score).float(), 10, scores=scores, groups=groups, top_groups=top_groups, group_score=group_score)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts", [4, 300])
def test_masks(cuda, experts, scores):
    """Without a bias a logit of -inf is chosen last.  With one its key is its bias, score 0; a bias of -inf is chosen last."""
    inf = math.inf
    logits = torch.full((3, experts), -inf)
    logits[0, 1:4] = torch.tensor([-2.0, -3.0, 0.0])
    logits[1, 2] = 5.0
    route = lambda bias: tl.route_experts(3, experts, 2, scores=scores, bias=bias is not None)(logits.cuda(), *(() if bias is None else (bias.cuda(),)))
    share = (torch.sigmoid if scores == "sigmoid" else lambda v: torch.exp(v))(torch.tensor([0.0, -2.0], dtype=torch.float64))
    share = (share / share.sum()).tolist()

    weights, ids, _, _ = route(None)
    assert ids.tolist() == [[3, 1], [2, 0], [0, 1]]
    assert torch.allclose(weights.cpu().double(), torch.tensor([share, [1, 0], [0, 0]], dtype=torch.float64), rtol=2e-6, atol=0)

    # scores are at most 1: what is masked with a bias of 2 goes first, with a weight of 0
    bias = torch.zeros(experts)
    bias[0] = 2.0
    weights, ids, _, _ = route(bias)
    assert ids.tolist() == [[0, 3], [0, 2], [0, 1]]
    assert torch.equal(weights.cpu(), torch.tensor([[0.0, 1.0], [0.0, 1.0], [0.0, 0.0]]))

    bias = torch.full((experts,), -inf)
    bias[1:3] = 0.0
    weights, ids, _, _ = route(bias)
    assert ids.tolist() == [[1, 2], [2, 1], [1, 2]]
    assert (weights[0] > 0).all() and torch.equal(weights[1:].cpu(), torch.tensor([[1.0, 0.0], [0.0, 0.0]]))


def test_masked_expert_by_its_bias(cuda):
    """Logistic scores 0, .119, .047, .5: keys .5, .02, -.05, .5."""
    logits, bias = torch.tensor([[-math.inf, -2.0, -3.0, 0.0]]), torch.tensor([0.5, -0.1, -0.1, 0.0])
    ids, weights = _check(logits, bias, 2, scores="sigmoid")
    assert ids.tolist() == [[0, 3]] and weights.tolist() == [[0.0, 1.0]]
    assert torch.equal(ids, ref.route(logits, bias, 2, "sigmoid")[0])
