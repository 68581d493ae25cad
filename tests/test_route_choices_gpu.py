"""Who is chosen where 32 bits cannot tell: groups whose biases all but cancel, more experts than a wave has in registers."""

import pytest
import torch

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
