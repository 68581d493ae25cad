"""RMSNorm, W4Experts and BitLinear on int8 rows: batches of no tokens, and what a call is checked for before it goes to a kernel."""

import pytest
import torch

import tilelang_amd as tl


@pytest.mark.parametrize("lead", [(0,), (0, 5), (3, 0)])
@pytest.mark.parametrize("int8", [False, True])
def test_norm_of_no_rows(lead, int8):
    """A step that has no token here: results of no rows, no launch."""
    norm = tl.RMSNorm(64, dtype="bfloat16", int8=int8)
    x = torch.zeros((*lead, 64))
    first = norm(x)
    both = norm(x, x)
    if int8:
        codes, scale = first
        assert codes.shape == x.shape and codes.dtype == torch.int8 and scale.shape == lead and scale.dtype == torch.float32
        assert [t.dtype for t in both] == [torch.int8, torch.float32, torch.bfloat16] and both[1].shape == lead
        linear = tl.BitLinear(128, 96)
        out = linear(codes.new_zeros((*lead, 128)), scale)
        assert out.shape == (*lead, 96) and out.dtype == torch.float16
    else:
        assert first.shape == x.shape and first.dtype == torch.bfloat16 and [t.dtype for t in both] == [torch.bfloat16] * 2
    assert both[-1].shape == both[0].shape == x.shape


@pytest.mark.parametrize("lead", [(0,), (0, 5), (3, 0)])
@pytest.mark.parametrize("weight_format", ["uint4", "mxfp4"])
def test_experts_of_no_tokens(lead, weight_format):
    layer = tl.W4Experts(256, 128, 4, 2, weight_format)
    x = torch.zeros((*lead, 256))
    for out in (layer(x), layer(x, x), layer(x, logits=torch.zeros((*lead, 4)))):
        assert out.shape == x.shape and out.dtype == layer.router.dtype
