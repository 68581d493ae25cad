"""A router's logits where a row's offsets come near 2^31."""

import pytest
import torch

import tilelang_amd as tl

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,experts,dtype", [(1, 1, torch.float16), (2, 1, torch.bfloat16)])
def test_rows_of_nearly_2_to_the_31(cuda, tokens, experts, dtype):
    K = 2**31 - 32
    print(f"router {tokens} x {experts} x {K} {dtype}", flush=True)
    x, w = torch.zeros((tokens, K), dtype=dtype, device=cuda), torch.zeros((experts, K), dtype=dtype, device=cuda)
    at = torch.tensor([0, 1, 127, 128, 2047, 2048, 2**30 - 1, 2**30, K - 2048, K - 33, K - 32, K - 1], device=cuda)
    values = torch.arange(1, len(at) + 1, device=cuda)
    x[:, at], w[:, at] = values.to(dtype), (values % 3 + 1).to(dtype)
    x[-1, at[-1]] = 100
    got = tl.router_logits(tokens, experts, K, dtype)(x, w).cpu()
    want = (x[:, at].double() @ w[:, at].double().t()).cpu()
    assert torch.equal(got.double(), want)
