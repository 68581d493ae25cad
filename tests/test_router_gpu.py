"""A router's logits against the product in 64 bits."""

import math

import pytest
import torch

import tilelang_amd as tl

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,experts,K", [
    (1, 1, 32), (1, 128, 4096), (2, 3, 64), (3, 60, 2880), (16, 16, 2048), (17, 33, 96), (40, 1024, 160), (64, 128, 4096), (257, 8, 2144), (300, 100, 224),
    (1000, 257, 128), (3000, 128, 96), (5000, 260, 32),
])
def test_logits(cuda, tokens, experts, K, dtype, with_bias, whole):
    print(f"router {tokens} x {experts} x {K} {dtype} {with_bias} {whole}", flush=True)
    gen = torch.Generator().manual_seed(tokens + experts)
    make = (lambda *s: torch.randint(-3, 4, s, generator=gen)) if whole else (lambda *s: torch.randn(s, generator=gen))
    x, w, b = make(tokens, K).to(dtype), make(experts, K).to(dtype), make(experts).to(dtype)
    held = [x.to(cuda), w.to(cuda), *([b.to(cuda)] if with_bias else [])]
    got = tl.router_logits(tokens, experts, K, dtype, with_bias)(*held)
    assert got.shape == (tokens, experts) and got.dtype == torch.float32
    want, size = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
    if with_bias:
        want, size = want + b.double(), size + b.double().abs()
    # whole numbers below 2^24 are exact; else K products added one by one, whatever the order, and the waves' sums and the bias
    off = 0.0 if whole else (K + 18) * 2.0**-24 * size
    assert ((got.cpu().double() - want).abs() <= off).all()


@pytest.mark.parametrize("tokens,experts", [(5, 7), (40, 20), (700, 130)])
def test_nan_stays_where_it_is(cuda, tokens, experts):
    gen = torch.Generator().manual_seed(1)
    x, w = torch.randn((tokens, 256), generator=gen).half(), torch.randn((experts, 256), generator=gen).half()
    x[tokens - 1, 3], w[2, 255] = math.nan, math.inf
    got = tl.router_logits(tokens, experts, 256)(x.to(cuda), w.to(cuda)).cpu()
    clean = torch.ones((tokens, experts), dtype=torch.bool)
    clean[tokens - 1], clean[:, 2] = False, False
    assert torch.isfinite(got[clean]).all() and not torch.isfinite(got[~clean]).any() and torch.isnan(got[tokens - 1]).all()
