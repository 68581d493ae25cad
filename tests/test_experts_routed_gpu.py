"""The experts' products of a GPU that has some of the experts: `routed` says of how many the ids are, and which kernel runs goes by it.
Whatever falls to these experts, few rows of many or all of them, the results are within the same bounds."""

import math

import pytest
import torch

import block_reference as ref
import tilelang_amd as tl
from tilelang_amd import _lib

pytestmark = pytest.mark.gpu


def _ids(gen, tokens, experts, top_k, routed, first, how):
    if how == "one":  # all pairs are the last experts' here
        return (torch.arange(top_k, dtype=torch.int32).expand(tokens, top_k) + first + experts - top_k).contiguous()
    wish = torch.rand((tokens, routed), generator=gen)
    if how == "local":  # all pairs are these experts', some of them more than others
        wish[:, first : first + experts] += 1 + torch.linspace(0, 1, experts)
    return wish.argsort(dim=1, descending=True)[:, :top_k].int().contiguous()


def _both(cuda, tokens, experts, top_k, hidden, inter, routed, first, how, residual=False, **fmt):
    gen = torch.Generator().manual_seed(tokens + routed)
    ids = _ids(gen, tokens, experts, top_k, routed, first, how)
    order, starts = ref.order(ids, experts, first)
    rows = int(starts[-1])
    assert how == "spread" or rows == tokens * top_k
    got = tl.experts_order(tokens, top_k, experts, first)(ids.to(cuda))
    assert torch.equal(got[0].cpu(), order) and torch.equal(got[1].cpu(), starts)
    w = ref.Weights(gen, experts, 2 * inter, hidden, device=cuda, **fmt)
    x = torch.randn((tokens, hidden), generator=gen).to(w.dtype)
    h = tl.experts_up(tokens, experts, top_k, inter, hidden, routed=routed, **fmt)(x.to(cuda), *w.on_device, *got)
    want, slack = ref.up(x, w, order, starts, top_k, inter, "silu")
    assert ref.agrees(h[:rows], want[:rows], slack[:rows], w.dtype)

    d = ref.Weights(gen, experts, hidden, inter, device=cuda, **fmt)
    h = torch.randn((tokens * top_k, inter), generator=gen).to(d.dtype)
    h[rows:] = math.nan
    weights = torch.rand((tokens, top_k), generator=gen)
    r = torch.randn((tokens, hidden), generator=gen).to(d.dtype) if residual else None
    kernel = tl.experts_down(tokens, experts, top_k, hidden, inter, residual=residual, first=first, routed=routed, **fmt)
    y = kernel(h.to(cuda), *d.on_device, *got, ids.to(cuda), weights.to(cuda), *([r.to(cuda)] if residual else []))
    assert ref.agrees(y, *ref.down(h, d, order, starts, weights, tokens, r), d.dtype)


FORMATS = [dict(), dict(group_size=32, with_zeros=True, with_bias=True), dict(weight_format="mxfp4", with_bias=True)]


@pytest.mark.parametrize("fmt", FORMATS, ids=["uint4", "zeros", "mxfp4"])
@pytest.mark.parametrize("how", ["spread", "local", "one"])
@pytest.mark.parametrize("tokens,experts,top_k,times,hidden,inter", [
    (1, 4, 2, 8, 256, 128), (3, 2, 2, 32, 256, 128), (40, 8, 4, 8, 256, 384), (150, 3, 2, 64, 384, 256), (900, 4, 2, 8, 256, 128), (1500, 2, 1, 64, 128, 256),
])
def test_rows_beyond_what_is_expected(cuda, tokens, experts, top_k, times, hidden, inter, how, fmt):
    print(f"routed {tokens} of {experts}x{times} top {top_k} {hidden} {inter} {how} {fmt}", flush=True)
    _both(cuda, tokens, experts, top_k, hidden, inter, experts * times, 5 if times > 4 else 0, how, residual=tokens % 20 == 0, **fmt)


@pytest.mark.parametrize("weight_format", ["uint4", "mxfp4"])
@pytest.mark.parametrize("how", ["spread", "local"])
@pytest.mark.parametrize("times", [1, 8, 64])
@pytest.mark.parametrize("tokens,experts,top_k", [(520, 2, 2), (1100, 3, 1)])
def test_slices_of_k(cuda, tokens, experts, top_k, times, how, weight_format):
    """Few columns of a long K: in slices where rows are expected, in none where few of the pairs are."""
    print(f"routed slices {tokens} of {experts}x{times} top {top_k} {how} {weight_format}", flush=True)
    mx, hidden, inter = weight_format == "mxfp4", 1152, 4096
    room = _lib.load_library().dq_experts_down_workspace_bytes(tokens, experts, top_k, hidden, inter, 32 if mx else 128, int(mx), experts * times)
    one = tokens * top_k * hidden * 4
    assert room in ((2 * one, 4 * one) if times == 1 else (one, 2 * one, 4 * one))
    _both(cuda, tokens, experts, top_k, hidden, inter, experts * times, 0, how, weight_format=weight_format)
