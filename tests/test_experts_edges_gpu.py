"""The experts' products and the order at the edges of what a call takes: up to eight pairs in every form, many choices a token, the
most pairs, scales of every size."""

import math

import pytest
import torch

import block_reference as ref
import tilelang_amd as tl

pytestmark = pytest.mark.gpu


def _both(cuda, ids, experts, hidden, inter, residual, first=0, **fmt):
    gen = torch.Generator().manual_seed(ids.numel())
    tokens, top_k = ids.shape
    order, starts = ref.order(ids, experts, first)
    rows = int(starts[-1])
    got = tl.experts_order(tokens, top_k, experts, first)(ids.to(cuda))
    assert torch.equal(got[0].cpu(), order) and torch.equal(got[1].cpu(), starts)
    w = ref.Weights(gen, experts, 2 * inter, hidden, device=cuda, **fmt)
    x = torch.randn((tokens, hidden), generator=gen).to(w.dtype)
    h = tl.experts_up(tokens, experts, top_k, inter, hidden, **fmt)(x.to(cuda), *w.on_device, *got)
    want, slack = ref.up(x, w, order, starts, top_k, inter, "silu")
    assert ref.agrees(h[:rows], want[:rows], slack[:rows], w.dtype)

    d = ref.Weights(gen, experts, hidden, inter, device=cuda, **fmt)
    h = torch.randn((tokens * top_k, inter), generator=gen).to(d.dtype)
    h[rows:] = math.nan
    weights = torch.rand((tokens, top_k), generator=gen)
    inside = (ids >= first) & (ids < first + experts)
    given = weights.masked_fill(~inside, math.nan)  # (of choices that are not here)
    r = torch.randn((tokens, hidden), generator=gen).to(d.dtype) if residual else None
    kernel = tl.experts_down(tokens, experts, top_k, hidden, inter, residual=residual, first=first, **fmt)
    y = kernel(h.to(cuda), *d.on_device, *got, ids.to(cuda), given.to(cuda), *([r.to(cuda)] if residual else []))
    assert ref.agrees(y, *ref.down(h, d, order, starts, weights, tokens, r), d.dtype)


FORMATS = [dict(), dict(group_size=32, with_zeros=True, with_bias=True), dict(weight_format="mxfp4", with_bias=True)]


@pytest.mark.parametrize("fmt", FORMATS, ids=["uint4", "zeros", "mxfp4"])
@pytest.mark.parametrize("how", ["spread", "twice", "foreign", "one"])
@pytest.mark.parametrize("tokens,top_k", [(1, 3), (1, 8), (2, 4), (4, 2), (8, 1), (7, 1), (3, 2)])
def test_up_to_eight_pairs(cuda, tokens, top_k, how, fmt):
    print(f"experts {tokens}x{top_k} {how} {fmt}", flush=True)
    gen = torch.Generator().manual_seed(tokens * top_k)
    experts, first = 20, 3
    ids = torch.rand((tokens, experts), generator=gen).argsort(dim=1)[:, :top_k].int() + first
    if how == "twice":
        ids[:, -1] = ids[:, 0]
    if how == "foreign":  # the first and the last choice are not here, and one is nobody's
        ids[0, 0], ids[-1, -1] = first - 1, first + experts
        ids[tokens // 2, top_k // 2] = -1
    if how == "one":
        ids[:] = first + experts - 1
    _both(cuda, ids.contiguous(), experts, 256, 384, tokens % 2 == 0, first, **fmt)


@pytest.mark.parametrize("fmt", FORMATS, ids=["uint4", "zeros", "mxfp4"])
@pytest.mark.parametrize("tokens,experts,top_k,inter", [(1, 40, 9, 256), (3, 40, 32, 128), (60, 48, 17, 256), (300, 32, 32, 128), (130, 33, 32, 4096)])
def test_many_choices(cuda, tokens, experts, top_k, inter, fmt):
    print(f"experts {tokens} of {experts} top {top_k} {inter} {fmt}", flush=True)
    gen = torch.Generator().manual_seed(experts)
    ids = torch.rand((tokens, experts), generator=gen).argsort(dim=1)[:, :top_k].int().contiguous()
    _both(cuda, ids, experts, 128, inter, tokens % 2 == 0, **fmt)


@pytest.mark.parametrize("tokens,top_k,experts", [(2**23, 1, 7), (2**18, 32, 1024)])
def test_order_of_the_most_pairs(cuda, tokens, top_k, experts):
    """Chunks of more than 2^15 pairs, counted in 16 bits, all of them one expert's too."""
    print(f"order {tokens}x{top_k} of {experts}", flush=True)
    ids = torch.randint(-1, experts, (tokens, top_k), generator=torch.Generator(device=cuda).manual_seed(1), device=cuda, dtype=torch.int32)
    for given in (ids, torch.full_like(ids, experts - 1)):
        flat = given.flatten().long()
        flat = torch.where(flat < 0, experts, flat)
        count = torch.bincount(flat, minlength=experts + 1)[:experts]
        order, starts = tl.experts_order(tokens, top_k, experts)(given)
        assert torch.equal(starts[1:].long(), count.cumsum(0)) and int(starts[0]) == 0
        want = flat.argsort(stable=True).int()
        want[int(starts[-1]) :] = -1
        assert torch.equal(order, want)


def test_route_of_the_most_pairs(cuda):
    tokens, experts, top_k = 2**20, 16, 8
    logits = torch.randn((tokens, experts), generator=torch.Generator(device=cuda).manual_seed(4), device=cuda)
    weights, ids, order, starts = tl.route_experts(tokens, experts, top_k)(logits)
    best = logits.double().argsort(dim=1, descending=True, stable=True)[:, :top_k]
    assert torch.equal(ids, best.int())
    assert torch.equal(order, best.flatten().argsort(stable=True).int())
    assert torch.equal(starts[1:].long(), torch.bincount(best.flatten(), minlength=experts).cumsum(0))


@pytest.mark.parametrize("tokens", [1, 20, 2000])
@pytest.mark.parametrize("byte", [0, 1, 127, 254, 255])
def test_scales_of_every_size(cuda, tokens, byte):
    """An MXFP4 scale is 2^(byte - 127), 2^127 at most; powers of two multiply without rounding.  (2^130 is an infinity in bf16.)"""
    N, K = 32, 128
    ids = torch.zeros((tokens, 1), dtype=torch.int32, device=cuda)
    order, starts = tl.experts_order(tokens, 1, 1)(ids)
    for x in (2.0 ** (127 - byte + 3), 2.0 ** round(0.75 * (127 - byte))):
        for code, value in ((1, 0.5), (2, 1.0), (3, 1.5)):
            packed = torch.full((1, N, K // 2), code | code << 4, dtype=torch.uint8, device=cuda)
            scale = torch.full((1, N, K // 32), byte, dtype=torch.uint8, device=cuda)
            h = torch.zeros((tokens, K), dtype=torch.bfloat16, device=cuda)
            h[:, 70] = x
            y = tl.experts_down(tokens, 1, 1, N, K, "mxfp4")(h, packed, scale, order, starts, ids, torch.ones((tokens, 1), device=cuda))
            assert (y.double() == value * 2.0 ** (min(byte, 254) - 127) * float(h[0, 70])).all()


@pytest.mark.parametrize("weight_format", ["uint4", "mxfp4"])
@pytest.mark.parametrize("tokens", [1, 9, 40, 700])
@pytest.mark.parametrize("N", [32, 96, 160, 288, 416])
def test_columns_in_blocks_of_32(cuda, N, tokens, weight_format):
    """N that is an odd number of blocks of 32: a tile's last blocks are not there."""
    print(f"experts {tokens} N={N} {weight_format}", flush=True)
    gen = torch.Generator().manual_seed(N + tokens)
    experts, top_k, K = 5, 2, 384
    ids = torch.rand((tokens, experts), generator=gen).argsort(dim=1)[:, :top_k].int().contiguous()
    order, starts = ref.order(ids, experts)
    got = order.to(cuda), starts.to(cuda)
    w = ref.Weights(gen, experts, 2 * N, K, weight_format, with_bias=True, device=cuda)
    x = torch.randn((tokens, K), generator=gen).to(w.dtype)
    h = tl.experts_up(tokens, experts, top_k, N, K, weight_format, activation="gelu", with_bias=True)(x.to(cuda), *w.on_device, *got)
    assert ref.agrees(h, *ref.up(x, w, order, starts, top_k, N, "gelu"), w.dtype)
    d = ref.Weights(gen, experts, N, K, weight_format, with_bias=True, device=cuda)
    h = torch.randn((tokens * top_k, K), generator=gen).to(d.dtype)
    weights, r = torch.rand((tokens, top_k), generator=gen), torch.randn((tokens, N), generator=gen).to(d.dtype)
    y = tl.experts_down(tokens, experts, top_k, N, K, weight_format, with_bias=True, residual=True)(h.to(cuda), *d.on_device, *got, ids.to(cuda), weights.to(cuda), r.to(cuda))
    assert ref.agrees(y, *ref.down(h, d, order, starts, weights, tokens, r), d.dtype)
