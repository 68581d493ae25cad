"""Norm and experts' products where offsets pass 32 bits: samples of the rows against the formulas in 64 bits."""

import pytest
import torch

import block_reference as ref
import tilelang_amd as tl

pytestmark = pytest.mark.gpu


class _Held:
    """Random weights on the device, of which an expert's values are looked at on the host."""

    def __init__(self, cuda, experts, rows, K, mx):
        gen = torch.Generator(device=cuda).manual_seed(experts)
        self.mx, self.dtype = mx, torch.bfloat16 if mx else torch.float16
        self.packed = torch.randint(0, 256, (experts, rows, K // 2), generator=gen, device=cuda, dtype=torch.uint8)
        if mx:
            self.scale = torch.randint(119, 124, (experts, rows, K // 32), generator=gen, device=cuda, dtype=torch.uint8)
        else:
            self.packed = self.packed.view(torch.int8)
            self.scale = (torch.rand((experts, rows, K // 128), generator=gen, device=cuda) / 16).half()

    def of(self, expert):
        packed, scale = self.packed[expert].cpu().view(torch.uint8), self.scale[expert].cpu()
        codes = torch.stack((packed & 15, packed >> 4), dim=-1).flatten(-2)
        w = ref.Weights.__new__(ref.Weights)
        w.bias = None
        if self.mx:
            w.value = ref.E2M1[codes.long()] * 2.0 ** (scale.double() - 127).repeat_interleave(32, dim=1)
        else:
            w.value = ((codes.double() - 8) * scale.double().repeat_interleave(128, dim=1)).half().double()
        w.value = w.value[None]
        return w


@pytest.mark.parametrize("tokens", [2, 4500])
@pytest.mark.parametrize("mx", [False, True])
def test_weights_beyond_4_gib(cuda, tokens, mx):
    """Few rows and many of the last of 300 experts; the first has the others."""
    print(f"weights beyond 4 GiB {tokens} {mx}", flush=True)
    experts, N, K = 300, 4096, 4096
    fmt = "mxfp4" if mx else "uint4"
    gen = torch.Generator().manual_seed(tokens)
    ids = torch.zeros((tokens, 1), dtype=torch.int32)
    ids[tokens // 2 :] = experts - 1
    order, starts = tl.experts_order(tokens, 1, experts)(ids.to(cuda))
    w = _Held(cuda, experts, 2 * N, K, mx)
    assert w.packed.numel() > 2**32
    x = torch.randn((tokens, K), generator=gen).to(w.dtype)
    h = tl.experts_up(tokens, experts, 1, N, K, fmt)(x.to(cuda), w.packed, w.scale, order, starts)
    rows = torch.tensor([tokens // 2, tokens - 1])  # (one choice a token, in the order of their ids: row p is token p)
    two = torch.tensor([0, 2], dtype=torch.int32)
    want, slack = ref.up(x[rows], w.of(experts - 1), torch.arange(2), two, 1, N, "silu")
    assert ref.agrees(h[rows], want, slack, w.dtype)
    del w
    w = _Held(cuda, 2 * experts, N, K, mx)
    order, starts = tl.experts_order(tokens, 1, 2 * experts)((ids + experts).to(cuda))
    weights = torch.ones((tokens, 1))
    y = tl.experts_down(tokens, 2 * experts, 1, N, K, fmt)(h, w.packed, w.scale, order, starts, (ids + experts).to(cuda), weights.to(cuda))
    want, slack = ref.down(h[rows], w.of(2 * experts - 1), torch.arange(2), two, weights[:2], 2, None)
    assert ref.agrees(y[rows], want, slack, w.dtype)


@pytest.mark.parametrize("mx", [False, True])
def test_rows_beyond_4_gib(cuda, mx):
    """More than 2^32 bytes of h, of the pairs' products and of the result."""
    print(f"rows beyond 4 GiB {mx}", flush=True)
    tokens, experts, top_k, wide, narrow = 65536, 8, 3, 16384, 128
    fmt = "mxfp4" if mx else "uint4"
    gen = torch.Generator().manual_seed(1)
    ids = torch.rand((tokens, experts), generator=gen).argsort(dim=1)[:, :top_k].int().contiguous()
    order, starts = tl.experts_order(tokens, top_k, experts)(ids.to(cuda))
    on = (order, starts)
    order, starts = order.cpu(), starts.cpu()
    w = _Held(cuda, experts, 2 * wide, narrow, mx)
    x = torch.randn((tokens, narrow), generator=gen).to(w.dtype)
    h = tl.experts_up(tokens, experts, top_k, wide, narrow, fmt)(x.to(cuda), w.packed, w.scale, *on)
    assert h.numel() * 2 > 2**32
    rows = torch.tensor([int(starts[-2]), len(order) - 1])  # of the last expert
    two = torch.tensor([0, 2], dtype=torch.int32)
    want, slack = ref.up(x[order[rows].long() // top_k], w.of(experts - 1), torch.tensor([0, 2]), two, 2, wide, "silu")
    assert ref.agrees(h[rows], want, slack, w.dtype)

    # the way back from narrow rows to wide ones; and from the wide ones
    weights = torch.rand((tokens, top_k), generator=gen)
    for n, k, given in ((wide, narrow, torch.randn((tokens * top_k, narrow), generator=gen).to(w.dtype).to(cuda)), (narrow, wide, h)):
        d = _Held(cuda, experts, n, k, mx)
        y = tl.experts_down(tokens, experts, top_k, n, k, fmt)(given, d.packed, d.scale, *on, ids.to(cuda), weights.to(cuda))
        place = torch.empty(len(order), dtype=torch.int64)
        place[order.long()] = torch.arange(len(order))
        for t in (0, tokens - 1):
            want, slack = torch.zeros((1, n), dtype=torch.float64), torch.zeros((1, n), dtype=torch.float64)
            for j in range(top_k):
                v, off = ref.down(given[place[t * top_k + j]][None], d.of(int(ids[t, j])), torch.tensor([0]), torch.tensor([0, 1]), weights[t : t + 1, j : j + 1], 1, None)
                want, slack = want + v, slack + off + 2.0**-23 * v.abs()
            assert ref.agrees(y[t : t + 1], want, slack, w.dtype)
        del y, d


def test_norm_beyond_2_to_the_32_elements(cuda):
    rows, dim = 140000, 32768
    x = torch.empty((rows, dim), dtype=torch.float16, device=cuda).uniform_(-1, 1, generator=torch.Generator(device=cuda).manual_seed(2))
    weight = torch.rand(dim, generator=torch.Generator().manual_seed(3)).half()
    y = tl.rms_norm(rows, dim)(x, weight.to(cuda))
    at = torch.tensor([0, rows // 2, rows - 1])
    want, _, slack, _ = ref.norm(x[at].cpu(), None, weight, 1e-6)
    assert ref.agrees(y[at], want, slack, torch.float16)
