"""RMSNorm and W4Experts in the calls of a server: a rank's part of the experts in a graph, parts of a prompt, batches of no tokens,
kernels that are made anew between replays."""

import pytest
import torch

import tilelang_amd as tl
from test_experts_layer import _filled
from tilelang_amd import experts as layers

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_a_part_of_the_experts_in_a_graph(cuda, tokens):
    """Captured once, replayed on other inputs, eager calls of the same layer and of other sizes between."""
    gen = torch.Generator().manual_seed(tokens)
    whole = _filled(gen, cuda, experts=10, top_k=3)
    part = tl.W4Experts(256, 128, 10, 3, first=4, held=5).to(cuda)
    part.load_state_dict({k: v if k == "router" else v[4:9] for k, v in whole.state_dict().items()})
    norm = tl.RMSNorm(256).to(cuda)

    def run(x, r):
        y, total = norm(x, r)
        return part(y, total)

    held = [torch.randn((tokens, 256), generator=gen).half().to(cuda) for _ in range(2)]
    run(*held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*held)
    for seed in range(4):
        fresh = [torch.randn((tokens, 256), generator=gen).half().to(cuda) for _ in range(2)]
        want = run(*fresh).clone()
        for n in range(1 + 70 * (seed == 1)):  # (more sizes than kernel objects are kept of)
            run(*(t[: 1 + n % tokens] for t in fresh))
        for h, f in zip(held, fresh):
            h.copy_(f)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_parts_of_a_prompt_by_bytes(cuda, monkeypatch):
    """Parts that bytes say are the parts, to the bit."""
    gen = torch.Generator().manual_seed(3)
    layer = _filled(gen, cuda)
    x, r = (torch.randn((50, 256), generator=gen).half().to(cuda) for _ in range(2))
    monkeypatch.setattr(layers, "PART_BYTES", 12 * 2 * (2 * 128 + 4 * 256))
    assert torch.equal(layer(x, r), torch.cat([layer(x[p : p + 12], r[p : p + 12]) for p in range(0, 50, 12)]))
    logits = torch.randn((50, 6), generator=gen).to(cuda)
    assert torch.equal(layer(x, logits=logits), torch.cat([layer(x[p : p + 12], logits=logits[p : p + 12]) for p in range(0, 50, 12)]))


def test_no_tokens_on_the_gpu(cuda):
    norm, layer = tl.RMSNorm(256, int8=True).to(cuda), tl.W4Experts(256, 128, 4, 2).to(cuda)
    x = torch.empty((0, 256), dtype=torch.float16, device=cuda)
    codes, scale, total = norm(x, x)
    assert codes.device == scale.device == total.device == layer(x, x).device == cuda and len(layer(x)) == len(scale) == 0


def test_rows_far_apart(cuda):
    x = torch.empty(2**31 + 64, dtype=torch.float16, device=cuda).as_strided((2, 64), (2**31, 1))
    x.copy_(torch.randn((2, 64), generator=torch.Generator().manual_seed(1)))
    norm = tl.RMSNorm(64).to(cuda)
    assert torch.equal(norm(x), norm(x.contiguous()))
