"""The experts' products against plain ones in 64 bits, over every way that rows can fall to experts."""

import math

import pytest
import torch

import block_reference as ref
import tilelang_amd as tl
from tilelang_amd import _lib

pytestmark = pytest.mark.gpu


def _ids(gen, tokens, experts, top_k, how):
    if how == "one":  # all tokens the same experts
        return torch.arange(top_k, dtype=torch.int32).expand(tokens, top_k).contiguous() + experts - top_k
    ids = torch.rand((tokens, experts), generator=gen)
    if how == "skewed":
        ids = ids - 0.9 * torch.linspace(0, 1, experts)
    ids = ids.argsort(dim=1, descending=True)[:, :top_k].int().contiguous()
    if how == "padded":  # places of the batch with no token, and ids that another GPU has
        ids[tokens // 2] = -1
        ids[torch.rand(ids.shape, generator=gen) < 0.2] = experts + 3
    if how == "twice":
        ids[:, -1] = ids[:, 0]
    return ids


def _same(got, want, slack, dtype, what):
    assert ref.agrees(got, want, slack, dtype), f"{what}: off by {float((got.double().cpu() - want).abs().max())}"


def _both(cuda, tokens, experts, top_k, hidden, inter, how="even", whole=False, activation="silu", residual=False, seed=0, **fmt):
    gen = torch.Generator().manual_seed(seed + tokens)
    ids = _ids(gen, tokens, experts, top_k, how)
    order, starts = ref.order(ids, experts)
    rows = int(starts[-1])
    sizes = dict(weight_format=fmt.get("weight_format", "uint4"), group_size=fmt.get("group_size"), with_zeros=fmt.get("with_zeros", False),
                 with_bias=fmt.get("with_bias", False))
    w = ref.Weights(gen, experts, 2 * inter, hidden, device=cuda, whole=whole, **sizes)
    x = (torch.randint(-2, 3, (tokens, hidden), generator=gen) if whole else torch.randn((tokens, hidden), generator=gen)).to(w.dtype)
    kernel = tl.experts_up(tokens, experts, top_k, inter, hidden, activation=activation, **sizes)
    on = [order.to(cuda), starts.to(cuda)]
    h = kernel(x.to(cuda), *w.on_device, *on)
    want, slack = ref.up(x, w, order, starts, top_k, inter, activation)
    assert h.shape == (tokens * top_k, inter)
    _same(h[:rows], want[:rows], slack[:rows], w.dtype, "up")

    d = ref.Weights(gen, experts, hidden, inter, device=cuda, whole=whole, **sizes)
    h = (torch.randint(-2, 3, (tokens * top_k, inter), generator=gen) if whole else torch.randn((tokens * top_k, inter), generator=gen)).to(d.dtype)
    h[rows:] = math.nan  # rows behind the last are not looked at
    weights = torch.randint(-4, 5, (tokens, top_k), generator=gen).float() if whole else torch.rand((tokens, top_k), generator=gen)
    r = torch.randn((tokens, hidden), generator=gen).to(d.dtype) if residual else None
    kernel = tl.experts_down(tokens, experts, top_k, hidden, inter, residual=residual, **sizes)
    y = kernel(h.to(cuda), *d.on_device, *on, ids.to(cuda), weights.to(cuda), *([r.to(cuda)] if residual else []))
    want, slack = ref.down(h, d, order, starts, weights, tokens, r)
    if whole and not residual:
        slack = slack * 0  # whole numbers below 2^24: every sum is exact
    _same(y, want, slack, d.dtype, "down")


FORMATS = [dict(), dict(group_size=64), dict(group_size=32, with_zeros=True), dict(with_zeros=True, with_bias=True), dict(weight_format="mxfp4"),
           dict(weight_format="mxfp4", with_bias=True)]


@pytest.mark.parametrize("fmt", FORMATS, ids=lambda f: "-".join(f"{k}={v}" for k, v in f.items()) or "uint4")
@pytest.mark.parametrize("tokens,experts,top_k,how", [
    (1, 1, 1, "even"), (1, 8, 2, "even"), (1, 60, 8, "even"), (2, 5, 5, "even"), (4, 128, 4, "even"), (16, 8, 1, "one"), (17, 3, 2, "one"), (33, 16, 4, "skewed"),
    (40, 7, 3, "padded"), (70, 4, 2, "skewed"), (150, 6, 2, "even"), (5, 9, 3, "twice"), (300, 2, 1, "skewed"),
])
def test_products(cuda, tokens, experts, top_k, how, fmt):
    print(f"experts {tokens} of {experts} top {top_k} {how} {fmt}", flush=True)
    _both(cuda, tokens, experts, top_k, 256, 128, how, residual=tokens % 2 == 0, activation="gelu" if experts == 5 else "silu", **fmt)


@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("fmt,hidden,inter", [
    (dict(), 128, 128), (dict(group_size=32), 384, 640), (dict(with_zeros=True), 1408, 256), (dict(group_size=64, with_bias=True), 640, 1152),
    (dict(weight_format="mxfp4"), 64, 64), (dict(weight_format="mxfp4", with_bias=True), 192, 320), (dict(weight_format="mxfp4"), 2880, 576),
])
@pytest.mark.parametrize("tokens,experts,top_k", [(1, 4, 2), (19, 5, 2), (130, 4, 2)])
def test_sizes(cuda, tokens, experts, top_k, fmt, hidden, inter, whole):
    print(f"experts {tokens} of {experts} top {top_k} {hidden} {inter} {fmt} whole={whole}", flush=True)
    if whole and hidden * inter > 384 * 640:
        hidden, inter = 384, 384  # (sums stay below 2^24, and fp16's largest)
    _both(cuda, tokens, experts, top_k, hidden, inter, whole=whole, **fmt)


@pytest.mark.parametrize("fmt", FORMATS, ids=lambda f: "-".join(f"{k}={v}" for k, v in f.items()) or "uint4")
@pytest.mark.parametrize("tokens,experts,top_k,how,hidden,inter", [
    (1100, 2, 1, "even", 128, 256), (1024, 1, 1, "one", 256, 384), (700, 3, 1, "one", 384, 128), (3500, 70, 1, "skewed", 128, 128), (900, 5, 3, "padded", 256, 128),
    (1400, 4, 2, "skewed", 640, 256), (100, 5, 2, "skewed", 256, 384), (3500, 70, 1, "padded", 128, 256), (2500, 70, 2, "skewed", 384, 128),
    (40, 2, 2, "one", 640, 128), (130, 300, 2, "even", 128, 128), (600, 300, 8, "even", 128, 128),
])
def test_many_rows(cuda, tokens, experts, top_k, how, hidden, inter, fmt):
    print(f"experts {tokens} of {experts} top {top_k} {how} {hidden} {inter} {fmt}", flush=True)
    _both(cuda, tokens, experts, top_k, hidden, inter, how, residual=tokens % 4 == 0, **fmt)


@pytest.mark.parametrize("fmt,inter", [
    (dict(), 4096), (dict(group_size=64, with_bias=True), 4224), (dict(group_size=32, with_zeros=True), 2176), (dict(with_zeros=True, with_bias=True), 8192),
    (dict(weight_format="mxfp4"), 4096), (dict(weight_format="mxfp4", with_bias=True), 4224),
], ids=str)
@pytest.mark.parametrize("tokens,experts,top_k,how,hidden", [(500, 2, 1, "even", 1152), (330, 3, 2, "skewed", 1024), (520, 3, 1, "padded", 1152), (300, 2, 2, "one", 1152)])
def test_slices_of_k(cuda, tokens, experts, top_k, how, hidden, fmt, inter):
    """Few experts and columns: "down" cuts K into slices, of units of 256 and what is left."""
    print(f"experts slices {tokens} of {experts} top {top_k} {how} {hidden} {inter} {fmt}", flush=True)
    mx = fmt.get("weight_format") == "mxfp4"
    room = _lib.load_library().dq_experts_down_workspace_bytes(tokens, experts, top_k, hidden, inter, fmt.get("group_size") or (32 if mx else 128), int(mx), experts)
    assert room in (2 * tokens * top_k * hidden * 4, 4 * tokens * top_k * hidden * 4)
    _both(cuda, tokens, experts, top_k, hidden, inter, how, residual=tokens % 40 == 0, **fmt)


@pytest.mark.parametrize("weight_format", ["uint4", "mxfp4"])
def test_nothing_to_do(cuda, weight_format):
    """No token has an expert here: h is left as it was, y is the residual."""
    gen = torch.Generator().manual_seed(3)
    tokens, experts, top_k, N, K = 6, 4, 2, 64, 128
    w = ref.Weights(gen, experts, N, K, weight_format, device=cuda)
    ids = torch.full((tokens, top_k), -1, dtype=torch.int32, device=cuda)
    order, starts = tl.experts_order(tokens, top_k, experts)(ids)
    assert (order == -1).all() and (starts == 0).all()
    r = torch.randn((tokens, N), generator=gen).to(w.dtype).to(cuda)
    h = torch.full((tokens * top_k, K), math.nan, dtype=w.dtype, device=cuda)
    y = tl.experts_down(tokens, experts, top_k, N, K, weight_format, residual=True)(h, *w.on_device, order, starts, ids, torch.ones((tokens, top_k), device=cuda), r)
    assert torch.equal(y, r)


@pytest.mark.parametrize("tokens", [1, 40])
def test_infinities_stay_in_their_rows(cuda, tokens):
    gen = torch.Generator().manual_seed(9)
    experts, top_k, N, K = 8, 2, 64, 128
    w = ref.Weights(gen, experts, 2 * N, K, device=cuda)
    ids = _ids(gen, tokens, experts, top_k, "even")
    order, starts = ref.order(ids, experts)
    x = torch.randn((tokens, K), generator=gen).half()
    x[tokens // 2, 5] = math.nan
    h = tl.experts_up(tokens, experts, top_k, N, K)(x.to(cuda), *w.on_device, order.to(cuda), starts.to(cuda)).cpu()
    bad = order // top_k == tokens // 2
    assert torch.isnan(h[bad]).all() and torch.isfinite(h[~bad]).all()


def _layer(cuda, tokens, experts, top_k, hidden, inter, weight_format="uint4"):
    """The kernel objects of a layer and their constant operands, and what one pass through them computes."""
    gen = torch.Generator().manual_seed(12)
    w_up = ref.Weights(gen, experts, 2 * inter, hidden, weight_format, device=cuda)
    w_down = ref.Weights(gen, experts, hidden, inter, weight_format, device=cuda)
    dtype = "bfloat16" if weight_format == "mxfp4" else "float16"
    norm, route = tl.rms_norm(tokens, hidden, dtype=dtype, residual=True), tl.route_experts(tokens, experts, top_k, dtype=dtype)
    up, down = (make(tokens, experts, top_k, *sizes, weight_format, **more) for make, sizes, more in
                ((tl.experts_up, (inter, hidden), {}), (tl.experts_down, (hidden, inter), {"residual": True})))
    gain = torch.ones(hidden, dtype=w_up.dtype, device=cuda)
    gate = torch.randn((experts, hidden), generator=gen).to(w_up.dtype).to(cuda) / 16

    def run(x, residual):
        y, total = norm(x, residual, gain)
        logits = (y[:, None].float() * gate.float()).sum(dim=2).to(w_up.dtype)
        weights, ids, order, starts = route(logits)
        h = up(y, *w_up.on_device, order, starts)
        return down(h, *w_down.on_device, order, starts, ids, weights, total)

    def make(seed):
        g = torch.Generator().manual_seed(seed)
        return [torch.randn((tokens, hidden), generator=g).to(w_up.dtype).to(cuda) for _ in range(2)]

    return run, make


@pytest.mark.parametrize("weight_format", ["uint4", "mxfp4"])
@pytest.mark.parametrize("tokens", [1, 24, 200])
def test_layer_in_a_graph(cuda, tokens, weight_format):
    """Captured once, replayed on other inputs, with the program's own work between; two graphs at once on streams of their own."""
    print(f"experts in a graph {tokens} {weight_format}", flush=True)
    run, make = _layer(cuda, tokens, 16, 4, 256, 128, weight_format)
    graphs = []
    for seed in (0, 1):
        held = make(seed)
        run(*held)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(*held)
        graphs.append((graph, held, out, torch.cuda.Stream()))
    for seed in range(10, 14):
        wants = []
        for n, (graph, held, out, stream) in enumerate(graphs):
            fresh = make(seed + 100 * n)
            wants.append(run(*fresh).clone())
            for h, f in zip(held, fresh):
                h.copy_(f)
        torch.cuda.synchronize()
        for graph, _, _, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, out, _), want in zip(graphs, wants):
            assert torch.equal(out, want)


@pytest.mark.parametrize("tokens", [3, 90])
def test_layer_on_two_streams(cuda, tokens):
    """The same kernel objects on two streams at once: neither's scratch is the other's."""
    run, make = _layer(cuda, tokens, 12, 3, 384, 256)
    inputs = [make(s) for s in range(6)]
    wants = [run(*i).clone() for i in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for n, i in enumerate(inputs):
        with torch.cuda.stream(streams[n % 2]):
            outs.append(run(*i))
    torch.cuda.synchronize()
    for out, want in zip(outs, wants):
        assert torch.equal(out, want)
