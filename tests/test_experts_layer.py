"""RMSNorm and W4Experts: what they refuse and how they hold weights, on the CPU; on the GPU their results against the formulas on
what the layer holds, next to BitLinear, and whole decoder blocks."""

import pytest
import torch

import block_reference as ref
import tilelang_amd as tl
from tilelang_amd import experts as layers
from tilelang_amd.w4linear import dequantize_w4_reference


@pytest.mark.parametrize("args,match", [(dict(dim=12), "multiple of 8"), (dict(dim=0), "multiple of 8"), (dict(dim=64, eps=0.0), "eps"), (dict(dim=64, dtype="float32"), "float16")])
def test_norm_refuses(args, match):
    with pytest.raises(ValueError, match=match):
        tl.RMSNorm(**args)


@pytest.mark.parametrize("changed,match", [
    (dict(top_k=5), "top_k=5"), (dict(hidden=200), "200"), (dict(width=100), "100"), (dict(weight_format="int4"), "weight_format"), (dict(group_size=48), "group_size"),
    (dict(weight_format="mxfp4", with_zeros=True), "zero points"), (dict(activation="relu"), "activation"), (dict(scores="tanh"), "scores"),
    (dict(groups=3), "groups"), (dict(first=3, held=2), "among 4"), (dict(held=0), "among 4"),
])
def test_experts_refuse(changed, match):
    with pytest.raises(ValueError, match=match):
        tl.W4Experts(**(dict(hidden=256, width=128, experts=4, top_k=2) | changed))


def _filled(gen, device="cpu", **more):
    args = dict(hidden=256, width=128, experts=6, top_k=2) | more
    layer = tl.W4Experts(**args)
    layer.router.copy_(torch.randn(layer.router.shape, generator=gen) / 16)
    if layer.router_bias is not None:
        layer.router_bias.copy_(torch.rand(layer.router_bias.shape, generator=gen))
    if layer.score_bias is not None:
        layer.score_bias.copy_(torch.rand(layer.score_bias.shape, generator=gen) / 4)
    for e in range(layer.held):
        w = [torch.randn(s, generator=gen) / 16 for s in ((layer.width, layer.hidden), (layer.width, layer.hidden), (layer.hidden, layer.width))]
        b = [torch.randn(n, generator=gen) for n in (layer.width, layer.width, layer.hidden)] if layer._bias else []
        layer.load_float_weight(e, *w, *b)
    return layer.to(device)


@pytest.mark.parametrize("more", [dict(), dict(with_zeros=True, bias=True, group_size=32), dict(weight_format="mxfp4", bias=True)])
def test_weights_as_they_are_loaded(more):
    """Quantised weights are within half a step of what was loaded; the state goes from one layer to another."""
    gen = torch.Generator().manual_seed(2)
    layer = tl.W4Experts(256, 128, 3, 2, **more)
    empty = _values(layer, "up")
    w = [torch.randn(s, generator=gen) / 16 for s in ((128, 256), (128, 256), (256, 128))]
    layer.load_float_weight(1, *w)
    value = _values(layer, "up")[1]
    # uint4: half a step of absmax / 7 (or, with zeros, one step of (max - min) / 15: codes and zero point are rounded), scales in fp16;
    # e2m1: half a step of 2 at 4 to 6, one of 2 above 6 (to 8), in units of the largest's power of two over 4
    most = torch.cat(w[:2]).abs().max().item()
    assert (value - torch.cat(w[:2]).double()).abs().max() <= most * (0.26 if "weight_format" in more else 0.14)
    assert torch.equal(_values(layer, "up")[[0, 2]], empty[[0, 2]])
    other = tl.W4Experts(256, 128, 3, 2, **more)
    other.load_state_dict(layer.state_dict())
    assert torch.equal(_values(other, "down"), _values(layer, "down"))
    with pytest.raises(ValueError, match="expert 3"):
        layer.load_float_weight(3, *w)
    with pytest.raises(ValueError, match="down is"):
        layer.load_float_weight(0, w[0], w[1], w[0])
    if not more.get("bias"):
        with pytest.raises(ValueError, match="without bias"):
            layer.load_float_weight(0, *w, down_bias=torch.zeros(256))


def test_types_of_a_converted_layer():
    layer = tl.W4Experts(256, 128, 4, 2, score_bias=True)
    layer.score_bias.fill_(1 / 3)
    assert layer.half().score_bias.dtype == torch.float32 and torch.equal(layer.score_bias, torch.full((4,), 1 / 3))


def _values(layer, name):
    """The held weights in 64 bits."""
    packed, scale = layer._buffers[name].cpu(), layer._buffers[name + "_scale"].cpu()
    codes = torch.stack((packed.view(torch.uint8) & 15, packed.view(torch.uint8) >> 4), dim=-1).flatten(-2)
    if layer._format["weight_format"] == "mxfp4":
        return ref.E2M1[codes.long()] * 2.0 ** (scale.double() - 127).repeat_interleave(32, dim=2)
    zeros = layer._buffers[name + "_zeros"]
    return torch.stack([dequantize_w4_reference(codes[e], scale[e], None if zeros is None else zeros[e].cpu(), layer.group_size) for e in range(len(codes))]).double()


def _held(layer, name):
    """The held weights as the reference takes them."""
    w = ref.Weights.__new__(ref.Weights)
    w.value, w.bias = _values(layer, name), None if not layer._bias else layer._buffers[name + "_bias"].cpu()
    return w


@pytest.mark.gpu
def test_mxfp4_weights_are_the_kernels(cuda):
    gen = torch.Generator().manual_seed(1)
    w = (torch.randn((48, 256), generator=gen) * torch.exp(4 * torch.randn((48, 1), generator=gen))).bfloat16()
    w[3, 64:96], w[4] = 0, 0
    w[5, 7] = 1e30
    codes, scale = layers.quantize_mxfp4(w)
    have = tl.quantize_bf16_mxfp4(48, 256)(w.to(cuda))
    assert torch.equal(have[0].cpu(), codes) and torch.equal(have[1].cpu(), scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_norm(cuda, dtype):
    gen = torch.Generator().manual_seed(4)
    layer = tl.RMSNorm(256, dtype=dtype)
    layer.weight.copy_(torch.randn(256, generator=gen))
    layer = layer.to(cuda)
    x, r = (torch.randn((3, 5, 256), generator=gen).to(dtype) for _ in range(2))
    wide = torch.randn((15, 512), generator=gen).to(dtype)
    # (the shared bounds: they count what rounding adds below fp16's smallest normal number, 2^-25, too)
    for got, rows in ((layer(x.to(cuda)), x), (layer(wide.to(cuda)[:, 256:]), wide[:, 256:]), (layer(x.to(cuda)[0, 0]), x[0, 0]), (layer(wide.to(cuda)[:, 4:260]), wide[:, 4:260])):
        want, _, slack, _ = ref.norm(rows.reshape(-1, 256), None, layer.weight.cpu(), layer.eps)
        assert got.shape == rows.shape and ref.agrees(got.reshape(-1, 256), want, slack, dtype)
    y, total = layer(x.to(cuda), r.to(cuda))
    want, h, slack, h_slack = ref.norm(x.view(-1, 256), r.view(-1, 256), layer.weight.cpu(), layer.eps)
    # (h's rounding in fp32 goes into y where x and r all but cancel)
    slack = slack + h_slack * (want / h).abs().nan_to_num(0.0)
    assert y.shape == total.shape == x.shape and ref.agrees(y.view(-1, 256), want, slack, dtype) and ref.agrees(total.view(-1, 256), h, h_slack, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("fragments,bias", [(False, True), (True, False)])
@pytest.mark.parametrize("rows", [1, 7, 200])
def test_norm_into_bitlinear(cuda, rows, fragments, bias):
    """The norm's int8 rows through BitLinear: the integer product is exact, two quotients in fp32 and the result's rounding follow."""
    gen = torch.Generator().manual_seed(rows)
    norm = tl.RMSNorm(2048, int8=True).to(cuda)
    linear = tl.BitLinear(2048, 96, prefill_fragments=fragments)
    weight = torch.randn((96, 2048), generator=gen)
    linear.load_float_weight(weight, torch.randn(96, generator=gen).half() if bias else None)
    linear = linear.to(cuda)
    if bias:
        linear.bias = linear.bias.to(cuda)
    x, r = (torch.randn((rows, 2048), generator=gen).half().to(cuda) for _ in range(2))
    codes, scale, total = norm(x, r)
    assert codes.dtype == torch.int8 and codes.shape == x.shape and scale.shape == (rows,) and torch.equal(total, (x.float() + r.float()).half())
    got = linear(codes, scale).cpu().double()
    ternary = tl.bitlinear.weight_quant(weight).double()
    want = codes.cpu().double() @ ternary.t() / scale.cpu().double()[:, None] / linear._sw_value
    off = want.abs() * (2.0**-11 + 2.0**-22) + 2.0**-25
    if bias:
        want = want + linear.bias.cpu().double()
        off = off + (want.abs() + off) * 2.0**-11
    assert ((got - want).abs() <= off).all()
    assert torch.equal(linear(codes[None], scale[None])[0].cpu().double(), got)


FORMATS = [dict(), dict(with_zeros=True, bias=True, group_size=64, activation="gelu"), dict(weight_format="mxfp4", bias=True)]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 5, 150])
@pytest.mark.parametrize("more", FORMATS, ids=["uint4", "zeros", "mxfp4"])
@pytest.mark.parametrize("routing", [dict(), dict(scores="sigmoid", router_bias=True, score_bias=True, groups=3, top_groups=2, group_score="sum2", factor=2.5)], ids=["softmax", "groups"])
def test_layer(cuda, tokens, more, routing):
    """The layer's steps, each against the formulas on what the one before gave, and the whole against the steps."""
    print(f"layer {tokens} {more} {routing}", flush=True)
    gen = torch.Generator().manual_seed(tokens)
    layer = _filled(gen, cuda, **more, **routing)
    dtype = layer.router.dtype
    x, r = (torch.randn((tokens, 256), generator=gen).to(dtype).to(cuda) for _ in range(2))
    product, route, sort, up, down, down_onto = layer._make(tokens)
    logits = product(x, layer.router, *([] if layer.router_bias is None else [layer.router_bias]))
    exact = x.cpu().double() @ layer.router.cpu().double().t()
    if layer.router_bias is not None:
        exact = exact + layer.router_bias.cpu().double()
    size = x.cpu().double().abs() @ layer.router.cpu().double().abs().t()
    assert sort is None and ((logits.cpu().double() - exact).abs() <= 274 * 2.0**-24 * (size + 1)).all()
    weights, ids, order, starts = route(logits) if layer.score_bias is None else route(logits, layer.score_bias)
    how = layer._routing
    want, shares = ref.route(logits, layer.score_bias, layer.top_k, how["scores"], how["groups"], how["top_groups"] or how["groups"], how["group_score"], how["renormalize"], how["factor"])
    assert torch.equal(ids.cpu(), want.int()) and torch.allclose(weights.cpu().double(), shares, rtol=2e-5, atol=0)
    got, plain, given = layer(x, r), layer(x), layer(x[None], logits=logits[None])[0]
    h = up(x, *[b for p in ("up", "up_scale", "up_zeros", "up_bias") if (b := layer._buffers[p]) is not None], order, starts)
    order, starts = order.cpu(), starts.cpu()
    assert ref.agrees(h, *ref.up(x, _held(layer, "up"), order, starts, layer.top_k, layer.width, layer._activation), dtype)
    assert ref.agrees(got, *ref.down(h, _held(layer, "down"), order, starts, weights, tokens, r), dtype)
    assert ref.agrees(plain, *ref.down(h, _held(layer, "down"), order, starts, weights, tokens, None), dtype)
    assert torch.equal(plain, given)


@pytest.mark.gpu
def test_many_logits_go_to_the_tiled_product(cuda, monkeypatch):
    """From some number of logits on the layer's router is the tiled GEMM: the same sums in another order."""
    gen = torch.Generator().manual_seed(6)
    layer = _filled(gen, cuda)
    x = torch.randn((90, 256), generator=gen).half().to(cuda)
    few = layer._make(90)[0](x, layer.router)
    monkeypatch.setattr(layers, "TILED_LOGITS", 512)
    product = layer._make(90)[0]
    size = x.cpu().double().abs() @ layer.router.cpu().double().abs().t()
    assert product.name == "matmul" and ((product(x, layer.router) - few).cpu().double().abs() <= 2 * 264 * 2.0**-24 * size).all()
    assert torch.isfinite(layer(x)).all()


@pytest.mark.gpu
def test_parts(cuda, monkeypatch):
    """More tokens than go at once are those parts."""
    gen = torch.Generator().manual_seed(8)
    layer = _filled(gen, cuda)
    x, r = (torch.randn((50, 256), generator=gen).half().to(cuda) for _ in range(2))
    monkeypatch.setattr(layers, "MAX_TOKENS", 16)
    whole = layer(x, r)
    assert torch.equal(whole, torch.cat([layer(x[p : p + 16], r[p : p + 16]) for p in range(0, 50, 16)]))
    monkeypatch.setattr(layers, "MAX_KERNELS", 2)
    for n in (1, 2, 3, 4):
        layer(x[:n])
    assert len(layer._kernels) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 40])
def test_ranks_that_share_a_layer(cuda, tokens):
    """The parts of two layers with some experts each add up to the layer with all."""
    gen = torch.Generator().manual_seed(5)
    whole = _filled(gen, cuda, experts=10, top_k=3)
    x = torch.randn((tokens, 256), generator=gen).half().to(cuda)
    total = torch.zeros((tokens, 256), dtype=torch.float64)
    for first, held in ((0, 4), (4, 6)):
        part = tl.W4Experts(256, 128, 10, 3, first=first, held=held).to(cuda)
        part.load_state_dict({k: v if k == "router" else v[first : first + held] for k, v in whole.state_dict().items()})
        total += part(x).cpu().double()
    want = whole(x).cpu().double()
    # three roundings to fp16, of the parts and of the whole; a part is at most the sum of its choices' sizes: twice the largest here
    most = total.abs().max()
    assert ((total - want).abs() <= 2.0**-11 * (2 * most + want.abs()) + 2.0**-20).all()


@pytest.mark.gpu
def test_blocks_over_a_cache(cuda):
    """Two decoder blocks, norm, attention, norm and experts: prompts in one pass give what token by token gives, and a decode step
    in a graph what it gives without."""
    gen = torch.Generator().manual_seed(11)
    hidden, heads, kv_heads, dim, count, length = 256, 4, 2, 64, 3, 6
    table = tl.rotary_table(64, dim, device=cuda)
    blocks = []
    for _ in range(2):
        attention = tl.W4Attention(hidden, heads, kv_heads, dim, table)
        for linear in (attention.qkv, attention.o):
            linear.load_float_weight(torch.randn((linear.out_features, linear.in_features), generator=gen) / 16)
        blocks.append((tl.RMSNorm(hidden).to(cuda), attention.to(cuda), tl.RMSNorm(hidden).to(cuda), _filled(gen, cuda)))

    def step(x, cache, rows):
        delta = torch.zeros_like(x)
        for i, (norm1, attention, norm2, experts) in enumerate(blocks):
            y, x = norm1(delta, x)
            y, x = norm2(attention(y, cache, rows, i), x)
            delta = experts(y)
        return x.float() + delta.float()

    tokens = torch.randn((count, length, hidden), generator=gen).half().to(cuda)

    def cache():
        return tl.PagedKVCache(count, pages=16, kv_heads=kv_heads, head_dim=dim, page_size=16, layers=2, device=cuda)

    at_once = cache()
    prompts = step(tokens.reshape(-1, hidden), at_once, at_once.extend([length] * count)).view(count, length, hidden)
    one = cache()
    for t in range(length):
        got = step(tokens[:, t].contiguous(), one, one.extend([1] * count))
    assert torch.isfinite(prompts).all()
    # other tiles add in another order and fp16 rounds between the steps; what is compared is a row's direction
    off = (prompts[:, -1] - got).norm(dim=-1) / got.norm(dim=-1)
    assert off.max() <= 2.0**-5

    # one more step, in a graph: what it writes into the cache it writes again, to the same slots
    rows = one.extend([1] * count)
    held = tokens[:, 0].clone()
    step(held, one, rows)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(held, one, rows)
    for t in range(3):
        want = step(tokens[:, t].contiguous(), one, rows)
        held.copy_(tokens[:, t])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.gpu
def test_the_example_runs(cuda, monkeypatch, capsys):
    import importlib.util
    import pathlib

    path = pathlib.Path(__file__).parent.parent / "examples" / "paged_decode.py"
    spec = importlib.util.spec_from_file_location("paged_decode", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    monkeypatch.setattr("sys.argv", ["paged_decode.py", "--layers", "1", "--steps", "2", "--cache", "int8"])
    example.main()
    assert "finite: True" in capsys.readouterr().out
