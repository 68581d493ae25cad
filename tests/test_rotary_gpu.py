"""Rotary positions against the formula in 64 bits on the kernel's own inputs; the gradient also against differences."""

import pytest
import torch

import tilelang_amd as tl
from kv_reference import HALF_ULP, rotate

pytestmark = pytest.mark.gpu

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def _inputs(seed, tokens, heads, dim, dtype, device, wide=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((tokens, heads + wide, dim), generator=gen).to(DTYPES[dtype]).to(device)
    return x[:, :heads], gen


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,rotary_dim,wide", [
    (1, 1, 8, 2, 0), (1, 40, 128, 128, 0), (3, 5, 64, 64, 2), (37, 3, 80, 32, 1), (7, 9, 96, 24, 0), (5, 4, 256, 256, 4),
    (2, 3, 512, 512, 0), (19, 2, 40, 6, 0), (1500, 20, 128, 64, 8), (900, 7, 72, 70, 0), (2, 1, 264, 136, 1),
    (123, 6, 80, 40, 2),
])
def test_rotary(cuda, tokens, heads, dim, rotary_dim, wide, interleaved, dtype):
    print(f"rotary {tokens}x{heads}x{dim} r={rotary_dim} wide={wide} {interleaved} {dtype}", flush=True)
    x, gen = _inputs(tokens + dim, tokens, heads, dim, dtype, cuda, wide)
    rows = 300
    table = tl.rotary_table(rows, rotary_dim, device=cuda)
    positions = torch.randint(0, rows, (tokens,), generator=gen, dtype=torch.int32).to(cuda)
    for inverse in (False, True):
        kernel = tl.rotary(tokens, heads, dim, positions=rows, rotary_dim=rotary_dim, interleaved=interleaved, inverse=inverse, dtype=dtype,
                           row_stride=(heads + wide) * dim)
        got = kernel(x, table, positions)
        want, slack = rotate(x, table, positions, rotary_dim, interleaved, inverse)
        assert got.shape == x.shape and got.is_contiguous()
        off = (got.double() - want).abs()
        # the exact value's rounding, once more where the fp32 error moves it over a boundary; 2^-25: fp16's smallest steps
        assert (off <= HALF_ULP[x.dtype] * want.abs() * 1.01 + slack * 1.01 + 2.0**-25).all(), off.max()
        assert torch.equal(got[..., rotary_dim:], x[..., rotary_dim:])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rotary_dim", [128, 48, 56, 20])
def test_rotary_in_place_in_a_fused_projection(cuda, interleaved, rotary_dim):
    tokens, heads, wide, dim = 700, 10, 3, 128
    x, gen = _inputs(3, tokens, heads, dim, "bfloat16", cuda, wide)
    whole = x._base if x._base is not None else x
    behind = whole[:, heads:].clone()
    table = tl.rotary_table(tokens, rotary_dim, device=cuda)
    positions = torch.arange(tokens, dtype=torch.int32, device=cuda).flip(0).contiguous()
    sizes = dict(positions=tokens, rotary_dim=rotary_dim, interleaved=interleaved, dtype="bfloat16", row_stride=(heads + wide) * dim)
    want = tl.rotary(tokens, heads, dim, **sizes)(x, table, positions)
    assert tl.rotary(tokens, heads, dim, in_place=True, **sizes)(x, table, positions) is None
    assert torch.equal(x, want) and torch.equal(whole[:, heads:], behind)


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_against_differences(cuda, interleaved):
    """f(x) = sum(w * rotary(x)): its derivative along e is (f(x + e) - f(x - e)) / 2, as f is linear, and <grad f, e>."""
    tokens, heads, dim, rotary_dim, rows = 9, 4, 64, 48, 4096
    gen = torch.Generator().manual_seed(11)
    # multiples of 1/8 below 4: x +- e are exact in fp16, so the only roundings are the kernel's
    x, e = (torch.randint(-31, 32, (tokens, heads, dim), generator=gen).to(cuda) / 8 for _ in range(2))
    w = torch.randn((tokens, heads, dim), generator=gen).half().to(cuda)
    table = tl.rotary_table(rows, rotary_dim, scaling="ramp", factor=8.0, original_positions=512, device=cuda)
    positions = torch.randint(0, rows, (tokens,), generator=gen, dtype=torch.int32).to(cuda)
    sizes = dict(positions=rows, rotary_dim=rotary_dim, interleaved=interleaved)
    forward, backward = tl.rotary(tokens, heads, dim, **sizes), tl.rotary(tokens, heads, dim, inverse=True, **sizes)
    up, down = (forward((x + s * e).half(), table, positions).double() for s in (1, -1))
    difference = (w.double() * (up - down)).sum() / 2
    gradient = backward(w, table, positions).double()
    along = (gradient * e.double()).sum()
    # every output and gradient element is rounded once
    slack = HALF_ULP[torch.float16] * 1.1 * ((w.double().abs() * (up.abs() + down.abs())).sum() / 2 + (gradient.abs() * e.double().abs()).sum())
    assert (difference - along).abs() <= slack


def test_long_positions(cuda):
    """At a million tokens the angles still have their 64-bit values: the table's, not a product's in fp32."""
    rows, dim = 1_000_001, 64
    table = tl.rotary_table(rows, dim, device=cuda)
    positions = torch.tensor([0, 1, 999_999, 1_000_000], dtype=torch.int32, device=cuda)
    x = torch.randn((4, 2, dim), generator=torch.Generator().manual_seed(5)).half().to(cuda)
    got = tl.rotary(4, 2, dim, positions=rows)(x, table, positions).double()
    f = 10000.0 ** (-2 * torch.arange(dim // 2, dtype=torch.float64) / dim)
    angle = (positions.cpu().double()[:, None] * f).to(cuda)[:, None]
    a, b = x[..., : dim // 2].double(), x[..., dim // 2 :].double()
    want = torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], dim=-1)
    assert ((got - want).abs() <= HALF_ULP[torch.float16] * 1.01 * want.abs() + 2.0**-21 * 8).all()


def test_position_outside_of_the_table_is_nan(cuda):
    for interleaved, rotary_dim in ((False, 32), (True, 32), (False, 10)):
        table = tl.rotary_table(4, rotary_dim, device=cuda)
        x = torch.ones((4, 2, 64), dtype=torch.float16, device=cuda)
        positions = torch.tensor([-1, 3, 4, 2**31 - 1], dtype=torch.int32, device=cuda)
        got = tl.rotary(4, 2, 64, positions=4, rotary_dim=rotary_dim, interleaved=interleaved)(x, table, positions)
        assert torch.isnan(got[[0, 2, 3], :, :rotary_dim]).all() and not torch.isnan(got[1]).any() and not torch.isnan(got[..., rotary_dim:]).any()


def test_graph_and_side_stream(cuda):
    tokens, heads, dim = 65, 12, 128
    x, _ = _inputs(8, tokens, heads, dim, "float16", cuda)
    table = tl.rotary_table(tokens, dim, device=cuda)
    positions = torch.arange(tokens, dtype=torch.int32, device=cuda)
    kernel = tl.rotary(tokens, heads, dim, positions=tokens)
    eager = kernel(x, table, positions)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = kernel(x, table, positions)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
