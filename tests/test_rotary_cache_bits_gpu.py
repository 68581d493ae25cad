"""Rotation and cache write bit by bit: every product and sum of the formula rounded by itself in fp32, whichever kernel takes the heads."""

import pytest
import torch

import tilelang_amd as tl

pytestmark = pytest.mark.gpu

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def _turned(x, table, positions, rotary_dim, interleaved, inverse=False):
    """In fp32, an operation at a time."""
    x, row, half = x.float(), table[positions.long()][:, None], rotary_dim // 2
    c, s = row[..., :half], row[..., half:]
    if inverse:
        s = -s
    first = torch.arange(half, device=x.device) * (2 if interleaved else 1)
    second = first + (1 if interleaved else half)
    a, b, y = x[..., first], x[..., second], x.clone()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    return y


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("dim,rotary_dim", [(128, 128), (80, 32), (80, 40), (72, 20), (256, 256), (40, 6)])
def test_rotation(cuda, dim, rotary_dim, inverse, interleaved, dtype):
    print(f"rotation's bits {dim} r={rotary_dim} inverse {inverse} interleaved {interleaved} {dtype}", flush=True)
    tokens, heads, rows = 500, 3, 5000
    gen = torch.Generator().manual_seed(dim + rotary_dim)
    x = torch.randn((tokens, heads, dim), generator=gen).to(DTYPES[dtype]).to(cuda)
    table = tl.rotary_table(rows, rotary_dim, device=cuda)
    positions = torch.randint(0, rows, (tokens,), generator=gen, dtype=torch.int32).to(cuda)
    got = tl.rotary(tokens, heads, dim, positions=rows, rotary_dim=rotary_dim, interleaved=interleaved, inverse=inverse, dtype=dtype)(x, table, positions)
    assert torch.equal(got, _turned(x, table, positions, rotary_dim, interleaved, inverse).to(got.dtype))


@pytest.mark.parametrize("cache", ["float8_e4m3fn", "int8"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary_dim", [(128, 128), (80, 40), (96, 20)])
def test_codes(cuda, dim, rotary_dim, interleaved, cache):
    """scale = most / top, code = x * (top / most) to the nearest, ties to even, of the fp32 keys and values."""
    print(f"codes {dim} r={rotary_dim} interleaved {interleaved} {cache}", flush=True)
    tokens, heads, kv_heads, rows, page_size = 4000, 2, 4, 5000, 16
    gen = torch.Generator().manual_seed(dim + rotary_dim)
    qkv = torch.randn((tokens, heads + 2 * kv_heads, dim), generator=gen).half().to(cuda)
    table = tl.rotary_table(rows, rotary_dim, device=cuda)
    positions = torch.randint(0, rows, (tokens,), generator=gen, dtype=torch.int32).to(cuda)
    slots = torch.arange(tokens, dtype=torch.int32, device=cuda)
    held, top = (torch.int8, 127.0) if cache == "int8" else (torch.float8_e4m3fn, 448.0)
    shape = (tokens // page_size, kv_heads, page_size, dim)
    kc, vc = (torch.zeros(shape, dtype=torch.uint8, device=cuda).view(held) for _ in range(2))
    ks, vs = (torch.zeros(shape[:3], device=cuda) for _ in range(2))
    tl.rotary_kv_cache_write(tokens, heads, kv_heads=kv_heads, head_dim=dim, pages=shape[0], page_size=page_size, positions=rows, rotary_dim=rotary_dim,
                             interleaved=interleaved, cache_dtype=cache)(qkv, table, positions, slots, kc, vc, ks, vs)
    keys = _turned(qkv[:, heads : heads + kv_heads], table, positions, rotary_dim, interleaved)
    for x, codes, scale in ((keys, kc, ks), (qkv[:, heads + kv_heads :].float(), vc, vs)):
        # (divided as tensors on the CPU: by a number torch multiplies with a rounded reciprocal)
        x = x.cpu()
        most = x.abs().amax(dim=-1)
        tops = torch.full_like(most, top)
        code = x * (tops / most)[..., None]
        code = code.round().clamp(-127, 127).to(held) if cache == "int8" else code.clamp(-448, 448).to(held)
        got = codes.view(torch.uint8).transpose(1, 2).reshape(tokens, kv_heads, dim).cpu()
        assert torch.equal(got, code.view(torch.uint8)) and torch.equal(scale.transpose(1, 2).reshape(tokens, kv_heads).cpu(), most / tops)


def test_more_heads_than_31_bits_of_elements(cuda):
    """A token of 2^23 heads of 256: the keys and values behind them begin beyond 2^31 elements."""
    heads, dim, rows = 2**23, 256, 4
    if torch.cuda.mem_get_info()[0] < 20 * 2**30:
        pytest.skip("not enough memory")
    print(f"one token of {heads} heads of {dim}", flush=True)
    qkv = torch.zeros((1, heads + 2, dim), dtype=torch.float16, device=cuda)
    gen = torch.Generator().manual_seed(1)
    some = torch.randn((1, 3, dim), generator=gen).half().to(cuda)
    qkv[:, heads - 1 :] = some
    table = tl.rotary_table(rows, dim, device=cuda)
    positions, slots = (torch.full((1,), n, dtype=torch.int32, device=cuda) for n in (3, 9))
    kc, vc = (torch.zeros((2, 1, 8, dim), dtype=torch.float16, device=cuda) for _ in range(2))
    q = tl.rotary_kv_cache_write(1, heads, kv_heads=1, head_dim=dim, pages=2, page_size=8, positions=rows)(qkv, table, positions, slots, kc, vc)
    turned = _turned(some[:, :2], table, positions, dim, False).half()
    assert torch.equal(q[:, -1], turned[:, 0]) and torch.equal(kc[1, :, 1], turned[:, 1]) and torch.equal(vc[1, :, 1], some[:, 2])
    assert not q[:, :-1].any() and (kc != 0).any(dim=-1).sum() == 1 and (vc != 0).any(dim=-1).sum() == 1
