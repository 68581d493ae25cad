"""The root-mean-square norm against the formula in 64 bits on the kernel's own inputs."""

import math

import pytest
import torch

import block_reference as ref
import tilelang_amd as tl

pytestmark = pytest.mark.gpu

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def _inputs(seed, rows, dim, dtype, wide=0, size=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, dim + wide), generator=gen) * size).to(DTYPES[dtype]).cuda()
    residual = (torch.randn((rows, dim), generator=gen) * size).to(DTYPES[dtype]).cuda()
    return x[:, :dim], residual, (1 + 0.3 * torch.randn(dim, generator=gen)).to(DTYPES[dtype]).cuda()


def _check(x, residual, weight, dtype, int8, eps=1e-6):
    rows, dim = x.shape
    kernel = tl.rms_norm(rows, dim, eps=eps, dtype=dtype, residual=residual is not None, int8=int8, row_stride=x.stride(0) if rows > 1 else None)
    got = kernel(x, *(() if residual is None else (residual,)), weight)
    got = [got] if isinstance(got, torch.Tensor) else got
    y, h, slack, h_slack = ref.norm(x, residual, weight, eps)
    if int8:
        most = y.abs().amax(dim=1).clamp(min=1e-5)
        assert got[0].dtype == torch.int8 and got[1].dtype == torch.float32
        # the largest value's error, its inverse and product
        assert ((got[1].double() * most / 127 - 1).abs() <= 34 * 2.0**-24).all()
        assert ((got[0].double() - y * got[1].double()[:, None]).abs() <= 0.5 + slack * got[1].double()[:, None] + 127 * 2.0**-24).all()
    else:
        assert ref.agrees(got[0], y, slack, DTYPES[dtype])
    if residual is not None:
        assert ref.agrees(got[-1], h, h_slack, DTYPES[dtype])
    assert all(g.is_contiguous() for g in got) and got[0].shape == (rows, dim)
    return got


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("rows,dim,wide", [
    (1, 8, 0), (1, 4096, 0), (3, 128, 8), (37, 64, 0), (17, 136, 0), (5, 512, 64), (9, 520, 0), (130, 2048, 0), (4, 2056, 0), (3, 2880, 16),
    (2, 4104, 0), (7, 5120, 0), (6, 8192, 0), (2, 8200, 24), (3, 11008, 0), (2, 16384, 0), (2, 16392, 0), (1, 32768, 0), (1100, 72, 0), (700, 1024, 0),
])
def test_norm(cuda, rows, dim, wide, int8, dtype):
    print(f"norm {rows}x{dim}+{wide} int8={int8} {dtype}", flush=True)
    x, residual, weight = _inputs(rows + dim, rows, dim, dtype, wide)
    _check(x, None, weight, dtype, int8)
    _check(x, residual, weight, dtype, int8)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("size,dtype", [(2e4, "float16"), (1e-4, "float16"), (1e25, "bfloat16"), (1e37, "bfloat16"), (1e-25, "bfloat16")])
@pytest.mark.parametrize("dim", [64, 1000, 9000])
def test_large_and_small(cuda, dim, size, dtype, residual):
    """Squares beyond fp32, and values far below eps."""
    print(f"norm of {size} dim={dim} {dtype} {residual}", flush=True)
    x, r, weight = _inputs(3, 5, dim, dtype, size=size)
    _check(x, r if residual else None, weight, dtype, False)


@pytest.mark.parametrize("dim", [128, 512, 4096, 10000])
def test_infinities_and_nan(cuda, dim):
    """They stay in their rows; rows of zeros give zeros."""
    x, residual, weight = _inputs(5, 9, dim, "float16")
    x[1, dim // 2], x[4, 3], x[6, dim - 1] = math.nan, math.inf, -math.inf
    x[2], residual[2] = 0, 0
    print(f"norm with NaN dim={dim}", flush=True)
    good = [0, 2, 3, 5, 7, 8]
    for int8 in (False, True):
        got = tl.rms_norm(9, dim, residual=True, int8=int8)(x, residual, weight)
        y, h, slack, _ = ref.norm(x, residual, weight, 1e-6)
        value = got[0].double() / got[1].double()[:, None] if int8 else got[0].double()
        off = 0.51 / got[1].double()[good][:, None] if int8 else ref.rounded(y, slack, torch.float16)[good]
        assert ((value - y)[good].abs() <= off).all() and (value[2] == 0).all()
        assert torch.isnan(value[1]).all()
        for r in (4, 6):
            assert torch.isnan(value[r]).all() if int8 else torch.isnan(value[r]).sum() == 1
        if int8:
            assert (got[0][[1, 4, 6]] == 0).all()
        assert torch.equal(torch.isfinite(got[-1]), torch.isfinite(h))


def test_small_rows_of_codes(cuda):
    """Below 1e-5 a row's codes shrink with it, as the activation quantiser's do."""
    x = torch.full((2, 256), 2.0**-20, dtype=torch.bfloat16, device=cuda)
    weight = torch.ones(256, dtype=torch.bfloat16, device=cuda)
    codes, scale = tl.rms_norm(2, 256, eps=1.0, dtype="bfloat16", int8=True)(x, weight)
    assert (scale.double() - 127e5).abs().max() <= 127e5 * 2.0**-22 and (codes == 12).all()  # 2^-20 * 127e5 = 12.1


def test_feeds_the_ternary_product(cuda):
    """The codes and scales go straight into the int8 x 2-bit product."""
    from tilelang_amd import quantize
    from tilelang_amd.kernels import bitlinear_int8xint2

    gen = torch.Generator().manual_seed(1)
    rows, dim, out = 33, 1024, 96
    x, residual, weight = _inputs(2, rows, dim, "float16")
    w = torch.randint(-1, 2, (out, dim), generator=gen)
    packed = quantize.general_compress((w + 2).to(torch.int8), source_bits=2).cuda()
    codes, scale, _ = tl.rms_norm(rows, dim, residual=True, int8=True)(x, residual, weight)
    got = bitlinear_int8xint2(rows, out, dim, 2.0)(codes, packed, scale)
    want = (codes.double().cpu() @ w.double().t()) / scale.double().cpu()[:, None] / 2.0
    # two quotients and the output's rounding
    assert ref.agrees(got, want, 3 * 2.0**-24 * want.abs(), torch.float16)
