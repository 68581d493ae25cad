"""RMSNorm, W4Experts and BitLinear on int8 rows: batches of no tokens, and what a call is checked for before it goes to a kernel."""

import ctypes
import pathlib
import subprocess
import sys

import pytest
import torch

import tilelang_amd as tl
from tilelang_amd import _lib, bitlinear
from tilelang_amd import experts as layers
from tilelang_amd.block_kernels import EXPERTS_MXFP4


@pytest.mark.parametrize("lead", [(0,), (0, 5), (3, 0)])
@pytest.mark.parametrize("int8", [False, True])
def test_norm_of_no_rows(lead, int8):
    """A step that has no token here: results of no rows, no launch."""
    norm = tl.RMSNorm(64, dtype="bfloat16", int8=int8)
    x = torch.zeros((*lead, 64))
    first = norm(x)
    both = norm(x, x)
    if int8:
        codes, scale = first
        assert codes.shape == x.shape and codes.dtype == torch.int8 and scale.shape == lead and scale.dtype == torch.float32
        assert [t.dtype for t in both] == [torch.int8, torch.float32, torch.bfloat16] and both[1].shape == lead
        linear = tl.BitLinear(128, 96)
        out = linear(codes.new_zeros((*lead, 128)), scale)
        assert out.shape == (*lead, 96) and out.dtype == torch.float16
    else:
        assert first.shape == x.shape and first.dtype == torch.bfloat16 and [t.dtype for t in both] == [torch.bfloat16] * 2
    assert both[-1].shape == both[0].shape == x.shape


@pytest.mark.parametrize("lead", [(0,), (0, 5), (3, 0)])
@pytest.mark.parametrize("weight_format", ["uint4", "mxfp4"])
def test_experts_of_no_tokens(lead, weight_format):
    layer = tl.W4Experts(256, 128, 4, 2, weight_format)
    x = torch.zeros((*lead, 256))
    for out in (layer(x), layer(x, x), layer(x, logits=torch.zeros((*lead, 4)))):
        assert out.shape == x.shape and out.dtype == layer.router.dtype


@pytest.mark.parametrize("hidden,width,top_k,tokens", [(7168, 2048, 8, 70000), (16384, 16384, 32, 65536), (4096, 14336, 2, 65536), (2560, 2560, 4, 65536), (128, 128, 1, 200000)])
def test_parts_take_bounded_memory(monkeypatch, hidden, width, top_k, tokens):
    """What goes through the experts at once: the rows between the two products and the sums' workspace stay below a bound."""
    with torch.device("meta"):
        layer = tl.W4Experts(hidden, width, 64, top_k)
        x = torch.empty((tokens, hidden), dtype=torch.float16)
    parts = []

    def one(rows, residual, logits):
        parts.append(rows.shape[0])
        return torch.empty_like(rows)

    monkeypatch.setattr(layer, "_pass", one)
    assert layer(x).shape == x.shape and sum(parts) == tokens
    for n in set(parts):
        room = _lib.load_library().dq_experts_down_workspace_bytes(n, 64, top_k, hidden, width, 128, 0, 64)
        assert room + n * top_k * width * 2 <= layers.PART_BYTES and n <= layers.MAX_TOKENS
    # no more parts than that takes
    assert len(parts) <= 2 + tokens // layers.MAX_TOKENS + tokens * top_k * (4 * hidden + 2 * width) // layers.PART_BYTES


def test_bitlinear_keeps_the_kernels_of_its_last_sizes(monkeypatch):
    """Prompts come in any number of rows: kernel objects are kept for the last ones, of either kind of rows."""
    made = []

    def make(M, N, K, *args, **more):
        made.append(M)
        return lambda x, weight, *scale: torch.zeros((M, N), dtype=torch.float16)

    monkeypatch.setattr(bitlinear.kernels, "bitlinear_int8xint2", make)
    monkeypatch.setattr(bitlinear.kernels, "bitlinear_fp16", make)
    layer = tl.BitLinear(128, 32)
    for M in range(1, 200):
        assert layer(torch.zeros((M, 128), dtype=torch.int8), torch.ones(M)).shape == (M, 32)
        assert layer(torch.zeros((M, 128), dtype=torch.float16)).shape == (M, 32)
        layer(torch.zeros((7, 128), dtype=torch.int8), torch.ones(7))
    assert len(layer._kernels) == len(layer._codes_kernels) == bitlinear.MAX_KERNELS
    assert made.count(7) == 2  # (one of a kind: in use, it stays; the fp16 rows' goes by when it was made)
    layer.load_packed_weight(layer.qweight, 2.0)
    assert not layer._kernels and not layer._codes_kernels


def test_rows_that_are_not_x_s_are_refused(monkeypatch):
    """A residual or logits of as many elements as x but of other rows, and an x of other rows than the layer's."""
    norm, layer = tl.RMSNorm(64), tl.W4Experts(256, 128, 4, 2)
    monkeypatch.setattr(layer, "_pass", lambda rows, residual, logits: torch.empty_like(rows))
    monkeypatch.setattr(layers.block_kernels, "rms_norm", lambda *a: lambda x, *r: [torch.empty_like(x) for _ in range(1 + (len(r) == 2))])
    x = torch.zeros((2, 3, 64))
    for shape in ((3, 2, 64), (2, 64, 3), (6, 32), (5, 64), (64,), (1, 3, 64), (2, 3, 128)):
        with pytest.raises(ValueError, match="RMSNorm: residual is"):
            norm(x, torch.zeros(shape))
    assert norm(x, torch.zeros((6, 64)))[1].shape == x.shape and norm(x[0], torch.zeros((1, 3, 64)))[0].shape == (3, 64)
    x = torch.zeros((2, 3, 256))
    for bad in (torch.zeros((2, 6, 128)), torch.zeros((2, 512)), torch.zeros((5, 0)), torch.zeros(512)):
        with pytest.raises(ValueError, match="W4Experts: x is"):
            layer(bad)
    for shape in ((3, 2, 256), (6, 128), (5, 256), (256,), (2, 256, 3)):
        with pytest.raises(ValueError, match="W4Experts: residual is"):
            layer(x, torch.zeros(shape))
    for shape in ((3, 2, 4), (6, 8), (7, 4), (2, 4, 3), (2, 3, 5)):
        with pytest.raises(ValueError, match="W4Experts: logits is"):
            layer(x, logits=torch.zeros(shape))
    with pytest.raises(ValueError, match="W4Experts: residual is"):
        layer(x[:0], x)
    assert layer(x, torch.zeros((6, 256)), torch.zeros((6, 4))).shape == x.shape
    assert layer(x[0, 0], x[0, 0], torch.zeros(4)).shape == (256,)


@pytest.mark.parametrize("apart", [2**31 - 8, 2**31, 2**33])
def test_norm_of_rows_far_apart(monkeypatch, apart):
    """Rows of x further apart than a kernel's row stride goes are copied together."""
    rms_norm, strides = layers.block_kernels.rms_norm, []

    def make(rows, dim, eps, dtype, residual, int8, stride):
        strides.append(rms_norm(rows, dim, eps, dtype, residual, int8, stride).params[0].strides)
        return lambda x, weight: torch.empty_like(x)

    norm = tl.RMSNorm(64)
    monkeypatch.setattr(layers.block_kernels, "rms_norm", make)
    x = torch.empty_strided((2, 64), (apart, 1), dtype=torch.float16, device="meta")
    assert norm(x).shape == (2, 64) and strides == [(apart, 1) if apart < 2**31 else None]


def test_down_refuses_rows_beyond_32_bit_offsets():
    """All choices of 16 tokens may be one expert's: 128 rows of 2^26 elements are 16 GiB from a tile's first to its last."""
    entry = dict(tokens=16, experts=2, top_k=32, N=32, K=2**26, group_size=32, format=EXPERTS_MXFP4, first=0, routed=2)
    assert tl.experts_down(16, 2, 2, 32, 2**26, "mxfp4").name == "experts_down"
    with pytest.raises(ValueError, match="128 rows of h"):
        tl.experts_down(16, 2, 32, 32, 2**26, "mxfp4")
    lib, p = _lib.load_library(), ctypes.c_void_p(1 << 20)  # (never followed: the checks come first)
    rc = lib.call_experts_down(p, p, p, None, None, p, p, p, p, None, p, p, 1 << 40, *entry.values(), None)
    assert rc == -1 and "128 rows of H" in lib.get_last_error().decode()


def test_no_workspace_for_sizes_that_calls_refuse():
    """In a process of its own: a quotient of the first's sizes ended it."""
    asked = [("down", (64, 8, 2, 64, 2**31 - 255, 128, 0, 8)), ("down", (64, 8, 2, 2**31 - 32, 2**31 - 128, 128, 0, 8)), ("down", (64, 2000, 2, 64, 256, 128, 0, 2000)),
             ("down", (64, 8, 33, 64, 256, 128, 0, 8)), ("order", (500, 2, 2**31 - 1)), ("order", (500, 33, 64))]
    code = "from tilelang_amd import _lib; lib = _lib.load_library(); print(" + ", ".join(f"lib.dq_experts_{name}_workspace_bytes(*{sizes})" for name, sizes in asked) + ")"
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=pathlib.Path(__file__).parent.parent)
    assert done.returncode == 0 and done.stdout.split() == ["0"] * len(asked), (done.returncode, done.stdout, done.stderr)


def test_scales_that_are_not_the_codes_are_refused(monkeypatch):
    monkeypatch.setattr(bitlinear.kernels, "bitlinear_int8xint2", lambda M, N, K, *args, **more: lambda x, weight, scale: torch.zeros((M, N), dtype=torch.float16))
    layer = tl.BitLinear(128, 32)
    codes = torch.zeros((2, 3, 128), dtype=torch.int8)
    for shape in ((3, 2), (2, 3, 2), (5,), (), (2, 1, 3)):
        with pytest.raises(ValueError, match="BitLinear: scale is"):
            layer(codes, torch.ones(shape))
    for bad in (torch.zeros((2, 3, 64), dtype=torch.int8), torch.zeros((2, 384), dtype=torch.int8)):
        with pytest.raises(ValueError, match="BitLinear: codes are"):
            layer(bad, torch.ones(bad.shape[:-1]))
    for shape in ((2, 3), (2, 3, 1), (6,), (6, 1)):
        assert layer(codes, torch.ones(shape)).shape == (2, 3, 32)
