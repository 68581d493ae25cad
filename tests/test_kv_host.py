"""Rotation, cache and attention without a GPU: what the factories, the kernel objects and the entry points refuse, and the
rotation's table."""

import ctypes
import math

import pytest
import torch

import tilelang_amd as tl
from tilelang_amd import _lib
from tilelang_amd.kv_kernels import CACHE_BF16, CACHE_F16, CACHE_FP8, CACHE_I8, DT_BF16, DT_F16

POOL = dict(kv_heads=2, head_dim=64, pages=3, page_size=16)


@pytest.mark.parametrize("make,match", [
    (lambda: tl.rotary(0, 1, 64, positions=1), "tokens must be positive"),
    (lambda: tl.rotary(1, 1, 60, positions=1), "head_dim=60"),
    (lambda: tl.rotary(1, 1, 520, positions=1), "head_dim=520"),
    (lambda: tl.rotary(1, 1, 64, positions=1, rotary_dim=65), "rotary_dim=65"),
    (lambda: tl.rotary(1, 1, 64, positions=1, rotary_dim=0), "rotary_dim=0"),
    (lambda: tl.rotary(1, 1, 64, positions=0), "positions must be positive"),
    (lambda: tl.rotary(1, 2, 64, positions=1, row_stride=64), "row_stride=64"),
    (lambda: tl.rotary(1, 2, 64, positions=1, row_stride=132), "row_stride=132"),
    (lambda: tl.rotary(1, 2, 64, positions=1, dtype="float32"), "dtype must be"),
    (lambda: tl.kv_cache_write(1, **POOL | {"page_size": 12}), "page_size=12"),
    (lambda: tl.kv_cache_write(1, **POOL | {"page_size": 4}), "page_size=4"),
    (lambda: tl.kv_cache_write(1, **POOL | {"head_dim": 264}), "head_dim=264"),
    (lambda: tl.kv_cache_write(1, **POOL | {"pages": 2**28}), "slots are 32-bit"),
    (lambda: tl.kv_cache_write(1, **POOL, cache_dtype="bfloat16"), "cache_dtype must be"),
    (lambda: tl.kv_cache_write(1, **POOL, cache_dtype="int32"), "cache_dtype must be"),
    (lambda: tl.rotary_kv_cache_write(1, 0, positions=1, **POOL), "heads must be positive"),
    (lambda: tl.rotary_kv_cache_write(1, 4, positions=1, rotary_dim=66, **POOL), "rotary_dim=66"),
    (lambda: tl.kv_cache_read(0, 1, max_pages=1, **POOL), "sequences must be positive"),
    (lambda: tl.paged_attention_decode(1, 3, max_pages=1, **POOL), "multiple of kv_heads"),
    (lambda: tl.paged_attention_decode(1, 4, max_pages=1, **POOL | {"head_dim": 72}), "head_dim=72"),
    (lambda: tl.paged_attention_decode(1, 4, max_pages=1, window=-1, **POOL), "window=-1"),
    (lambda: tl.paged_attention_decode(1, 4, max_pages=1, scale=math.inf, **POOL), "scale must be finite"),
    (lambda: tl.rotary_table(4, 7), "rotary_dim=7"),
    (lambda: tl.rotary_table(4, 8, scaling="twice"), "unknown scaling"),
    (lambda: tl.rotary_table(4, 8, scaling="bands"), "original_positions"),
])
def test_factories_refuse(make, match):
    with pytest.raises(ValueError, match=match):
        make()


def _operands(kernel, device="cpu"):
    return [torch.zeros(p.shape, dtype=p.dtype, device=device) for i, p in enumerate(kernel.params)
            if i not in kernel.result_idx and i not in kernel.workspace_idx]


@pytest.mark.parametrize("kernel", [
    tl.rotary(3, 2, 64, positions=5), tl.kv_cache_write(3, **POOL), tl.kv_cache_write(3, cache_dtype="int8", **POOL),
    tl.rotary_kv_cache_write(3, 4, positions=5, cache_dtype="float8_e4m3fn", **POOL), tl.kv_cache_read(2, 9, max_pages=2, **POOL),
    tl.paged_attention_decode(2, 4, max_pages=2, sinks=True, **POOL), tl.paged_attention_decode(2, 4, max_pages=900, with_lse=True, **POOL),
], ids=lambda k: k.name)
def test_kernel_objects_refuse(kernel):
    good = _operands(kernel)
    with pytest.raises(ValueError, match="device mismatch"):
        kernel(*good)
    with pytest.raises(ValueError, match="Expected .* inputs"):
        kernel(*good[:-1])


def test_view_of_wider_rows():
    """Which views a kernel object of a row stride takes (the look alone: no launch)."""
    p = tl.rotary(3, 2, 64, positions=5, row_stride=5 * 64).params[0]
    wide = torch.zeros((3, 5, 64), dtype=torch.float16)
    assert p.lies_as(wide[:, :2]) and p.lies_as(wide[:, 3:]) and not p.lies_as(torch.zeros((3, 2, 64), dtype=torch.float16))
    assert not p.lies_as(torch.zeros((3, 2, 128), dtype=torch.float16)[..., ::2])
    one = tl.rotary(1, 2, 64, positions=5, row_stride=5 * 64).params[0]
    assert one.lies_as(torch.zeros((1, 2, 64), dtype=torch.float16))


def _entry(name, **changed):
    """Calls an entry point with arguments that are good but for `changed`; the pointers are never followed: the checks come first."""
    p = ctypes.c_void_p(1 << 20)
    args = {
        "call_rotary": dict(X=p, Table=p, Positions=p, Out=p, tokens=2, heads=2, head_dim=64, rotary_dim=64, positions=3, row_stride=128,
                            interleaved=0, inverse=0, dtype=DT_F16),
        "call_kv_cache_write": dict(K=p, V=p, Slots=p, KCache=p, VCache=p, KScale=p, VScale=p, tokens=2, kv_heads=2, head_dim=64, pages=2,
                                    page_size=16, dtype=DT_F16, cache=CACHE_I8),
        "call_rotary_kv_cache_write": dict(QKV=p, Table=p, Positions=p, Slots=p, Q=p, KCache=p, VCache=p, KScale=p, VScale=p, tokens=2, heads=4,
                                           kv_heads=2, head_dim=64, rotary_dim=64, positions=3, pages=2, page_size=16, interleaved=0,
                                           dtype=DT_F16, cache=CACHE_FP8),
        "call_kv_cache_read": dict(KCache=p, VCache=p, KScale=p, VScale=p, PageTable=p, Starts=p, KV=p, sequences=1, tokens=2, kv_heads=2,
                                   head_dim=64, pages=2, page_size=16, max_pages=1, dtype=DT_F16, cache=CACHE_I8),
        "call_paged_attention_decode": dict(Q=p, KCache=p, VCache=p, KScale=p, VScale=p, PageTable=p, Lengths=p, Sinks=None, Out=p, Lse=None,
                                            Workspace=p, bytes=1 << 30, sequences=1, heads=4, kv_heads=2, head_dim=64, pages=2, page_size=16,
                                            max_pages=1, window=0, dtype=DT_F16, cache=CACHE_I8, scale=1.0),
    }[name]
    assert set(changed) <= set(args)
    lib = _lib.load_library()
    rc = getattr(lib, name)(*(args | changed).values(), None)
    return rc, lib.get_last_error().decode()


ODD = ctypes.c_void_p((1 << 20) + 2)


@pytest.mark.parametrize("name,changed,match", [
    ("call_rotary", dict(X=None), "non-NULL"),
    ("call_rotary", dict(Out=ODD), "16-byte aligned"),
    ("call_rotary", dict(Positions=ODD), "4-byte aligned"),
    ("call_rotary", dict(dtype=3), "dtype must be"),
    ("call_rotary", dict(tokens=0), "must be positive"),
    ("call_rotary", dict(tokens=1 << 25), "at most"),
    ("call_rotary", dict(head_dim=68), "head_dim must be"),
    ("call_rotary", dict(rotary_dim=63), "rotary_dim must be"),
    ("call_rotary", dict(positions=0), "must have a row"),
    ("call_rotary", dict(row_stride=120), "row_stride must be"),
    ("call_kv_cache_write", dict(page_size=24), "page_size must be"),
    ("call_kv_cache_write", dict(page_size=2048), "page_size must be"),
    ("call_kv_cache_write", dict(page_size=0), "page_size must be"),
    ("call_kv_cache_write", dict(pages=0), "must be positive"),
    ("call_kv_cache_write", dict(pages=1 << 30), "slots are 32-bit"),
    ("call_kv_cache_write", dict(cache=4), "unknown cache format"),
    ("call_kv_cache_write", dict(cache=CACHE_BF16), "same type"),
    ("call_kv_cache_write", dict(cache=CACHE_F16, dtype=DT_BF16), "same type"),
    ("call_kv_cache_write", dict(VScale=None), "8-bit cache"),
    ("call_kv_cache_write", dict(K=ODD), "16-byte"),
    ("call_kv_cache_write", dict(Slots=None), "non-NULL"),
    ("call_rotary_kv_cache_write", dict(heads=0), "heads must be positive"),
    ("call_rotary_kv_cache_write", dict(Q=None), "non-NULL"),
    ("call_rotary_kv_cache_write", dict(Table=ODD), "16-byte"),
    ("call_rotary_kv_cache_write", dict(head_dim=512, rotary_dim=2), "at most 256"),
    ("call_kv_cache_read", dict(sequences=0), "must be positive"),
    ("call_kv_cache_read", dict(PageTable=None), "PageTable"),
    ("call_kv_cache_read", dict(max_pages=1 << 28), "lengths are 32-bit"),
    ("call_kv_cache_read", dict(KV=ODD), "16-byte"),
    ("call_kv_cache_read", dict(kv_heads=8192), "524280 elements"),
    ("call_paged_attention_decode", dict(heads=5), "multiple of kv_heads"),
    ("call_paged_attention_decode", dict(head_dim=72), "head_dim must be"),
    ("call_paged_attention_decode", dict(window=-1), "window must be"),
    ("call_paged_attention_decode", dict(sequences=60000, max_pages=1 << 26), "the work that a call counts"),
    ("call_paged_attention_decode", dict(max_pages=(1 << 27) - 1), "lengths are 32-bit"),
    ("call_paged_attention_decode", dict(scale=math.nan), "scale must be finite"),
    ("call_paged_attention_decode", dict(sequences=70000), "at most 65535"),
    ("call_paged_attention_decode", dict(Lengths=None), "non-NULL"),
    ("call_paged_attention_decode", dict(Sinks=ODD), "4-byte"),
    ("call_paged_attention_decode", dict(max_pages=1000, bytes=16), "needs a 16-byte aligned workspace"),
    ("call_paged_attention_decode", dict(max_pages=1000, Workspace=None), "needs a 16-byte aligned workspace"),
])
def test_entry_points_refuse(name, changed, match):
    rc, message = _entry(name, **changed)
    assert rc == -1 and match in message and message.startswith(name), message


def test_table():
    """The angles of each scaling by their definitions, position by position."""
    r, base, rows, factor, trained = 16, 10000.0, 40, 4.0, 64
    plain = [base ** (-2 * i / r) for i in range(r // 2)]

    def bands(f):
        turns = trained * f / (2 * math.pi)
        share = min(1.0, max(0.0, (turns - 1.0) / 3.0))
        return share * f + (1 - share) * f / factor

    def index(turns):
        return r * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))

    def ramp(i, f):
        first, last = max(math.floor(index(4.0)), 0), min(math.ceil(index(1.0)), r - 1)
        share = 1 - min(1.0, max(0.0, (i - first) / (last - first)))
        return share * f + (1 - share) * f / factor

    grown = base * factor ** (r / (r - 2))
    want = {
        None: (plain, 1.0), "linear": ([f / factor for f in plain], 1.0), "base": ([grown ** (-2 * i / r) for i in range(r // 2)], 1.0),
        "bands": ([bands(f) for f in plain], 1.0), "ramp": ([ramp(i, f) for i, f in enumerate(plain)], 0.1 * math.log(factor) + 1.0),
    }
    for scaling, (f, magnitude) in want.items():
        got = tl.rotary_table(rows, r, scaling=scaling, factor=factor, original_positions=trained)
        assert got.shape == (rows, r) and got.dtype == torch.float32
        for p in (0, 1, 17, rows - 1):
            for i in range(r // 2):
                assert abs(float(got[p, i]) - magnitude * math.cos(p * f[i])) < 1e-7 * 2
                assert abs(float(got[p, r // 2 + i]) - magnitude * math.sin(p * f[i])) < 1e-7 * 2
    # the slowest angle of a grown base is slowed by the factor, the fastest kept
    assert abs(want["base"][0][-1] * factor / plain[-1] - 1) < 1e-12 and want["base"][0][0] == plain[0]


def test_workspace_is_named_without_a_gpu():
    room = _lib.load_library().dq_paged_attention_workspace_bytes
    assert room(1, 32, 8, 128, 16, 1, 0, CACHE_F16) == 0  # one tile: nothing to join
    assert room(1, 32, 8, 128, 16, 1000, 0, CACHE_F16) > 0
    assert room(0, 32, 8, 128, 16, 1000, 0, CACHE_F16) == 0 and room(1, 33, 8, 128, 16, 1000, 0, CACHE_F16) == 0


def test_a_window_beyond_every_length():
    room = _lib.load_library().dq_paged_attention_workspace_bytes
    sizes = (1, 32, 8, 128, 16, 1000)
    for window in (16000 - 31, 16000, 2**31 - 32, 2**31 - 1):
        assert room(*sizes, window, CACHE_F16) == room(*sizes, 0, CACHE_F16)
    pool = dict(kv_heads=2, head_dim=64, pages=8, page_size=16, max_pages=4)
    for window in (64, 2**31, 2**32 + 5):  # 32 bits of the last are 5
        assert tl.paged_attention_decode(1, 4, window=window, **pool)._native_spec[2][7] == 64
