"""Norm, routing and the experts' products without a GPU: what the factories, the kernel objects and the entry points refuse, and what
the workspaces are."""

import ctypes
import math

import pytest
import torch

import tilelang_amd as tl
from tilelang_amd import _lib
from tilelang_amd.block_kernels import DT_F32, EXPERTS_MXFP4, EXPERTS_UINT4
from tilelang_amd.kv_kernels import DT_F16

ROUTE, PRODUCT = dict(tokens=5, experts=16, top_k=2), dict(tokens=5, experts=16, top_k=2, N=64, K=256)


@pytest.mark.parametrize("make,match", [
    (lambda: tl.rms_norm(0, 64), "rows must be positive"),
    (lambda: tl.rms_norm(2**31, 64), "below 2\\^31"),
    (lambda: tl.rms_norm(1, 60), "dim=60"),
    (lambda: tl.rms_norm(1, 32776), "dim=32776"),
    (lambda: tl.rms_norm(1, 64, eps=0), "eps must be"),
    (lambda: tl.rms_norm(1, 64, eps=math.nan), "eps must be"),
    (lambda: tl.rms_norm(1, 64, dtype="float32"), "dtype must be"),
    (lambda: tl.rms_norm(2, 64, row_stride=56), "row_stride=56"),
    (lambda: tl.rms_norm(2, 64, row_stride=68), "row_stride=68"),
    (lambda: tl.rms_norm(2, 64, row_stride=2**31), "row_stride="),
    (lambda: tl.router_logits(0, 16, 64), "tokens"),
    (lambda: tl.router_logits(1, 1025, 64), "experts"),
    (lambda: tl.router_logits(1, 16, 48), "K=48"),
    (lambda: tl.router_logits(1, 16, 64, "float32"), "dtype must be"),
    (lambda: tl.route_experts(**ROUTE | {"tokens": 0}), "tokens"),
    (lambda: tl.route_experts(**ROUTE | {"experts": 1025}), "experts"),
    (lambda: tl.route_experts(**ROUTE | {"top_k": 33}), "top_k"),
    (lambda: tl.route_experts(**ROUTE | {"top_k": 17}), "top_k=17"),
    (lambda: tl.route_experts(**ROUTE | {"tokens": 2**22 + 1}), "pairs"),
    (lambda: tl.route_experts(**ROUTE, groups=3), "groups=3"),
    (lambda: tl.route_experts(**ROUTE, groups=0), "groups=0"),
    (lambda: tl.route_experts(130, 260, 2, groups=65), "groups=65"),
    (lambda: tl.route_experts(**ROUTE, groups=4, top_groups=5), "top_groups=5"),
    (lambda: tl.route_experts(**ROUTE | {"top_k": 5}, groups=4, top_groups=1), "top_k=5"),
    (lambda: tl.route_experts(**ROUTE, scores="tanh"), "scores must be"),
    (lambda: tl.route_experts(**ROUTE, group_score="min"), "group_score must be"),
    (lambda: tl.route_experts(**ROUTE, factor=math.inf), "factor must be"),
    (lambda: tl.route_experts(**ROUTE, dtype="int32"), "dtype must be"),
    (lambda: tl.experts_order(5, 2, 16, first=-1), "first=-1"),
    (lambda: tl.experts_order(5, 2, 16, first=2**31 - 16), "first="),
    (lambda: tl.experts_up(**PRODUCT | {"K": 192}), "K=192"),
    (lambda: tl.experts_up(**PRODUCT | {"K": 32}, weight_format="mxfp4"), "K=32"),
    (lambda: tl.experts_up(**PRODUCT | {"N": 48}), "N=48"),
    (lambda: tl.experts_up(**PRODUCT | {"N": 2**20, "K": 2**12}), "2\\^31 weights"),
    (lambda: tl.experts_up(**PRODUCT | {"tokens": 2**21, "K": 1024}), "2\\^30 elements"),
    (lambda: tl.experts_up(**PRODUCT, weight_format="int8"), "weight_format must be"),
    (lambda: tl.experts_up(**PRODUCT, group_size=256), "group_size=256"),
    (lambda: tl.experts_up(**PRODUCT, weight_format="mxfp4", group_size=64), "group_size=64"),
    (lambda: tl.experts_up(**PRODUCT, weight_format="mxfp4", with_zeros=True), "zero points"),
    (lambda: tl.experts_up(**PRODUCT, activation="relu"), "activation must be"),
    (lambda: tl.experts_down(**PRODUCT, first=-3), "first=-3"),
    (lambda: tl.experts_up(**PRODUCT, routed=15), "routed=15"),
    (lambda: tl.experts_down(**PRODUCT, routed=2**31), "routed="),
    (lambda: tl.experts_down(**PRODUCT | {"K": 0}), "K=0"),
])
def test_factories_refuse(make, match):
    with pytest.raises(ValueError, match=match):
        make()


def _operands(kernel, device="cpu"):
    return [torch.zeros(p.shape, dtype=p.dtype, device=device) for i, p in enumerate(kernel.params)
            if i not in kernel.result_idx and i not in kernel.workspace_idx]


@pytest.mark.parametrize("kernel", [
    tl.router_logits(3, 8, 64, with_bias=True), tl.rms_norm(3, 64), tl.rms_norm(3, 64, residual=True, int8=True), tl.route_experts(**ROUTE, bias=True), tl.route_experts(500, 16, 2), tl.experts_order(500, 2, 16),
    tl.experts_up(**PRODUCT, with_zeros=True, with_bias=True), tl.experts_down(**PRODUCT, weight_format="mxfp4", residual=True),
], ids=lambda k: k.name)
def test_kernel_objects_refuse(kernel):
    good = _operands(kernel)
    with pytest.raises(ValueError, match="device mismatch"):
        kernel(*good)
    with pytest.raises(ValueError, match="Expected .* inputs"):
        kernel(*good[:-1])


def test_view_of_wider_rows():
    """Which views a norm of a row stride takes (the look alone: no launch)."""
    p = tl.rms_norm(3, 64, row_stride=192).params[0]
    wide = torch.zeros((3, 192), dtype=torch.float16)
    assert p.lies_as(wide[:, :64]) and p.lies_as(wide[:, 128:]) and not p.lies_as(torch.zeros((3, 64), dtype=torch.float16))


def _entry(name, **changed):
    """Calls an entry point with arguments that are good but for `changed`; the pointers are never followed: the checks come first."""
    p = ctypes.c_void_p(1 << 20)
    product = dict(B=p, Scale=p, Zeros=p, Bias=p, Order=p, Starts=p)
    sizes = dict(tokens=4, experts=8, top_k=2, N=64, K=256, group_size=64, format=EXPERTS_UINT4)
    args = {
        "call_rms_norm": dict(X=p, Residual=p, Weight=p, Y=p, Sum=p, Scale=p, rows=2, dim=64, row_stride=64, int8=1, dtype=DT_F16, eps=1e-6),
        "call_router_logits": dict(X=p, W=p, Bias=None, Logits=p, tokens=2, experts=8, K=64, dtype=DT_F16),
        "call_route_experts": dict(Logits=p, Bias=p, Weights=p, Ids=p, Order=p, Starts=p, Workspace=None, bytes=0, tokens=4, experts=8, top_k=2, scores=0, groups=2,
                                   top_groups=1, group_score=1, renormalize=1, dtype=DT_F32, factor=1.0),
        "call_experts_order": dict(Ids=p, Order=p, Starts=p, Workspace=None, bytes=0, tokens=4, top_k=2, experts=8, first=0),
        "call_experts_up": dict(X=p, **product, H=p, **sizes, activation=0, routed=8),
        "call_experts_down": dict(H=p, **product, Ids=p, Weights=p, Residual=p, C=p, Workspace=p, bytes=1 << 30, **sizes, first=0, routed=8),
    }[name]
    assert set(changed) <= set(args)
    args |= changed
    if name == "call_experts_order":  # (top_k before experts there)
        args = {k: args[k] for k in ("Ids", "Order", "Starts", "Workspace", "bytes", "tokens", "top_k", "experts", "first")}
    lib = _lib.load_library()
    rc = getattr(lib, name)(*args.values(), None)
    return rc, lib.get_last_error().decode()


ODD = ctypes.c_void_p((1 << 20) + 2)


@pytest.mark.parametrize("name,changed,match", [
    ("call_rms_norm", dict(X=None), "non-NULL"),
    ("call_rms_norm", dict(Y=ODD), "16-byte"),
    ("call_rms_norm", dict(Scale=ODD), "4-byte"),
    ("call_rms_norm", dict(Sum=None), "go together"),
    ("call_rms_norm", dict(int8=0), "Scale goes with"),
    ("call_rms_norm", dict(Scale=None), "Scale goes with"),
    ("call_rms_norm", dict(rows=0), "rows must be"),
    ("call_rms_norm", dict(dim=68), "dim must be"),
    ("call_rms_norm", dict(dim=1 << 16, row_stride=1 << 16), "dim must be"),
    ("call_rms_norm", dict(row_stride=56), "row_stride must be"),
    ("call_rms_norm", dict(dtype=DT_F32), "dtype must be"),
    ("call_rms_norm", dict(eps=-1.0), "eps must be"),
    ("call_router_logits", dict(tokens=0), "tokens must be"),
    ("call_router_logits", dict(tokens=(1 << 23) + 1), "at most"),
    ("call_router_logits", dict(experts=1025), "experts must be"),
    ("call_router_logits", dict(K=0), "K must be"),
    ("call_router_logits", dict(K=40), "K must be"),
    ("call_router_logits", dict(dtype=DT_F32), "dtype must be"),
    ("call_router_logits", dict(Logits=None), "non-NULL"),
    ("call_router_logits", dict(W=ODD), "16-byte"),
    ("call_router_logits", dict(Bias=ctypes.c_void_p((1 << 20) + 1)), "2-byte"),
    ("call_route_experts", dict(tokens=0), "tokens must be"),
    ("call_route_experts", dict(tokens=1 << 30), "pairs in a call"),
    ("call_route_experts", dict(experts=2000), "experts must be"),
    ("call_route_experts", dict(top_k=0), "top_k must be"),
    ("call_route_experts", dict(top_k=5), "top_k=5"),
    ("call_route_experts", dict(groups=3), "groups must be"),
    ("call_route_experts", dict(top_groups=3), "top_groups must be"),
    ("call_route_experts", dict(scores=2), "unknown scores"),
    ("call_route_experts", dict(group_score=-1), "unknown group_score"),
    ("call_route_experts", dict(factor=math.nan), "factor must be"),
    ("call_route_experts", dict(dtype=9), "dtype must be"),
    ("call_route_experts", dict(Starts=None), "non-NULL"),
    ("call_route_experts", dict(Logits=ODD), "4-byte"),
    ("call_route_experts", dict(tokens=400), "needs a 16-byte aligned workspace"),
    ("call_experts_order", dict(first=-1), "first must be"),
    ("call_experts_order", dict(first=(1 << 31) - 8), "first must be"),
    ("call_experts_order", dict(Ids=None), "non-NULL"),
    ("call_experts_order", dict(Order=ODD), "4-byte"),
    ("call_experts_order", dict(tokens=400, bytes=8, Workspace=ctypes.c_void_p(1 << 20)), "needs a 16-byte aligned workspace"),
    ("call_experts_up", dict(format=2), "unknown weight format"),
    ("call_experts_up", dict(K=64), "K must be"),
    ("call_experts_up", dict(N=40), "N must be"),
    ("call_experts_up", dict(group_size=16), "group_size must be"),
    ("call_experts_up", dict(format=EXPERTS_MXFP4, group_size=32), "no zero points"),
    ("call_experts_up", dict(N=1 << 20, K=1 << 12), "2^31 weights"),
    ("call_experts_up", dict(tokens=1 << 22, K=512), "2^30 elements"),
    ("call_experts_up", dict(H=None), "non-NULL"),
    ("call_experts_up", dict(B=ODD), "16-byte"),
    ("call_experts_up", dict(Bias=ODD), "16-byte"),
    ("call_experts_up", dict(Order=ctypes.c_void_p((1 << 20) + 1)), "4-byte"),
    ("call_experts_up", dict(activation=2), "unknown activation"),
    ("call_experts_up", dict(routed=7), "routed must be"),
    ("call_experts_down", dict(routed=0), "routed must be"),
    ("call_experts_down", dict(Weights=None), "non-NULL"),
    ("call_experts_down", dict(Residual=ODD), "16-byte"),
    ("call_experts_down", dict(first=-1), "first must be"),
    ("call_experts_down", dict(tokens=400, bytes=100), "needs a 16-byte aligned workspace"),
    ("call_experts_down", dict(tokens=400, Workspace=None), "needs a 16-byte aligned workspace"),
])
def test_entry_points_refuse(name, changed, match):
    rc, message = _entry(name, **changed)
    assert rc == -1 and match in message and message.startswith(name), message


def test_workspaces_are_named_without_a_gpu():
    lib = _lib.load_library()
    order, down = lib.dq_experts_order_workspace_bytes, lib.dq_experts_down_workspace_bytes
    assert order(1, 8, 128) == order(32, 8, 128) == order(64, 1, 8) == 0  # one workgroup has them all
    assert order(65, 1, 8) >= 5 * 8 * 2 and order(2**18, 32, 1024) <= 256 * 1024 * 2
    assert order(0, 8, 128) == order(2**30, 8, 128) == order(-1, 8, 128) == 0
    # a value a pair, and slices of K where there are few tiles
    assert down(4096, 8, 2, 4096, 14336, 128, EXPERTS_UINT4, 8) == 4096 * 2 * 4096 * 4
    assert down(64, 8, 2, 4096, 14336, 128, EXPERTS_UINT4, 8) in (2 * 64 * 2 * 4096 * 4, 4 * 64 * 2 * 4096 * 4)
    assert down(0, 8, 2, 64, 256, 128, EXPERTS_UINT4, 8) == 0 and down(2**30, 8, 2, 64, 256, 32, EXPERTS_MXFP4, 8) == 0
    assert down(64, 8, 2, 4096, 14336, 128, EXPERTS_UINT4, 64) == 64 * 2 * 4096 * 4  # (two rows an expert: no tiles)


def test_results_of_a_kernel_object():
    """Which parameters come back, in their order."""
    names = lambda k: [k.params[i].name for i in k.result_idx]
    assert names(tl.rms_norm(2, 64)) == ["y"] and names(tl.rms_norm(2, 64, residual=True)) == ["y", "sum"]
    assert names(tl.rms_norm(2, 64, int8=True, residual=True)) == ["codes", "scale", "sum"]
    assert names(tl.route_experts(500, 16, 2)) == ["weights", "ids", "order", "starts"] and names(tl.experts_order(500, 2, 16)) == ["order", "starts"]
    assert names(tl.experts_up(**PRODUCT)) == ["h"] and names(tl.experts_down(**PRODUCT)) == ["y"]
