"""Kernel factories of the rest of a decoder block around 4-bit weights: the norm, the routing of tokens to experts, and the
experts' products.

As in :mod:`kernels`, a factory takes sizes and types and returns a :class:`~tilelang_amd.adapter.KernelAdapter` bound to an
entry point of ``libdqgemm.so`` (``include/dqgemm.h``); its call checks every operand and launches on torch's current stream.

A layer of experts is four calls: ``logits = router_logits(...)(x, W)``; ``weights, ids, order, starts = route_experts(...)(logits)`` chooses
the experts of every token and sorts the pairs (token, choice) by expert; ``h = experts_up(...)(x, ..., order, starts)`` has a row for
every pair in that order, and ``y = experts_down(...)(h, ..., order, starts, ids, weights)`` one for every token again.
"""

from __future__ import annotations

import math

import torch

from . import _lib
from .adapter import KernelAdapter, KernelParam
from .kernels import _dtype
from .kv_kernels import DT_BF16, DT_F16, _kernel, _positive, _type16

DT_F32 = 3
SCORES = {"softmax": 0, "sigmoid": 1}
GROUP_SCORES = {"max": 0, "sum2": 1}
ACTIVATIONS = {"silu": 0, "gelu": 1}
EXPERTS_UINT4, EXPERTS_MXFP4 = 0, 1

MAX_NORM_DIM, MAX_EXPERTS, MAX_TOP_K, MAX_GROUPS = 32768, 1024, 32, 64
#: (token, choice) pairs that a call takes
MAX_PAIRS = 2**23
#: elements of the tokens' rows
MAX_ELEMENTS = 2**30


def _one_of(fn: str, name: str, value, values: dict) -> int:
    if value not in values:
        raise ValueError(f"{fn}: {name} must be one of {tuple(values)} (got {value!r})")
    return values[value]


def _first(fn: str, first: int, experts: int) -> None:
    if not 0 <= first <= 2**31 - 1 - experts:
        raise ValueError(f"{fn}: first={first} must be from 0 to 2^31 - 1 - experts={experts}")


def rms_norm(rows: int, dim: int, eps: float = 1e-6, dtype="float16", residual: bool = False, int8: bool = False,
             row_stride: int | None = None) -> KernelAdapter:
    """Root-mean-square norm: ``y = kernel(x, Weight)``, ``y = Weight * x / sqrt(mean(x ** 2) + eps)`` over rows ``[rows, dim]``.

    ``residual``: ``y, sum = kernel(x, Residual, Weight)`` is the norm of ``x + Residual``, which comes back as ``sum``, rounded (the
    norm is of the sum before that).  ``int8``: instead of ``y`` come its codes and their scales, ``codes, scale[, sum] = kernel(...)``:
    ``scale = 127 / max(max|y|, 1e-5)`` fp32 ``[rows]``, ``codes = round(y * scale)`` int8, what :func:`bitlinear_int8xint2` takes; a row
    with an infinity or a NaN gives zeros and a scale that is NaN.  ``row_stride``: elements from one row of ``x`` to the next where
    it is a view of wider rows.  ``dim`` is a multiple of 8, at most 32768.  Sums are fp32.
    """
    fn = "rms_norm"
    _positive(fn, rows=rows)
    if dim <= 0 or dim % 8 or dim > MAX_NORM_DIM:
        raise ValueError(f"{fn}: dim={dim} must be a multiple of 8, at most {MAX_NORM_DIM}")
    t = _type16(fn, dtype)
    stride = dim if row_stride is None else row_stride
    if stride < dim or stride % 8 or stride > 2**31 - 8:
        raise ValueError(f"{fn}: row_stride={stride} must be a multiple of 8 and at least dim={dim}, below 2^31")
    if rows >= 2**31:
        raise ValueError(f"{fn}: rows={rows} must be below 2^31")
    eps = float(eps)
    if not (eps > 0 and math.isfinite(eps)):
        raise ValueError(f"{fn}: eps must be positive and finite (got {eps})")
    params = [KernelParam("x", t, (rows, dim), strides=None if stride == dim else (stride, 1))]
    if residual:
        params.append(KernelParam("Residual", t, (rows, dim)))
    params.append(KernelParam("Weight", t, (dim,)))
    first = len(params)
    params.append(KernelParam("codes", torch.int8, (rows, dim)) if int8 else KernelParam("y", t, (rows, dim)))
    if int8:
        params.append(KernelParam("scale", torch.float32, (rows,)))
    if residual:
        params.append(KernelParam("sum", t, (rows, dim)))
    results = list(range(first, len(params)))
    slots = (0, 1 if residual else None, first - 1, first, results[-1] if residual else None, first + 1 if int8 else None)
    return _kernel(fn, "call_rms_norm", params, results, slots, (rows, dim, stride, int(int8), DT_BF16 if t == torch.bfloat16 else DT_F16), eps)


def _pairs(fn: str, tokens: int, experts: int, top_k: int) -> None:
    _positive(fn, tokens=tokens, experts=experts, top_k=top_k)
    if experts > MAX_EXPERTS or top_k > MAX_TOP_K:
        raise ValueError(f"{fn}: at most {MAX_EXPERTS} experts and top_k={MAX_TOP_K} (got {experts} and {top_k})")
    if tokens * top_k > MAX_PAIRS:
        raise ValueError(f"{fn}: {top_k} choices of {tokens} tokens: at most {MAX_PAIRS} pairs in a call")


def router_logits(tokens: int, experts: int, K: int, dtype="float16", with_bias: bool = False) -> KernelAdapter:
    """A router's logits: ``logits = kernel(x, W[, Bias])`` fp32 ``[tokens, experts]`` ``= x @ W.T (+ Bias)`` for ``x`` ``[tokens, K]``, ``W`` ``[experts, K]``
    and ``Bias`` ``[experts]`` in fp16 or bf16; sums are fp32, ``K`` is a multiple of 32."""
    fn = "router_logits"
    _pairs(fn, tokens, experts, 1)
    if K <= 0 or K % 32:
        raise ValueError(f"{fn}: K={K} must be a positive multiple of 32")
    held = _type16(fn, dtype)
    params = [KernelParam("x", held, (tokens, K)), KernelParam("W", held, (experts, K))]
    if with_bias:
        params.append(KernelParam("Bias", held, (experts,)))
    out = len(params)
    params.append(KernelParam("logits", torch.float32, (tokens, experts)))
    return _kernel(fn, "call_router_logits", params, [out], (0, 1, 2 if with_bias else None, out), (tokens, experts, K, DT_BF16 if held == torch.bfloat16 else DT_F16))


def route_experts(tokens: int, experts: int, top_k: int, scores: str = "softmax", bias: bool = False, groups: int = 1, top_groups: int | None = None,
                  group_score: str = "max", renormalize: bool = True, factor: float = 1.0, dtype="float32") -> KernelAdapter:
    """Which experts a token goes to: ``weights, ids, order, starts = kernel(logits[, Bias])``, ``logits`` ``[tokens, experts]`` of ``dtype``
    (float32, float16 or bfloat16).

    A score is the ``"softmax"`` over a token's logits, or the ``"sigmoid"`` of each.  ``ids`` int32 ``[tokens, top_k]`` are the experts with
    the largest keys, the best first, of equal ones the lowest index first; a key is the score plus ``Bias`` fp32 ``[experts]``
    (``bias``; it balances the experts' load and is no part of the weights), or else the logit.  ``groups``: the experts are that many
    groups of neighbours, and only the ``top_groups`` best of them count, by the largest key of each (``group_score="max"``) or the
    sum of its two largest (``"sum2"``; without a bias: of scores).  ``weights`` fp32 ``[tokens, top_k]`` are the chosen scores, divided
    by their sum (``renormalize``), times ``factor``.  A logit of -inf has a score of 0 and without a bias is chosen last; with one its key is
    its bias, and a bias of -inf is chosen last.  A NaN is chosen first and shows in the weights.
    Choices do not depend on how an exponential is rounded: where 32 bits cannot tell two scores apart, 64 do.

    ``order`` and ``starts`` are :func:`experts_order`'s of the same ids.
    """
    fn = "route_experts"
    _pairs(fn, tokens, experts, top_k)
    t = _dtype(dtype)
    if t not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError(f"{fn}: dtype must be float32, float16 or bfloat16 (got {dtype!r})")
    score, two = _one_of(fn, "scores", scores, SCORES), _one_of(fn, "group_score", group_score, GROUP_SCORES)
    if groups <= 0 or groups > MAX_GROUPS or experts % groups:
        raise ValueError(f"{fn}: groups={groups} must be from 1 to {MAX_GROUPS} and divide experts={experts}")
    top_groups = groups if top_groups is None else top_groups
    if not 1 <= top_groups <= groups:
        raise ValueError(f"{fn}: top_groups={top_groups} must be from 1 to groups={groups}")
    if top_k > top_groups * (experts // groups):
        raise ValueError(f"{fn}: top_k={top_k} choices of the {top_groups * (experts // groups)} experts of {top_groups} groups")
    factor = float(factor)
    if not math.isfinite(factor):
        raise ValueError(f"{fn}: factor must be finite")
    params = [KernelParam("logits", t, (tokens, experts))]
    if bias:
        params.append(KernelParam("Bias", torch.float32, (experts,)))
    first = len(params)
    params += [KernelParam("weights", torch.float32, (tokens, top_k)), KernelParam("ids", torch.int32, (tokens, top_k)),
               KernelParam("order", torch.int32, (tokens * top_k,)), KernelParam("starts", torch.int32, (experts + 1,))]
    room = int(_lib.load_library().dq_experts_order_workspace_bytes(tokens, top_k, experts))
    if room:
        params.append(KernelParam("Workspace", torch.uint8, (room,)))
    slots = (0, 1 if bias else None, first, first + 1, first + 2, first + 3, first + 4 if room else None)
    ints = (tokens, experts, top_k, score, groups, top_groups, two, int(renormalize), {torch.float16: DT_F16, torch.bfloat16: DT_BF16}.get(t, DT_F32))
    return _kernel(fn, "call_route_experts", params, list(range(first, first + 4)), slots, ints, factor, room, [first + 4] if room else [])


def experts_order(tokens: int, top_k: int, experts: int, first: int = 0) -> KernelAdapter:
    """The pairs of ``ids`` sorted by expert: ``order, starts = kernel(ids)``, ``ids`` int32 ``[tokens, top_k]``.

    ``order`` int32 ``[tokens * top_k]`` names pairs, ``token * top_k + choice``: those of expert ``first + e`` stand at ``starts[e] ..
    starts[e + 1] - 1`` (``starts`` int32 ``[experts + 1]``), in ascending order.  Pairs of other ids (experts that another GPU has; -1:
    no token, in a padded batch) are in none, and the places behind ``starts[experts]`` hold -1.
    """
    fn = "experts_order"
    _pairs(fn, tokens, experts, top_k)
    _first(fn, first, experts)
    params = [KernelParam("ids", torch.int32, (tokens, top_k)), KernelParam("order", torch.int32, (tokens * top_k,)),
              KernelParam("starts", torch.int32, (experts + 1,))]
    room = int(_lib.load_library().dq_experts_order_workspace_bytes(tokens, top_k, experts))
    if room:
        params.append(KernelParam("Workspace", torch.uint8, (room,)))
    return _kernel(fn, "call_experts_order", params, [1, 2], (0, 1, 2, 3 if room else None), (tokens, top_k, experts, first), None, room, [3] if room else [])


class _Weights:
    """The experts' weights as an operand: parameters, and what the entry points are told about them."""

    def __init__(self, fn, experts, rows, N, K, weight_format, group_size, with_zeros, with_bias):
        if weight_format not in ("uint4", "mxfp4"):
            raise ValueError(f"{fn}: weight_format must be 'uint4' or 'mxfp4' (got {weight_format!r})")
        mx = weight_format == "mxfp4"
        self.dtype = torch.bfloat16 if mx else torch.float16
        group_size = (32 if mx else 128) if group_size is None else group_size
        if group_size not in ((32,) if mx else (32, 64, 128)):
            raise ValueError(f"{fn}: group_size={group_size} must be {'32 with mxfp4' if mx else '32, 64 or 128'}")
        if mx and with_zeros:
            raise ValueError(f"{fn}: mxfp4 weights have no zero points")
        unit = 64 if mx else 128
        if K <= 0 or K % unit:
            raise ValueError(f"{fn}: K={K} must be a positive multiple of {unit}")
        if N <= 0 or N % 32:
            raise ValueError(f"{fn}: N={N} must be a positive multiple of 32")
        if N * K > 2**31:
            raise ValueError(f"{fn}: N={N}, K={K}: at most 2^31 weights an expert and projection")
        groups = (experts, rows, K // group_size)
        self.params = [KernelParam("B", torch.uint8 if mx else torch.int8, (experts, rows, K // 2), packed=True),
                       KernelParam("Scale", torch.uint8 if mx else torch.float16, groups, packed=mx)]
        self.zeros = self.bias = None
        if with_zeros:
            self.zeros = len(self.params)
            self.params.append(KernelParam("Zeros", torch.float16, groups))
        if with_bias:
            self.bias = len(self.params)
            self.params.append(KernelParam("Bias", self.dtype, (experts, rows)))
        self.ints = (group_size, EXPERTS_MXFP4 if mx else EXPERTS_UINT4)

    def slots(self, first: int) -> tuple:
        """The four pointer arguments of the weights, whose parameters begin at ``first``."""
        return (first, first + 1, None if self.zeros is None else first + self.zeros, None if self.bias is None else first + self.bias)


def _routed(fn: str, routed: int | None, experts: int) -> int:
    routed = experts if routed is None else routed
    if not experts <= routed < 2**31:
        raise ValueError(f"{fn}: routed={routed} must be at least experts={experts}")
    return routed


def _activations(fn: str, rows: int, width: int) -> None:
    if rows * width > MAX_ELEMENTS:
        raise ValueError(f"{fn}: {rows} tokens of {width} elements: at most 2^30 elements")


def experts_up(tokens: int, experts: int, top_k: int, N: int, K: int, weight_format: str = "uint4", group_size: int | None = None,
               with_zeros: bool = False, activation: str = "silu", with_bias: bool = False, routed: int | None = None) -> KernelAdapter:
    """The experts' gate and up projections: ``h = kernel(x, B, Scale[, Zeros][, Bias], order, starts)``, ``x`` ``[tokens, K]``, ``h`` ``[tokens *
    top_k, N]``: row ``p`` is ``act(x[t] @ gate.T + gate_bias) * (x[t] @ up.T + up_bias)`` for token ``t = order[p] // top_k`` and the expert
    whose rows are about ``p``.  Rows behind ``starts[experts]`` are not written.

    ``B`` ``[experts, 2 N, K / 2]``: an expert's gate rows, then its up rows, ``Bias`` ``[experts, 2 N]``.  ``weight_format``: ``"uint4"``, fp16
    activations and the weights of :func:`dequantize_gemv` with ``source_format="int"`` (``Scale`` fp16 ``[experts, 2 N, K / group_size]``,
    groups of 32, 64 or 128) or, ``with_zeros``, ``"uint"`` codes with fp16 zero points; or ``"mxfp4"``, bf16 activations and the weights of
    :func:`matmul_bf16_mxfp4` with ``weight_format="e2m1"`` and ``scale_bias=127``.  ``activation``: ``"silu"`` or ``"gelu"`` (the tanh form).
    ``K`` is a multiple of 128 (mxfp4: 64), ``N`` of 32.  Sums are fp32.  ``routed``: of how many experts the ids are, where these are some of
    them: which kernel is taken goes by it, and nothing else.
    """
    fn = "experts_up"
    _pairs(fn, tokens, experts, top_k)
    w = _Weights(fn, experts, 2 * N, N, K, weight_format, group_size, with_zeros, with_bias)
    act = _one_of(fn, "activation", activation, ACTIVATIONS)
    routed = _routed(fn, routed, experts)
    _activations(fn, tokens, K)
    params = [KernelParam("x", w.dtype, (tokens, K)), *w.params]
    n = len(params)
    params += [KernelParam("order", torch.int32, (tokens * top_k,)), KernelParam("starts", torch.int32, (experts + 1,)),
               KernelParam("h", w.dtype, (tokens * top_k, N))]
    return _kernel(fn, "call_experts_up", params, [n + 2], (0, *w.slots(1), n, n + 1, n + 2), (tokens, experts, top_k, N, K, *w.ints, act, routed))


def experts_down(tokens: int, experts: int, top_k: int, N: int, K: int, weight_format: str = "uint4", group_size: int | None = None,
                 with_zeros: bool = False, with_bias: bool = False, residual: bool = False, first: int = 0, routed: int | None = None) -> KernelAdapter:
    """The way back from the experts: ``y = kernel(h, B, Scale[, Zeros][, Bias], order, starts, ids, weights[, Residual])``, ``h`` ``[tokens *
    top_k, K]`` in the sorted order, ``y`` ``[tokens, N]``: a token's choices, each ``h[p] @ down.T + bias`` times its weight, added in their
    order, onto ``Residual`` ``[tokens, N]`` (``residual``).

    ``B`` ``[experts, N, K / 2]``, ``Bias`` ``[experts, N]``, formats as for :func:`experts_up`.  ``first``: the id of the first of these experts,
    as for :func:`experts_order`, ``routed`` as for :func:`experts_up`; choices of other ids add nothing.  Sums are fp32; a call gives the same bits every time.
    """
    fn = "experts_down"
    _pairs(fn, tokens, experts, top_k)
    w = _Weights(fn, experts, N, N, K, weight_format, group_size, with_zeros, with_bias)
    _first(fn, first, experts)
    routed = _routed(fn, routed, experts)
    _activations(fn, tokens, K)
    if min(tokens * top_k, 128) * K > 2**31:
        raise ValueError(f"{fn}: K={K}: at most 2^31 elements of 128 rows of h, or of all where they are fewer")
    params = [KernelParam("h", w.dtype, (tokens * top_k, K)), *w.params]
    n = len(params)
    params += [KernelParam("order", torch.int32, (tokens * top_k,)), KernelParam("starts", torch.int32, (experts + 1,)),
               KernelParam("ids", torch.int32, (tokens, top_k)), KernelParam("weights", torch.float32, (tokens, top_k))]
    if residual:
        params.append(KernelParam("Residual", w.dtype, (tokens, N)))
    out = len(params)
    params.append(KernelParam("y", w.dtype, (tokens, N)))
    room = int(_lib.load_library().dq_experts_down_workspace_bytes(tokens, experts, top_k, N, K, *w.ints, routed))
    if room:
        params.append(KernelParam("Workspace", torch.uint8, (room,)))
    slots = (0, *w.slots(1), n, n + 1, n + 2, n + 3, n + 4 if residual else None, out, out + 1 if room else None)
    return _kernel(fn, "call_experts_down", params, [out], slots, (tokens, experts, top_k, N, K, *w.ints, first, routed), None, room, [out + 1] if room else [])
