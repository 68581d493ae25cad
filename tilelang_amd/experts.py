"""The norms and the experts of a decoder block on the kernels: :class:`RMSNorm` in front of a projection, and :class:`W4Experts` in
place of the block's other half, next to :class:`~tilelang_amd.attention.W4Attention`.

A block is ``h, x = norm1(a, x)``, ``a = attention(h, cache, rows)``, ``h, x = norm2(a, x)``, ``a = experts(h)``: what a half gives is added
to the residual in the next norm's launch.
"""

from __future__ import annotations

import torch
from torch import nn

from . import block_kernels, kernels, quantize
from .adapter import kept
from .w4linear import quantize_w4

#: kernel objects (sets of them) that a layer keeps: prompts come in any number of rows
MAX_KERNELS = 64
#: tokens that go through the experts at once, and bytes of the rows between the two products and of "down"'s workspace that these take
#: at most; more go in parts
MAX_TOKENS = 65536
PART_BYTES = 2**33
#: from this many logits on the tiled GEMM is ahead (4096 tokens, 256 experts, 7168 wide 57 us and 77; 16384, 32 of 2880 25 and 21)
TILED_LOGITS = 2**20


def _kept(held: dict, key, make):
    return kept(held, key, make, MAX_KERNELS)


def _whole(t: torch.Tensor) -> torch.Tensor:
    """``t``, or a copy of it, contiguous and from a multiple of 16 bytes on, as the kernels take it."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _check_rows(fn: str, name: str, t: torch.Tensor, x: torch.Tensor, width: int) -> None:
    """That ``t`` has a row of ``width`` for each of ``x``'s: the same leading sizes, or one of the two flat."""
    if t.shape[:-1] == x.shape[:-1] and t.shape[-1] == width:
        return
    flat = (t.dim() == 2 or x.dim() == 2) and t.shape[-1:] == (width,) and t.shape[:-1].numel() == x.shape[:-1].numel()
    if not flat:
        raise ValueError(f"{fn}: {name} is {tuple(t.shape)}, not a row of {width} for each of x, {tuple(x.shape)}")


class RMSNorm(nn.Module):
    """``weight * x / sqrt(mean(x ** 2) + eps)`` over rows of fp16 or bf16.

    ``norm(x)`` is ``y``; ``norm(x, residual)`` is ``(y, x + residual)``, the norm that of the sum before it is rounded.  ``int8``: in place of ``y``
    come ``(codes, scale)``, which :class:`~tilelang_amd.bitlinear.BitLinear` takes: ``norm(x)`` is ``(codes, scale)``, ``norm(x, residual)``
    ``(codes, scale, x + residual)``.  Rows of ``x`` may lie apart (a slice of a wider projection's columns).  ``residual`` has ``x``'s shape, or one
    of them is flat, a row a token.  A batch of no tokens has results of no rows.
    """

    def __init__(self, dim: int, eps: float = 1e-6, dtype=torch.float16, int8: bool = False):
        super().__init__()
        block_kernels.rms_norm(1, dim, eps, dtype, int8=int8)  # (says what is wrong with these now)
        self.dim, self.eps, self.int8 = dim, eps, int8
        self.register_buffer("weight", torch.ones((dim,), dtype=kernels._dtype(dtype)))
        self._kernels: dict = {}

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        lead, dtype = x.shape[:-1], self.weight.dtype
        if residual is not None and residual.shape != x.shape:
            _check_rows("RMSNorm", "residual", residual, x, self.dim)
        rows = x if x.dim() == 2 else x.reshape(lead.numel(), x.shape[-1])
        if rows.dtype != dtype:
            rows = rows.to(dtype)
        stride = rows.stride(0) if rows.shape[0] > 1 else self.dim
        if rows.stride(1) != 1 or not self.dim <= stride < 2**31 or stride % 8 or rows.data_ptr() % 16:
            rows, stride = _whole(rows), self.dim
        n = rows.shape[0]
        if n == 0 and rows.shape[1] == self.dim:  # (a batch of no tokens: nothing to launch)
            out = [rows.new_empty(x.shape, dtype=torch.int8), rows.new_empty(lead, dtype=torch.float32)] if self.int8 else [rows.new_empty(x.shape)]
            out += [] if residual is None else [rows.new_empty(x.shape)]
            return out[0] if len(out) == 1 else tuple(out)
        kern = _kept(self._kernels, (n, stride, residual is not None, dtype),
                     lambda: block_kernels.rms_norm(n, self.dim, self.eps, dtype, residual is not None, self.int8, stride))
        if residual is None:
            out = kern(rows, self.weight)
        else:
            out = kern(rows, _whole(residual.to(dtype).reshape(-1, self.dim)), self.weight)
        out = list(out) if isinstance(out, (list, tuple)) else [out]
        if len(lead) != 1:
            out = [t.view(lead if t.dim() == 1 else (*lead, self.dim)) for t in out]
        return out[0] if len(out) == 1 else tuple(out)


def quantize_mxfp4(weight: torch.Tensor):
    """``weight[N, K]`` -> ``(codes [N, K / 2] uint8, scale [N, K / 32] uint8)``, as :func:`~tilelang_amd.quantize_bf16_mxfp4` has them with
    ``scale_bias=127``, on any device."""
    N, K = weight.shape
    if K % 32:
        raise ValueError(f"quantize_mxfp4: K={K} is not a multiple of 32")
    w = weight.to(torch.bfloat16).float().reshape(N, K // 32, 32)
    most = w.abs().amax(dim=2)
    e = torch.where(most > 0, torch.frexp(most).exponent - 3, -127).clamp(-127, 128)
    codes = quantize.encode_fp4_e2m1_values(torch.ldexp(w, -e[..., None]).reshape(N, K))
    return quantize.pack_fp4_e2m1_codes(codes).view(torch.uint8), (e + 127).to(torch.uint8)


class W4Experts(nn.Module):
    """Experts around 4-bit weights with their router: every token's ``top_k`` best of ``experts``, each ``down(act(gate(x)) * up(x))``, added
    with the router's weights.

    ``hidden`` and ``width`` are the sizes outside and inside of an expert.  ``weight_format``, ``group_size``, ``with_zeros``, ``activation`` and
    ``bias`` are as for :func:`experts_up`; the logits are ``x @ router.T``, with ``router_bias`` ``+ router_bias``; ``scores``, ``score_bias``, ``groups``, ``top_groups``, ``group_score``, ``renormalize`` and ``factor`` as for
    :func:`route_experts`.  Activations are fp16 with ``"uint4"`` weights, bf16 with ``"mxfp4"``; logits are fp32.

    ``first`` and ``held``: this layer has only the experts from ``first`` on, ``held`` of them (a rank of several that share a layer): its output
    is their part of the sum, and the parts of all ranks are to be added.
    """

    def __init__(self, hidden: int, width: int, experts: int, top_k: int, weight_format: str = "uint4", group_size: int | None = None,
                 with_zeros: bool = False, activation: str = "silu", bias: bool = False, scores: str = "softmax", router_bias: bool = False, score_bias: bool = False,
                 groups: int = 1, top_groups: int | None = None, group_score: str = "max", renormalize: bool = True, factor: float = 1.0,
                 first: int = 0, held: int | None = None):
        super().__init__()
        self.hidden, self.width, self.experts, self.top_k = hidden, width, experts, top_k
        held = experts - first if held is None else held
        if not (0 <= first and 0 < held and first + held <= experts):
            raise ValueError(f"W4Experts: experts from {first} on, {held} of them, are not among {experts}")
        self.first, self.held = first, held
        mx = weight_format == "mxfp4"
        self.group_size = (32 if mx else 128) if group_size is None else group_size
        self._format = dict(weight_format=weight_format, group_size=self.group_size, with_zeros=with_zeros)
        self._activation, self._bias, self._router_bias = activation, bias, router_bias
        self._routing = dict(scores=scores, bias=score_bias, groups=groups, top_groups=top_groups, group_score=group_score, renormalize=renormalize,
                             factor=factor)
        self._kernels: dict = {}
        self._make(1)  # (says what is wrong with these now)
        dtype = torch.bfloat16 if mx else torch.float16

        def packed(name, rows, k):
            self.register_buffer(name, torch.zeros((held, rows, k // 2), dtype=torch.uint8 if mx else torch.int8))
            scale = (held, rows, k // self.group_size)
            self.register_buffer(name + "_scale", torch.full(scale, 127, dtype=torch.uint8) if mx else torch.ones(scale, dtype=dtype))
            self.register_buffer(name + "_zeros", torch.full(scale, 8.0, dtype=dtype) if with_zeros else None)
            self.register_buffer(name + "_bias", torch.zeros((held, rows), dtype=dtype) if bias else None)

        self.register_buffer("router", torch.zeros((experts, hidden), dtype=dtype))
        self.register_buffer("router_bias", torch.zeros((experts,), dtype=dtype) if router_bias else None)
        self.register_buffer("score_bias", torch.zeros((experts,), dtype=torch.float32) if score_bias else None)
        packed("up", 2 * width, hidden)
        packed("down", hidden, width)

    def _apply(self, fn, *args, **kwargs):
        # (the kernels read it in fp32 whatever type a model is turned into: it is moved, not converted)
        kept = self._buffers["score_bias"]
        super()._apply(fn, *args, **kwargs)
        if kept is not None and self._buffers["score_bias"].dtype != torch.float32:
            self._buffers["score_bias"] = kept.to(self._buffers["score_bias"].device)
        return self

    def load_float_weight(self, expert: int, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor, gate_bias: torch.Tensor | None = None,
                          up_bias: torch.Tensor | None = None, down_bias: torch.Tensor | None = None) -> None:
        """One expert's weights, quantised: ``gate`` and ``up`` ``[width, hidden]``, ``down`` ``[hidden, width]``; ``expert`` counts from ``first``."""
        if not 0 <= expert < self.held:
            raise ValueError(f"load_float_weight: expert {expert} of {self.held}")
        for name, w, shape in (("gate", gate, (self.width, self.hidden)), ("up", up, (self.width, self.hidden)), ("down", down, (self.hidden, self.width))):
            if tuple(w.shape) != shape:
                raise ValueError(f"load_float_weight: {name} is {tuple(w.shape)}, not {shape}")
        if not self._bias and not (gate_bias is None and up_bias is None and down_bias is None):
            raise ValueError("load_float_weight: a layer without bias")
        both = None
        if self._bias:
            none = torch.zeros(self.width)
            both = torch.cat([none if b is None else b.detach().cpu().float() for b in (gate_bias, up_bias)])
        for name, w, b in (("up", torch.cat([gate.detach().cpu(), up.detach().cpu()]), both), ("down", down.detach().cpu(), down_bias)):
            if self._format["weight_format"] == "mxfp4":
                codes, scale = quantize_mxfp4(w)
                zeros = None
            else:
                codes, scale, zeros = quantize_w4(w, self.group_size, self._format["with_zeros"])
                codes = quantize.general_compress(codes.to(torch.int8), 4)
            for key, value in ((name, codes), (name + "_scale", scale), (name + "_zeros", zeros), (name + "_bias", b)):
                if self._buffers[key] is not None:
                    self._buffers[key][expert].copy_(value if value is not None else torch.zeros(()))

    def _make(self, tokens: int):
        """The kernel objects of a number of tokens: logits, choices, the order of this layer's experts where that is another, both products."""
        sizes = (tokens, self.held, self.top_k)
        dtype = "bfloat16" if self._format["weight_format"] == "mxfp4" else "float16"
        if tokens * self.experts < TILED_LOGITS or self._router_bias:
            logits = block_kernels.router_logits(tokens, self.experts, self.hidden, dtype, self._router_bias)
        else:
            logits = kernels.matmul(tokens, self.experts, self.hidden, in_dtype=dtype, out_dtype="float32")
        return (logits,
                block_kernels.route_experts(tokens, self.experts, self.top_k, **self._routing),
                None if self.held == self.experts else block_kernels.experts_order(tokens, self.top_k, self.held, self.first),
                block_kernels.experts_up(*sizes, self.width, self.hidden, activation=self._activation, with_bias=self._bias, routed=self.experts,
                                         **self._format),
                *(block_kernels.experts_down(*sizes, self.hidden, self.width, with_bias=self._bias, residual=residual, first=self.first, routed=self.experts,
                                             **self._format)
                  for residual in (False, True)))

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None, logits: torch.Tensor | None = None) -> torch.Tensor:
        """``x`` ``[..., hidden]`` -> the same; ``residual`` of that shape is added in the same launch.  ``logits`` fp32 ``[..., experts]``: in place of
        the router's.  (Either may be flat, a row a token.)  A batch of no tokens has a result of no rows."""
        dtype = self.router.dtype
        if x.shape[-1] != self.hidden:
            _check_rows("W4Experts", "x", x, x, self.hidden)
        if residual is not None and residual.shape != x.shape:
            _check_rows("W4Experts", "residual", residual, x, self.hidden)
        if logits is not None:
            _check_rows("W4Experts", "logits", logits, x, self.experts)
        if x.numel() == 0:  # (a batch of no tokens: nothing to launch)
            return x.new_empty(x.shape, dtype=dtype)
        rows = _whole(x.to(dtype).reshape(-1, self.hidden))
        r = None if residual is None else _whole(residual.to(dtype).reshape(-1, self.hidden))
        given = None if logits is None else _whole(logits.float().reshape(-1, self.experts))
        # (a pair's row of h, and its product in fp32: slices of K, which have one each, are only where there are few pairs)
        pair = 2 * self.width + 4 * self.hidden
        n, most = rows.shape[0], max(1, min(MAX_TOKENS, block_kernels.MAX_ELEMENTS // max(self.hidden, self.width), PART_BYTES // (self.top_k * pair)))
        if n <= most:
            out = self._pass(rows, r, given)
        else:
            out = torch.cat([self._pass(*(None if t is None else t[at : at + most] for t in (rows, r, given))) for at in range(0, n, most)])
        return out.view(x.shape)

    def _pass(self, x, residual, logits):
        product, route, sort, up, down, down_onto = _kept(self._kernels, x.shape[0], lambda: self._make(x.shape[0]))
        if logits is None:
            logits = product(x, self.router, *(() if self.router_bias is None else (self.router_bias,)))
        weights, ids, order, starts = route(logits) if self.score_bias is None else route(logits, self.score_bias)
        if sort is not None:
            order, starts = sort(ids)

        def held(name):
            return [b for part in ("", "_scale", "_zeros", "_bias") if (b := self._buffers[name + part]) is not None]

        h = up(x, *held("up"), order, starts)
        onto = () if residual is None else (residual,)
        return (down if residual is None else down_onto)(h, *held("down"), order, starts, ids, weights, *onto)
