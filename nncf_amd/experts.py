"""Mixture-of-experts layers on compressed expert stacks: tokens are routed to their experts, the experts' products run
grouped by expert on the packed weights, and a token's answers are summed by their weights.

`nncf.compress_weights` lowers an expert stack [experts, out, in] like any other weight (3-D weights:
src/nncf/quantization/algorithms/weight_compression/weight_lowering.py:57-81 along the last axis); `compress_experts` does that
for the two stacks of a gated expert layer and returns the module that answers with them.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from nncf_amd import _lib
from nncf_amd import decompressors as dcmp
from nncf_amd.errors import InternalError
from nncf_amd.linear import (_DTYPES, PackedWeight, activation_grad, activation_of, grad_input, packed_weight, ptr, refuse_transforms,
                             rows_of, workspace_bytes, workspace_of)
from nncf_amd.parameters import CompressWeightsMode, as_config


class ExpertRouting(NamedTuple):
    """Where the tokens of one call go.  A slot is token * top_k + place; rows are the slots in the order of their experts.

    weights   float32 [tokens, top_k]     share of each chosen expert in the token's answer (differentiable)
    experts   int32   [tokens, top_k]     the chosen experts, falling by logit; -1: the token is masked
    rows      int32   [tokens, top_k]     the row of each slot, -1: masked
    slots     int32   [tokens * top_k]    the slot of each row, -1 behind the last
    offsets   int32   [experts + 1]       expert e owns the rows [offsets[e], offsets[e + 1])
    """
    weights: torch.Tensor
    experts: torch.Tensor
    rows: torch.Tensor
    slots: torch.Tensor
    offsets: torch.Tensor


def _route(logits, top_k, renormalize, mask):
    """(weights, every integer of the routing in one tensor)."""
    tokens, experts = logits.shape
    rows, ldl = rows_of(logits, experts)
    slots = tokens * top_k
    weights = torch.empty((tokens, top_k), dtype=torch.float32, device=logits.device)
    ints = torch.empty(3 * slots + experts + 1, dtype=torch.int32, device=logits.device)
    at = ints.data_ptr()
    L = _lib.lib()
    ws = workspace_of(workspace_bytes("nncf_amd_route_experts_workspace", tokens, experts, top_k), logits.device)
    _lib.check(L.nncf_amd_route_experts(rows.data_ptr(), _lib.dtype_id(rows), ldl, tokens, experts, top_k, int(renormalize), ptr(mask),
                                        weights.data_ptr(), at, at + 4 * slots, at + 8 * slots, at + 12 * slots, ptr(ws),
                                        0 if ws is None else ws.numel(), _lib.raw_stream(logits)))
    return weights, ints


def _routing(weights, ints) -> "ExpertRouting":
    tokens, top_k = weights.shape
    s = tokens * top_k
    ids, rows, slots, offsets = ints.split((s, s, s, ints.numel() - 3 * s))
    return ExpertRouting(weights, ids.view(tokens, top_k), rows.view(tokens, top_k), slots, offsets)


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k, renormalize, mask):
        with _lib.on_device_of(logits):
            weights, ints = _route(logits, top_k, renormalize, mask)
        ctx.save_for_backward(logits, weights, ints)
        ctx.renormalize = renormalize
        ctx.mark_non_differentiable(ints)
        ctx.set_materialize_grads(False)
        return weights, ints

    @staticmethod
    @once_differentiable
    def backward(ctx, dweights, _):
        if dweights is None:
            return None, None, None, None
        refuse_transforms("route_experts", dweights)
        logits, weights, ints = ctx.saved_tensors
        tokens, experts = logits.shape
        rows, ldl = rows_of(logits, experts)
        dweights = dweights.contiguous()
        dlogits = torch.empty((tokens, experts), dtype=logits.dtype, device=logits.device)
        with _lib.on_device_of(logits):
            _lib.check(_lib.lib().nncf_amd_route_experts_grad(
                rows.data_ptr(), _lib.dtype_id(rows), ldl, tokens, experts, weights.shape[1], int(ctx.renormalize), weights.data_ptr(),
                ints.data_ptr(), dweights.data_ptr(), dlogits.data_ptr(), _lib.raw_stream(logits)))
        return dlogits, None, None, None


def route_experts(logits: torch.Tensor, top_k: int, renormalize: bool = True, token_mask: Optional[torch.Tensor] = None) -> ExpertRouting:
    """Chooses the `top_k` experts of every token and orders the (token, expert) pairs by expert.

    logits        [tokens, experts], float32, float16 or bfloat16
    renormalize   the weights are the softmax over the chosen logits (they sum to 1), else their part of the softmax over all
    token_mask    bool [tokens]: tokens with False (padding) go to no expert, their answer is zero

    Ties go to the lower expert number; a NaN logit ranks below every number; a row of -inf has weights 0.  Weights are float32
    and differentiable in `logits`."""
    what = "route_experts"
    _lib.require_gpu(logits, what)
    refuse_transforms(what, logits)
    if logits.ndim != 2 or logits.shape[1] < 1:
        raise InternalError(f"{what}: logits [tokens, experts] expected, got shape {tuple(logits.shape)}")
    if logits.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise InternalError(f"{what}: unsupported logits dtype {logits.dtype}")
    if not 1 <= top_k <= logits.shape[1]:
        raise ValueError(f"{what}: top_k = {top_k} of {logits.shape[1]} experts")
    if token_mask is not None:
        if token_mask.dtype != torch.bool or tuple(token_mask.shape) != (logits.shape[0],) or token_mask.device != logits.device:
            raise InternalError(f"{what}: token_mask is bool [{logits.shape[0]}] on {logits.device}")
        token_mask = token_mask.contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        return _routing(*_Route.apply(logits, top_k, bool(renormalize), token_mask))
    with _lib.on_device_of(logits):
        return _routing(*_route(logits, top_k, renormalize, token_mask))


def _check_routing(routing: ExpertRouting, x: torch.Tensor, what: str, experts: Optional[int] = None):
    """(tokens, top_k) of a routing whose tensors are as `route_experts` makes them."""
    if not isinstance(routing, ExpertRouting):
        raise InternalError(f"{what}: expected the ExpertRouting of route_experts, got {type(routing).__name__}")
    weights, _, rows, slots, offsets = routing
    tokens, top_k = rows.shape
    if (weights.shape != rows.shape or slots.shape != (tokens * top_k,) or offsets.ndim != 1 or weights.dtype != torch.float32
            or rows.dtype != torch.int32 or slots.dtype != torch.int32 or offsets.dtype != torch.int32
            or not (weights.is_contiguous() and rows.is_contiguous() and slots.is_contiguous() and offsets.is_contiguous())):
        raise InternalError(f"{what}: the routing's tensors are not as route_experts makes them")
    index = x.get_device()
    if rows.get_device() != index or weights.get_device() != index or slots.get_device() != index or offsets.get_device() != index:
        raise InternalError(f"{what}: the routing is on {rows.device}, the activations on {x.device}")
    if experts is not None and routing.offsets.numel() != experts + 1:
        raise InternalError(f"{what}: a routing over {routing.offsets.numel() - 1} experts for a stack of {experts}")
    return tokens, top_k


def _expert_forward(x, w: PackedWeight, slots, offsets, rows: int, top_k: int, gather: bool, act: int, width: int, want_slope: bool):
    src, ldx = rows_of(x, w.k)
    y = torch.empty((rows, width), dtype=x.dtype, device=x.device)
    slope = torch.empty((rows, w.n), dtype=torch.float32, device=x.device) if want_slope else None
    L = _lib.lib()
    ws = workspace_of(workspace_bytes("nncf_amd_expert_linear_workspace", src.data_ptr() & 15, ldx, src.shape[0], int(gather), rows,
                                      w.n, w.k, w.codes.data_ptr() & 15, w.mode, w.group_size, w.experts, act), x.device)
    _lib.check(L.nncf_amd_expert_linear(ptr(src), _DTYPES[x.dtype], ldx, src.shape[0], ptr(slots) if gather else None, top_k,
                                        ptr(offsets), w.experts, rows, w.n, w.k, ptr(w.codes), w.mode, w.group_size,
                                        ptr(w.scale), ptr(w.zero_point), act, ptr(y), width, ptr(slope), ptr(ws),
                                        0 if ws is None else ws.numel(), _lib.raw_stream(x)))
    return y, slope


class _ExpertLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, slots, offsets, places, gather, act, width):
        with _lib.on_device_of(x):
            y, slope = _expert_forward(x, w, slots, offsets, slots.shape[0], places.shape[1], gather, act, width, act != 0)
        ctx.save_for_backward(slope, w.codes, w.scale, w.zero_point, offsets, places)
        ctx.weight, ctx.act, ctx.dtype, ctx.gather = w[3:], act, x.dtype, gather
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        refuse_transforms("expert_linear", dy)
        slope, codes, scale, zp, offsets, places = ctx.saved_tensors
        w = PackedWeight(codes, scale, zp, *ctx.weight)
        with _lib.on_device_of(dy):
            dz, ldz, _ = activation_grad(dy, slope, w.n, ctx.act, ctx.dtype, True, False)
            # a token's rows are added up in fp32 and rounded once
            dx = grad_input(dz, ldz, w, offsets, ctx.dtype, fp32=ctx.gather)
            if ctx.gather:
                dx = _combine(dx, None, places, ctx.dtype)
        return dx, None, None, None, None, None, None, None


def expert_linear(x: torch.Tensor, packed: torch.Tensor, decompressor, routing: ExpertRouting, gather: bool = True,
                  activation: Optional[str] = None) -> torch.Tensor:
    """act(x_r W_e^T) for every row r of the routing and its expert e, with W = decompressor(packed) [experts, out, in].

    x         gather: [tokens, in], row r reads the token of its slot; else [tokens * top_k, in] in the order of the rows
              (what another `expert_linear` returned)
    returns   [tokens * top_k, out] (swiglu: out / 2) in the order of the rows; rows that no token has are zero

    Activations, types and gradients as in `nncf_amd.linear.compressed_linear`; differentiable in x.  The workspace of many rows
    or of x's gradient is two bytes per weight of the whole stack."""
    what = "expert_linear"
    _lib.require_gpu(x, what)
    refuse_transforms(what, x)
    w = packed_weight(packed, decompressor, x, 3, what)
    act, width = activation_of(activation, w.n, what)
    tokens, top_k = _check_routing(routing, x, what, w.experts)
    rows = tokens * top_k
    if x.ndim != 2 or tuple(x.shape) != (tokens if gather else rows, w.k):
        raise InternalError(f"{what}: x of shape {tuple(x.shape)}, expected {(tokens if gather else rows, w.k)}")
    if torch.is_grad_enabled() and x.requires_grad:
        return _ExpertLinear.apply(x, w, routing.slots, routing.offsets, routing.rows, bool(gather), act, width)
    with _lib.on_device_of(x):
        return _expert_forward(x, w, routing.slots, routing.offsets, rows, top_k, bool(gather), act, width, False)[0]


def _combine(y, weights, places, dtype):
    tokens, top_k = places.shape
    n = y.shape[1]
    src, ldy = rows_of(y, n) if n else (y, 0)
    out = torch.empty((tokens, n), dtype=dtype, device=y.device)
    _lib.check(_lib.lib().nncf_amd_combine_experts(ptr(src), _lib.dtype_id(src), ldy, src.shape[0], ptr(weights), ptr(places),
                                                   tokens, top_k, n, ptr(out), _DTYPES[dtype], _lib.raw_stream(y)))
    return out


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, places, slots):
        with _lib.on_device_of(y):
            out = _combine(y, weights, places, y.dtype)
        ctx.save_for_backward(y, weights, places, slots)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        refuse_transforms("combine_experts", dout)
        y, weights, places, slots = ctx.saved_tensors
        tokens, top_k = places.shape
        n = y.shape[1]
        need_y, need_w = ctx.needs_input_grad[:2]
        src, ldy = rows_of(y, n)
        dy = torch.empty(y.shape, dtype=y.dtype, device=y.device) if need_y else None
        dw = torch.empty((tokens, top_k), dtype=torch.float32, device=y.device) if need_w else None
        dout = dout.contiguous()
        with _lib.on_device_of(y):
            _lib.check(_lib.lib().nncf_amd_combine_experts_grad(
                ptr(dout), _DTYPES[y.dtype], ptr(src), ldy, ptr(weights), ptr(places), ptr(slots), tokens, top_k, n,
                ptr(dy), ptr(dw), _lib.raw_stream(y)))
        return dy, dw, None, None


def combine_experts(y: torch.Tensor, routing: ExpertRouting) -> torch.Tensor:
    """[tokens, n]: the sum of a token's rows of y [tokens * top_k, n] (float16 or bfloat16) by their weights, in float32 and
    rounded once; a masked token's is zero.  Differentiable in y and routing.weights."""
    what = "combine_experts"
    _lib.require_gpu(y, what)
    tokens, top_k = _check_routing(routing, y, what)
    refuse_transforms(what, y, routing.weights)
    if y.dtype not in _DTYPES:
        raise InternalError(f"{what}: rows are float16 or bfloat16, got {y.dtype}")
    if y.ndim != 2 or y.shape[0] != tokens * top_k or y.shape[1] < 1:
        raise InternalError(f"{what}: y of shape {tuple(y.shape)} for {tokens * top_k} rows")
    if torch.is_grad_enabled() and (y.requires_grad or routing.weights.requires_grad):
        return _Combine.apply(y, routing.weights, routing.rows, routing.slots)
    with _lib.on_device_of(y):
        return _combine(y, routing.weights, routing.rows, y.dtype)


# ---------------------------------------------------------------------------------------------------------------- layer
class CompressedExperts(nn.Module):
    """A gated expert layer on compressed stacks: out = sum_e weight_e * down_e(silu(gate_e x) * up_e x), gate_up
    [experts, 2 * inter, hidden] with the gate's rows first, down [experts, hidden, inter]."""

    def __init__(self, gate_up: torch.Tensor, gate_up_decompressor: nn.Module, down: torch.Tensor, down_decompressor: nn.Module, top_k: int,
                 renormalize: bool = True):
        super().__init__()
        self.gate_up = nn.Parameter(gate_up, requires_grad=False)
        self.down = nn.Parameter(down, requires_grad=False)
        self.gate_up_decompressor = gate_up_decompressor
        self.down_decompressor = down_decompressor
        self.top_k, self.renormalize = top_k, renormalize

    def forward(self, hidden: torch.Tensor, router_logits: torch.Tensor, token_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """hidden [..., hidden], router_logits [..., experts] (token_mask [...]): the experts' answer in hidden's shape."""
        flat = hidden.reshape(-1, hidden.shape[-1])
        routing = route_experts(router_logits.reshape(-1, router_logits.shape[-1]), self.top_k, self.renormalize,
                                None if token_mask is None else token_mask.reshape(-1))
        inner = expert_linear(flat, self.gate_up, self.gate_up_decompressor, routing, activation="swiglu")
        rows = expert_linear(inner, self.down, self.down_decompressor, routing, gather=False)
        return combine_experts(rows, routing).reshape(hidden.shape)


def _expert_decompressor(cfg, cw, shape, dtype):
    mode = cfg.mode
    if mode == CompressWeightsMode.INT8_SYM:
        return dcmp.INT8SymmetricWeightsDecompressor(cw.scale, result_dtype=dtype)
    if mode == CompressWeightsMode.INT8_ASYM:
        return dcmp.INT8AsymmetricWeightsDecompressor(cw.scale, cw.zero_point, result_dtype=dtype)
    gs = cfg.group_size
    grouped = tuple(shape) if gs == -1 else tuple(shape[:-1]) + (shape[-1] // gs, gs)
    kw = dict(compressed_weight_shape=grouped, result_shape=tuple(shape), result_dtype=dtype)
    if mode == CompressWeightsMode.INT4_SYM:
        return dcmp.INT4SymmetricWeightsDecompressor(cw.scale, **kw)
    if mode == CompressWeightsMode.INT4_ASYM:
        return dcmp.INT4AsymmetricWeightsDecompressor(cw.scale, cw.zero_point, **kw)
    if mode == CompressWeightsMode.NF4:
        return dcmp.NF4WeightsDecompressor(cw.scale, **kw)
    if mode == CompressWeightsMode.MXFP4:
        return dcmp.MXFP4WeightsDecompressor(cw.codebook.reshape(cw.scale.shape), **kw)
    raise InternalError(f"no decompressor for {mode}")


def compress_experts(gate_up: torch.Tensor, down: torch.Tensor, config, top_k: int, renormalize: bool = True) -> CompressedExperts:
    """Compresses the stacks of a gated expert layer (gate_up [experts, 2 * inter, hidden], down [experts, hidden, inter],
    float16 or bfloat16, on the GPU) with one configuration and returns the layer that answers with them."""
    from nncf_amd.weight_lowering import compress_weights_packed_batched

    config = as_config(config)
    if gate_up.ndim != 3 or down.ndim != 3 or gate_up.shape[0] != down.shape[0] or gate_up.shape[1] != 2 * down.shape[2] \
            or gate_up.shape[2] != down.shape[1]:
        raise InternalError(f"compress_experts: gate_up {tuple(gate_up.shape)} and down {tuple(down.shape)} do not belong together")
    if gate_up.dtype not in _DTYPES or down.dtype != gate_up.dtype:
        raise InternalError(f"compress_experts: float16 or bfloat16 stacks, got {gate_up.dtype} and {down.dtype}")
    parts = []
    for w in (gate_up, down):
        cw = compress_weights_packed_batched([w], config, want_e8m0=True)[0]
        codes = cw.tensor if config.num_bits == 4 else cw.tensor.reshape(w.shape)
        parts += [codes, _expert_decompressor(config, cw, w.shape, w.dtype)]
    return CompressedExperts(*parts, top_k=top_k, renormalize=renormalize)
