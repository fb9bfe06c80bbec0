"""Products with compressed weights: what a compressed layer computes, without its weight in between.

The reference's Torch backend answers with a compressed layer in two steps, the decompressor module on every read of the weight
(src/nncf/torch/quantization/layers.py:1303-1460) and a library product.  `compressed_linear` multiplies by the packed codes
themselves, with bias, activation and residual in the product's epilogue and with the gradients that reach the activations
(adapters that are trained beside frozen compressed weights).  The weight's values are bit for bit those of the decompressor,
sums are fp32 and the result is rounded once.

`fuse_compressed_linears` lets every `nn.Linear` of a compressed model answer this way.
"""
from __future__ import annotations

import functools
import math
import types
from typing import NamedTuple, Optional, Tuple

import torch
from torch import nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from nncf_amd import _lib
from nncf_amd import decompressors as dcmp
from nncf_amd.errors import InternalError

ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4, "swiglu": 5}
_SWIGLU = ACTIVATIONS["swiglu"]
_DTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


class PackedWeight(NamedTuple):
    """A compressed weight as the kernels take it: [experts, n, k] codes with their scales and zero points."""
    codes: torch.Tensor
    scale: torch.Tensor
    zero_point: Optional[torch.Tensor]
    mode: int
    experts: int
    n: int
    k: int
    group_size: int


_MODE_OF = {dcmp.INT8AsymmetricWeightsDecompressor: "int8_asym", dcmp.INT8SymmetricWeightsDecompressor: "int8_sym",
            dcmp.INT4AsymmetricWeightsDecompressor: "int4_asym", dcmp.INT4SymmetricWeightsDecompressor: "int4_sym",
            dcmp.NF4WeightsDecompressor: "nf4", dcmp.MXFP4WeightsDecompressor: "mxfp4"}


def _mode_or_none(decompressor) -> Optional[str]:
    """The mode whose codes `decompressor` decompresses as this package does; None for another's, also of a subclass that overrides
    its forward (the weight would not be the one that the kernels multiply by)."""
    mode = _MODE_OF.get(type(decompressor))
    if mode is None:
        for cls, mode in _MODE_OF.items():
            if isinstance(decompressor, cls):
                return mode if type(decompressor).forward is cls.forward else None
        return None
    return mode


def _mode_of(decompressor) -> str:
    mode = _mode_or_none(decompressor)
    if mode is None:
        raise InternalError(f"{type(decompressor).__name__} is not a decompressor of this package")
    return mode


def weight_dtype_of(decompressor) -> torch.dtype:
    """Type of the weight that `decompressor` returns."""
    if decompressor.result_dtype is not None:
        return decompressor.result_dtype
    scale = decompressor._buffers["_scale"]
    return scale.dtype if scale.is_floating_point() else torch.float16


_transforms_active = torch._C._are_functorch_transforms_active


def transformed(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether one of `tensors` carries a forward-mode tangent or comes from a function transform (torch.func)."""
    if forward_ad._current_level < 0 and not _transforms_active():
        return False
    return any(t is not None and (torch._C._functorch.is_functorch_wrapped_tensor(t) or forward_ad.unpack_dual(t).tangent is not None)
               for t in tensors)


def refuse_transforms(what: str, *tensors: Optional[torch.Tensor]) -> None:
    if transformed(*tensors):
        raise InternalError(f"{what}: forward-mode derivatives and function transforms are not supported")


def packed_weight(packed: torch.Tensor, decompressor, x: torch.Tensor, ndim: int, what: str) -> PackedWeight:
    """`packed` and its decompressor as the kernels take them; ndim: 2 for [n, k], 3 for [experts, n, k]."""
    mode = _mode_of(decompressor)
    dtype, device = x.dtype, x.get_device()
    if dtype not in _DTYPES:
        raise InternalError(f"{what}: activations are float16 or bfloat16, got {dtype}")
    if weight_dtype_of(decompressor) != dtype:
        raise InternalError(f"{what}: activations are {dtype}, the decompressed weight is {weight_dtype_of(decompressor)}")
    buffers = decompressor._buffers  # (module attributes are looked up through several dictionaries)
    scale, zp = buffers["_scale"], buffers.get("_zero_point")
    four = mode not in ("int8_sym", "int8_asym")
    if four:
        grouped = tuple(decompressor.compressed_weight_shape)
        shape = grouped if decompressor.result_shape is None else tuple(decompressor.result_shape)
    else:
        shape = grouped = tuple(packed.shape)
    elements, n_groups = math.prod(shape), scale.numel()
    if len(shape) != ndim or elements == 0:
        raise InternalError(f"{what}: the weight is {ndim}-dimensional and not empty, got shape {shape}")
    n, k = shape[-2:]
    group_size = elements // n_groups if n_groups else 0
    if tuple(scale.shape) != grouped[:-1] + (1,) or group_size * n_groups != elements or k % group_size:
        raise InternalError(f"{what}: scales {tuple(scale.shape)} do not divide a weight of shape {shape} ({grouped}) into groups")
    if packed.dtype != (torch.int8 if mode == "int8_sym" else torch.uint8):
        raise InternalError(f"{what}: packed codes of type {packed.dtype} for mode {mode}")
    if packed.numel() != (elements // 2 if four else elements):
        raise InternalError(f"{what}: {packed.numel()} bytes of codes for a weight of shape {shape}, mode {mode}")
    if scale.dtype != (torch.uint8 if mode == "mxfp4" else torch.float16):
        raise InternalError(f"{what}: scales of type {scale.dtype} for mode {mode}")
    if packed.get_device() != device or scale.get_device() != device or (zp is not None and zp.get_device() != device):
        raise InternalError(f"{what}: the weight is on {packed.device} and {scale.device}, the activations on {x.device}")
    if zp is not None:
        if zp.dtype != torch.uint8 or zp.numel() != ((n_groups + 1) // 2 if four else n_groups):
            raise InternalError(f"{what}: {zp.numel()} bytes of zero points ({zp.dtype}) for {n_groups} groups, mode {mode}")
        if not zp.is_contiguous():
            zp = zp.contiguous()
    return PackedWeight(packed if packed.is_contiguous() else packed.contiguous(), scale if scale.is_contiguous() else scale.contiguous(), zp,
                        _lib.MODE_ID[mode], shape[0] if ndim == 3 else 1, n, k, group_size)


def activation_of(activation: Optional[str], n: int, what: str) -> Tuple[int, int]:
    """(number of the activation, columns of the result)."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"{what}: unknown activation {activation!r}, expected one of {list(ACTIVATIONS)}")
    act = ACTIVATIONS[activation]
    if act != _SWIGLU:
        return act, n
    if n % 2:
        raise ValueError(f"{what}: swiglu needs an even number of weight rows, got {n}")
    return act, n // 2


def rows_of(t: torch.Tensor, width: int) -> Tuple[torch.Tensor, int]:
    """`t` [..., width] as rows of consecutive elements and their distance (copied where its strides do not allow it)."""
    if t.ndim != 2:
        t = t.reshape(-1, width)
    if t.is_contiguous():
        return t, width
    if (width > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < width):
        return t.contiguous(), width
    return t, t.stride(0) if t.shape[0] > 1 else width


def ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


@functools.lru_cache(maxsize=8192)
def workspace_bytes(query: str, *numbers: int) -> int:
    """What a size query of the library answers: it depends on its numbers alone (on addresses by their alignment to 16 bytes)."""
    return getattr(_lib.lib(), query)(*numbers)


def workspace_of(nbytes: int, device) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def activation_grad(dy: torch.Tensor, slope: Optional[torch.Tensor], n: int, act: int, dtype: torch.dtype, want_dz: bool, want_dbias: bool):
    """(dz, its row stride, dbias) of the epilogue: dz = dy * slope, rounded to `dtype`, the type that the product behind it reads."""
    width = n // 2 if act == _SWIGLU else n
    dy, ldd = rows_of(dy, width)
    m = dy.shape[0]
    if act == 0 and not want_dbias:
        return dy, ldd, None
    L = _lib.lib()
    copies = want_dz and act != 0  # without an activation dz is dy
    dz = torch.empty((m, n), dtype=dtype, device=dy.device) if copies else None
    dbias = torch.empty(n, dtype=dtype, device=dy.device) if want_dbias else None
    ws = workspace_of(workspace_bytes("nncf_amd_activation_grad_workspace", m, n) if want_dbias else 0, dy.device)
    _lib.check(L.nncf_amd_activation_grad(ptr(dy), _DTYPES[dtype], ldd, ptr(slope), m, n, act, ptr(dz), n, ptr(dbias),
                                          ptr(ws), 0 if ws is None else ws.numel(), _lib.raw_stream(dy)))
    return (dz, n, dbias) if copies else (dy, ldd, dbias)


def grad_input(dz: torch.Tensor, ldz: int, w: PackedWeight, offsets: Optional[torch.Tensor], dtype: torch.dtype,
               fp32: bool = False) -> torch.Tensor:
    L = _lib.lib()
    m = dz.shape[0]
    dx = torch.empty((m, w.k), dtype=torch.float32 if fp32 else dtype, device=dz.device)
    ws = workspace_of(workspace_bytes("nncf_amd_linear_grad_input_workspace", dz.data_ptr() & 15, ldz, m, w.n, w.k, w.experts), dz.device)
    _lib.check(L.nncf_amd_linear_grad_input(ptr(dz), _DTYPES[dtype], ldz, ptr(offsets), w.experts, m, w.n, w.k, ptr(w.codes),
                                            w.mode, w.group_size, ptr(w.scale), ptr(w.zero_point), ptr(dx), w.k, int(fp32),
                                            ptr(ws), 0 if ws is None else ws.numel(), _lib.raw_stream(dz)))
    return dx


def _forward(x, w: PackedWeight, bias, act: int, width: int, residual, want_slope: bool):
    """(y [m, width], slope [m, n] or None) of rows x [..., k]."""
    rows, ldx = rows_of(x, w.k)
    m = rows.shape[0]
    y = torch.empty((m, width), dtype=x.dtype, device=x.device)
    slope = torch.empty((m, w.n), dtype=torch.float32, device=x.device) if want_slope else None
    res, ldr = (None, 0) if residual is None else rows_of(residual, width)
    L = _lib.lib()
    ws = workspace_of(workspace_bytes("nncf_amd_compressed_linear_workspace", rows.data_ptr() & 15, ldx, m, w.n, w.k,
                                      w.codes.data_ptr() & 15, w.mode, w.group_size, act), x.device)
    _lib.check(L.nncf_amd_compressed_linear(ptr(rows), _DTYPES[x.dtype], ldx, m, w.n, w.k, ptr(w.codes), w.mode, w.group_size,
                                            ptr(w.scale), ptr(w.zero_point), ptr(bias), act, ptr(res), ldr,
                                            ptr(y), width, ptr(slope), ptr(ws), 0 if ws is None else ws.numel(),
                                            _lib.raw_stream(x)))
    return y, slope


class _CompressedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, bias, residual, w, act, width):
        with _lib.on_device_of(x):
            y, slope = _forward(x, w, bias, act, width, residual, act != 0 and (ctx.needs_input_grad[0] or ctx.needs_input_grad[1]))
        ctx.save_for_backward(slope, w.codes, w.scale, w.zero_point)
        ctx.weight, ctx.act, ctx.shape, ctx.dtype = w[3:], act, x.shape, x.dtype
        return y.reshape(x.shape[:-1] + (width,))

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        refuse_transforms("compressed_linear", dy)
        slope, codes, scale, zp = ctx.saved_tensors
        w = PackedWeight(codes, scale, zp, *ctx.weight)
        need_x, need_bias, need_residual = ctx.needs_input_grad[:3]
        dx = dbias = None
        if need_x or need_bias:
            with _lib.on_device_of(dy):
                dz, ldz, dbias = activation_grad(dy, slope, w.n, ctx.act, ctx.dtype, need_x, need_bias)
                if need_x:
                    dx = grad_input(dz, ldz, w, None, ctx.dtype).reshape(ctx.shape)
        return dx, dbias, dy if need_residual else None, None, None, None


def compressed_linear(x: torch.Tensor, packed: torch.Tensor, decompressor, bias: Optional[torch.Tensor] = None,
                      activation: Optional[str] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x W^T + bias) + residual with W = decompressor(packed), which is never written to memory in the layer's place.

    x            [..., in_features], float16 or bfloat16, any strides; the type of the decompressed weight
    packed       the packed codes of a [out_features, in_features] weight, with their decompressor (`nncf_amd.decompressors`)
    bias         [out_features] in x's type
    activation   None, "relu", "gelu", "gelu_tanh", "silu", or "swiglu": the first half of W's rows is the gate, the result
                 silu(gate) * up has out_features / 2 columns
    residual     the result's shape and type

    Differentiable in x, bias and residual (in reverse mode, not twice); the weight is frozen.  With an activation the backward
    pass keeps its slope at every sum, in fp32 (4 bytes for each of rows x out_features); the gradient of the sums is rounded to
    x's type for the product that gives x's, as autograd's would be, so that one carries two roundings.  From some hundreds of
    rows on, and for x's gradient, a call takes a workspace of two bytes per weight."""
    what = "compressed_linear"
    _lib.require_gpu(x, what)
    refuse_transforms(what, x, bias, residual)
    w = packed_weight(packed, decompressor, x, 2, what)
    act, width = activation_of(activation, w.n, what)
    if x.ndim < 1 or x.shape[-1] != w.k:
        raise InternalError(f"{what}: x of shape {tuple(x.shape)} for a weight with {w.k} input features")
    if bias is not None:
        if tuple(bias.shape) != (w.n,) or bias.dtype != x.dtype or bias.device != x.device:
            raise InternalError(f"{what}: bias {tuple(bias.shape)} {bias.dtype} on {bias.device}, expected ({w.n},) {x.dtype} on {x.device}")
    if residual is not None:
        if tuple(residual.shape) != tuple(x.shape[:-1]) + (width,) or residual.dtype != x.dtype or residual.device != x.device:
            raise InternalError(f"{what}: residual {tuple(residual.shape)} {residual.dtype} on {residual.device}, expected "
                                f"{tuple(x.shape[:-1]) + (width,)} {x.dtype} on {x.device}")
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _CompressedLinear.apply(x, bias, residual, w, act, width)
    with _lib.on_device_of(x):
        y, _ = _forward(x, w, bias, act, width, residual, False)
    return y if x.ndim == 2 else y.reshape(x.shape[:-1] + (width,))


# ------------------------------------------------------------------------------------------------------------- models
_LINEAR_FORWARD = nn.Linear.forward


def _only_decompressed(mod: nn.Module):
    """The parametrizations of `mod`'s weight if a decompressor of this package is all they are (an adapter may have joined it, or
    left), as it was made: no hooks, nor scales that were cast (`model.float()` does).  Else None."""
    parametrizations = mod._modules.get("parametrizations")
    plist = None if parametrizations is None else parametrizations._modules.get("weight")
    if plist is None or len(plist) != 1:
        return None
    dec = plist[0]
    if _mode_or_none(dec) is None or dec._forward_hooks or dec._forward_pre_hooks or "forward" in dec.__dict__:
        return None
    return plist if dec._buffers["_scale"].dtype in (torch.float16, torch.uint8) else None


def _fused_forward(self, x: torch.Tensor) -> torch.Tensor:
    plist = _only_decompressed(self)
    if plist is None or not x.is_cuda or torch.is_autocast_enabled("cuda") or x.dtype != weight_dtype_of(plist[0]):
        return nn.Linear.forward(self, x)  # a library product of the weight as it is now, as before
    bias = self.bias
    if transformed(x, bias):
        return nn.Linear.forward(self, x)
    return compressed_linear(x, plist.original, plist[0], bias=bias)


def _answers_as_linear(mod: nn.Module) -> bool:
    """Whether `mod` answers by nn.Linear's own forward (or by the one it was given here): not a subclass that overrides it
    (adapters) nor a module whose forward was replaced (offloading, wrappers), which would lose what they add."""
    if not isinstance(mod, nn.Linear) or type(mod).forward is not _LINEAR_FORWARD:
        return False
    own = mod.__dict__.get("forward")
    return own is None or getattr(own, "__func__", None) is _fused_forward


def fuse_compressed_linears(model: nn.Module) -> int:
    """Lets every `nn.Linear` of a compressed model (`nncf_amd.compress_weights`, `load_compressed`) whose weight is float16 or
    bfloat16 answer through `compressed_linear` instead of decompressing its weight and calling a library product.  In place;
    parameters, state_dict keys and `save_compressed` stay as they are, results differ by the sums' order only; their
    gradients can be taken once.  A subclass with a forward of its own, or a module whose forward was replaced, stays as it is;
    calls on the CPU, under autocast, in another type, in forward mode or under a function transform go the former way.  Returns
    how many modules now answer so."""
    count = 0
    for mod in model.modules():
        plist = _only_decompressed(mod) if _answers_as_linear(mod) else None
        if plist is None or weight_dtype_of(plist[0]) not in _DTYPES:
            continue
        if mod.bias is not None and mod.bias.dtype != weight_dtype_of(plist[0]):
            continue
        mod.forward = types.MethodType(_fused_forward, mod)
        count += 1
    return count
