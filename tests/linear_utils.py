"""Compressed weights from random codes, the plain products in 64 bits, and the bounds of their comparison (shared by the tests
of nncf_amd.linear and nncf_amd.experts)."""
import math

import torch

MODES = ("int4_sym", "int4_asym", "nf4", "mxfp4", "int8_asym", "int8_sym")
FOUR = MODES[:4]


def make_weight(mode, gs, shape, dtype, seed=0, device="cuda"):
    """(packed, decompressor) of a weight [(experts,) n, k] with every code value; gs == -1: one group per row."""
    from nncf_amd import decompressors as D
    g = torch.Generator(device="cpu").manual_seed(seed)
    k = shape[-1]
    lead = tuple(shape[:-1])
    groups = 1 if gs == -1 else k // gs
    pshape = lead + ((1,) if gs == -1 else (groups, 1))
    n = math.prod(shape)
    kw = dict(result_dtype=dtype)
    scale = (torch.rand(pshape, generator=g) * 0.02 + 0.002).to(torch.float16).to(device)
    if mode.startswith("int8"):
        codes = torch.randint(0, 256, shape, dtype=torch.uint8, generator=g).to(device)
        if mode == "int8_sym":
            return codes.view(torch.int8), D.INT8SymmetricWeightsDecompressor(scale / 8, **kw)
        zp = torch.randint(0, 256, pshape, dtype=torch.uint8, generator=g).to(device)
        return codes, D.INT8AsymmetricWeightsDecompressor(scale / 8, zp, **kw)
    packed = torch.randint(0, 256, (n // 2, 1), dtype=torch.uint8, generator=g).to(device)
    kw.update(compressed_weight_shape=tuple(shape) if gs == -1 else lead + (groups, gs), result_shape=tuple(shape))
    if mode == "mxfp4":
        return packed, D.MXFP4WeightsDecompressor(torch.randint(116, 122, pshape, dtype=torch.uint8, generator=g).to(device), **kw)
    if mode == "nf4":
        return packed, D.NF4WeightsDecompressor(scale, **kw)
    if mode == "int4_sym":
        return packed, D.INT4SymmetricWeightsDecompressor(scale, **kw)
    zp = torch.randint(0, 16, pshape, dtype=torch.uint8, generator=g).to(device)
    return packed, D.INT4AsymmetricWeightsDecompressor(scale, zp, **kw)


def act64(z, act):
    if act == "relu":
        return torch.relu(z)
    if act == "gelu":
        return torch.nn.functional.gelu(z)
    if act == "gelu_tanh":
        return torch.nn.functional.gelu(z, approximate="tanh")
    if act == "silu":
        return torch.nn.functional.silu(z)
    if act == "swiglu":
        a, b = z.chunk(2, dim=-1)
        return torch.nn.functional.silu(a) * b
    return z


def plain(x, w, bias=None, act=None, residual=None, dy=None):
    """(y, bound of |got - y|, dx, its bound, dbias, its bound) in 64 bits for operands of one 16-bit type.

    With u = 2^-24 a sum of K products in any order of fp32 additions, rounded or truncated, is off by at most 2 K u sum|x w|;
    the bias adds 2 u of what it meets.  Every activation here has a slope of at most 1.2 (swiglu: its product rule) and is
    computed to a relative 16 u or better of |z|; y is rounded once to its type (half a step).  Backward: dz is rounded to the
    type (half a step of it), and act' is taken at z rounded to the type: |z act''(z)| <= 1 for these activations, so dz is off
    by another half step of |dy| (swiglu: of |dy| times the other factor, whose own rounding counts too)."""
    u, half = 2.0 ** -24, torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps  # a subnormal's step
    X, W = x.double(), w.double()
    z = X @ W.t()
    mag = X.abs() @ W.abs().t()
    if bias is not None:
        z = z + bias.double()
        mag = mag + bias.double().abs()
    ez = 2 * (x.shape[-1] + 2) * u * mag
    y = act64(z, act)
    if act == "swiglu":
        a, b = z.chunk(2, dim=-1)
        ea, eb = ez.chunk(2, dim=-1)
        ey = 1.2 * ea * (b.abs() + eb) + eb * a.abs() + 32 * u * (a * b).abs()
    else:
        ey = ez * (1.2 if act else 1.0) + (16 * u * z.abs() if act else 0)
    if residual is not None:
        y = y + residual.double()
        ey = ey + 2 * u * (y.abs() + residual.double().abs())
    by = ey + half * (y.abs() + ey) + tiny
    if dy is None:
        return y, by
    D = dy.double()
    zz = z.detach().requires_grad_(True)
    dz = torch.autograd.grad(act64(zz, act), zz, D)[0] if act else D
    if act == "swiglu":
        a, b = z.chunk(2, dim=-1)
        slack = torch.cat((D.abs() * 2.2 * b.abs(), D.abs() * 1.2 * a.abs()), dim=-1) * half
        slope = torch.cat((D.abs() * (b.abs() + 1), D.abs()), dim=-1)
        slack = slack + 1.2 * slope * torch.maximum(ez, torch.cat((ez.chunk(2, -1)[1], ez.chunk(2, -1)[0]), -1))
    elif act:
        slack = D.abs() * half + D.abs() * ez + 32 * u * D.abs() * (1 + z.abs())
        if act == "relu":  # the slope jumps where the sign of z is not settled
            slack = slack + torch.where(z.abs() <= ez, D.abs(), torch.zeros_like(D))
    else:
        slack = torch.zeros_like(dz)
    edz = slack + half * (dz.abs() + slack) * (1 if act else 0) + (tiny if act else 0)
    dx = dz @ W
    edx = edz @ W.abs() + 2 * dz.shape[-1] * u * ((dz.abs() + edz) @ W.abs())
    bdx = edx + half * (dx.abs() + edx) + tiny
    db = dz.sum(0)
    edb = slack.sum(0) + 2 * (dz.shape[0] + 2) * u * (dz.abs() + slack).sum(0)
    bdb = edb + half * (db.abs() + edb) + tiny
    return y, by, dx, bdx, db, bdb


def assert_within(got, ref, bound, what=""):
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    off = (got.double() - ref).abs() - bound
    worst = off.argmax().item() if off.numel() else 0
    assert not off.numel() or bool((off <= 0).all()), (
        what, f"{int((~(off <= 0)).sum())} of {off.numel()} values out of bounds, worst at {worst}: "
        f"{got.reshape(-1)[worst].item()} for {ref.reshape(-1)[worst].item()} +- {bound.reshape(-1)[worst].item()}")
