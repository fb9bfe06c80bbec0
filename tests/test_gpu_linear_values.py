"""GPU: values at the ends of their types in compressed weights (nncf_amd.linear), against the plain product in 64 bits with the
bounds of tests/linear_utils.py."""
import pytest
import torch

from tests.linear_utils import assert_within, make_weight, plain

pytestmark = pytest.mark.gpu


def _rows(m, k, dtype, seed):
    return torch.randn(m, k, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _nibbles(values):
    return (values[..., 0::2] | (values[..., 1::2] << 4)).reshape(-1, 1).contiguous()


@pytest.mark.parametrize("m", [1, 5, 16, 33, 64, 130, 300])
@pytest.mark.parametrize("mode,gs,n,k,dtype", [("int4_sym", 64, 64, 320, torch.bfloat16), ("int4_sym", 32, 48, 352, torch.bfloat16),
                                               ("int4_sym", 32, 33, 32, torch.bfloat16), ("int4_asym", 64, 80, 448, torch.bfloat16),
                                               ("int4_asym", 32, 16, 96, torch.bfloat16), ("int4_sym", 64, 130, 4160, torch.bfloat16),
                                               ("mxfp4", 32, 64, 416, torch.float16), ("mxfp4", 32, 16, 4128, torch.float16)])
def test_a_large_scale_meets_its_own_codes_only(mode, gs, n, k, dtype, m):
    """The last group's scale is so large that codes of other groups would leave fp16 under it, while its own do not: the weight is
    finite, and what lies behind the end of k must not bring an infinity in (times x's zeros it would be NaN)."""
    from nncf_amd.linear import compressed_linear
    packed, dec = make_weight(mode, gs, (n, k), dtype, seed=k)
    codes = torch.randint(0, 16, (n, k), dtype=torch.uint8, generator=torch.Generator().manual_seed(m)).cuda()
    last = codes[:, k - gs:]
    last.remainder_(2)  # mxfp4: 0 and 0.5
    if mode == "mxfp4":
        dec._scale[:, -1] = 127 + 15
        codes[:, : min(32, k - gs)] = 7  # 6
    else:
        if mode == "int4_sym":
            last.add_(7)  # -1 and 0
        else:
            dec._zero_point.zero_()  # 0 and 1
        dec._scale[:, -1] = 16000.0
        codes[:, : min(32, k - gs)] = 15
        codes[:, 0] = 0 if mode == "int4_sym" and k > gs else codes[:, 0]
    packed.copy_(_nibbles(codes))
    w = dec(packed)
    assert bool(torch.isfinite(w).all())
    x = _rows(m, k, dtype, m) * (2.0 ** -10)
    y, by = plain(x, w)
    assert_within(compressed_linear(x, packed, dec), y, by)


def _identity(k, dtype):
    """A weight of ones on the diagonal: the sums are x itself."""
    from nncf_amd import decompressors as D
    return torch.eye(k, dtype=torch.int8, device="cuda"), D.INT8SymmetricWeightsDecompressor(torch.ones(k, 1, device="cuda"), result_dtype=dtype)


def _every_value(dtype, k, reach):
    """All numbers of a 16-bit type up to `reach` on both sides as rows of k (the last one filled up with zeros)."""
    v = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16).view(dtype)
    v = v[torch.isfinite(v) & (v.abs() <= reach)]
    return torch.cat((v, v.new_zeros(-v.numel() % k))).view(-1, k).cuda()


def _in_pieces(x, m, call):
    return torch.cat([call(x[r:r + m]) for r in range(0, x.shape[0], m)])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("m", [1, 100, 1024])
def test_activations_are_right_to_their_last_place(m, act, dtype):
    """Every value of x: an activation is off by a share of ITSELF, also far out on the left, where it is small.  With u = 2^-24:
    the exponential of an argument a, rounded twice or three times on its way, is off by 3 u |a| of itself, its instruction, a
    reciprocal and a handful of products, sums of positive terms and a fitted polynomial (7e-7) by 40 u; then y is rounded once.
    |a| is z^2 / 2, 2 sqrt(2 / pi) |z + 0.044715 z^3| or |z|.  z's factor may be flushed below the smallest normal number, 2^-126:
    that takes 2^-126 |z| from the product, and the product itself may be flushed."""
    from nncf_amd.linear import compressed_linear
    k, u = 256, 2.0 ** -24
    packed, dec = _identity(k, dtype)
    x = _every_value(dtype, k, 80.0 if act == "silu" else 12.5)
    got = _in_pieces(x, m, lambda t: compressed_linear(t, packed, dec, activation=act))
    z = x.double()
    if act == "gelu":
        want, a = z * 0.5 * torch.erfc(-z * 0.5 ** 0.5), z * z / 2
    else:
        a = z if act == "silu" else 1.5957691216057308 * (z + 0.044715 * z ** 3)
        want = z * torch.sigmoid(a)
    off = want.abs() * (40 * u + 3 * u * a.abs()) + 2.0 ** -126 * (1 + z.abs())
    half = torch.finfo(dtype).eps / 2
    assert_within(got, want, off + (want.abs() + off) * half + torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [1, 1024])
def test_the_slope_of_gelu_is_right_to_its_last_place(m, dtype):
    """As above for Phi(z) + z phi(z) with dy = 1: each of the two is off by a share of itself, dz is rounded once, dx (one product)
    once more without another error."""
    from nncf_amd.linear import compressed_linear
    k, u = 256, 2.0 ** -24
    packed, dec = _identity(k, dtype)
    x = _every_value(dtype, k, 12.5)

    def gradient(t):
        t = t.clone().requires_grad_(True)
        return torch.autograd.grad(compressed_linear(t, packed, dec, activation="gelu"), t, torch.ones_like(t))[0]
    got = _in_pieces(x, m, gradient)
    z = x.double()
    cdf, rest = 0.5 * torch.erfc(-z * 0.5 ** 0.5), z * torch.exp(-z * z / 2) * 0.3989422804014327
    want = cdf + rest
    off = (cdf + rest.abs()) * (40 * u + 3 * u * z * z / 2) + 2.0 ** -126 * (1 + z.abs())
    half = torch.finfo(dtype).eps / 2
    assert_within(got, want, off + (want.abs() + off) * half + torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 16, 64, 256, 2048])
@pytest.mark.parametrize("mode", ["int4_sym", "int4_asym", "nf4", "mxfp4", "int8_asym", "int8_sym"])
def test_subnormal_weights_are_the_decompressor_s_bit_for_bit(mode, rows, dtype):
    """x = unit rows, so a result is the weight itself: with scales of fp16's subnormal range (integer modes, NF4) or the lowest
    bytes of E8M0, most weights are below their type's smallest normal number.  No way of the product flushes them."""
    from nncf_amd.linear import compressed_linear
    k, n = 256, 64
    packed, dec = make_weight(mode, -1 if mode.startswith("int8") else 32, (n, k), dtype, seed=1)
    if mode == "mxfp4":  # bytes 0 ... 126
        dec._scale.copy_((torch.arange(dec._scale.numel(), device="cuda") % 127).to(torch.uint8).view_as(dec._scale))
    else:
        dec._scale.copy_((torch.rand(dec._scale.shape, generator=torch.Generator().manual_seed(2)) * 4e-7 + 6e-8).half())
    w = dec(packed)
    below = (w != 0) & (w.abs() < torch.finfo(dtype).tiny)
    assert int(below.sum()) >= (50 if mode == "mxfp4" else n * k // 2 if dtype == torch.float16 else 0)
    eye = torch.eye(k, dtype=dtype, device="cuda").repeat(8, 1)
    got = torch.cat([compressed_linear(eye[r:r + rows], packed, dec) for r in range(0, max(k, rows), rows)])
    assert torch.equal(got, w.t().repeat(8, 1)[: got.shape[0]])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 64, 256])
def test_subnormal_activations_count(rows, dtype):
    from nncf_amd.linear import compressed_linear
    packed, dec = make_weight("int8_sym", -1, (64, 256), dtype, seed=1)
    dec._scale.fill_(1.0)
    step = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    x = torch.zeros(256, 256, dtype=dtype, device="cuda").fill_diagonal_(4 * step)
    got = torch.cat([compressed_linear(x[r:r + rows], packed, dec) for r in range(0, 256, rows)])
    assert torch.equal(got, (dec(packed).double().t() * 4 * step).to(dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_subnormal_weights_in_the_gradient(dtype):
    """dy = unit rows: dx is a row of the weight."""
    from nncf_amd.linear import compressed_linear
    for mode in ("int4_asym", "int8_sym", "mxfp4"):
        packed, dec = make_weight(mode, -1 if mode == "int8_sym" else 32, (256, 64), dtype, seed=3)
        if mode == "mxfp4":
            dec._scale.copy_((torch.arange(dec._scale.numel(), device="cuda") % 100).to(torch.uint8).view_as(dec._scale))
        else:
            dec._scale.copy_((torch.rand(dec._scale.shape, generator=torch.Generator().manual_seed(4)) * 4e-7 + 6e-8).half())
        x = torch.zeros(256, 64, dtype=dtype, device="cuda", requires_grad=True)
        dx = torch.autograd.grad(compressed_linear(x, packed, dec), x, torch.eye(256, dtype=dtype, device="cuda"))[0]
        assert torch.equal(dx, dec(packed))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu", "swiglu"])
@pytest.mark.parametrize("m", [1, 60, 333])
def test_the_gradient_of_x_is_rounded_twice(m, act, dtype):
    """Between dy and dx only dz is rounded to 16 bits (half a step), and dx itself: the slopes are those of the fp32 sums.  With u
    = 2^-24: a sum z of K products is off by ez <= 2 (K + 2) u sum|x w|, a slope by at most 1.2 ez and by 32 u (1 + |z|) of its
    arithmetic (swiglu: that of silu times the other half, which is off by its own ez); dz by that and half a step; dx, a sum of N
    products, by 2 N u of their magnitudes."""
    from nncf_amd.linear import compressed_linear
    from tests.linear_utils import act64
    n, k, u, half = 320, 256, 2.0 ** -24, torch.finfo(dtype).eps / 2
    packed, dec = make_weight("int4_sym", 64, (n, k), dtype, seed=m)
    x = (_rows(m, k, dtype, m) * 0.3).requires_grad_()
    y = compressed_linear(x, packed, dec, activation=act)
    dy = _rows(m, y.shape[-1], dtype, m + 2)
    y.backward(dy)
    w, d = dec(packed).double(), dy.double()
    z = (x.detach().double() @ w.t()).requires_grad_()
    dz = torch.autograd.grad(act64(z, act), z, d)[0]
    z = z.detach()
    ez = 2 * (k + 2) * u * (x.detach().double().abs() @ w.abs().t())
    if act == "swiglu":
        (a, b), (ea, eb) = z.chunk(2, -1), ez.chunk(2, -1)
        off = torch.cat((d.abs() * (1.2 * (ea * b.abs() + eb) + 32 * u * (1 + a.abs()) * b.abs()),
                         d.abs() * (1.2 * ea + 32 * u * (1 + a.abs()) * (1 + a.abs()))), -1)
    else:
        off = d.abs() * (1.2 * ez + 32 * u * (1 + z.abs()))
        if act == "relu":  # the slope jumps where the sign of z is not settled
            off = off + torch.where(z.abs() <= ez, d.abs(), torch.zeros_like(d))
    step = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    off = off + half * (dz.abs() + off) + step
    want = dz @ w
    off = off @ w.abs() + 2 * n * u * ((dz.abs() + off) @ w.abs())
    assert_within(x.grad, want, off + half * (want.abs() + off) + step)
    # The same in the mean, where a slope kept in 16 bits would show (it would add another rounding of dz, half as much again to
    # what follows): a rounding is uniform over a step of its value, step^2 / 12 in the mean square, and those of dz meet in dx
    # independently.  Some 10^4 of them leave a few hundredths to chance; a fifth is allowed.
    if dtype == torch.bfloat16 and act != "relu" and m > 1:
        def step2(v):
            return torch.exp2(2 * torch.floor(torch.log2(v.abs().clamp(min=1e-30)))) * torch.finfo(dtype).eps ** 2 / 12
        expected = step2(dz) @ w.square() + step2(want)
        assert (x.grad.double() - want).square().sum() <= 1.2 * expected.sum()
