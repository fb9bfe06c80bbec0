"""GPU: gradients of more rows than one axis of a grid has blocks for (nncf_amd.linear), against the plain product in 64 bits."""
import pytest
import torch

from tests.linear_utils import assert_within, make_weight, plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["relu", "swiglu", None])
def test_gradients_of_two_million_rows(act):
    from nncf_amd.linear import compressed_linear
    dtype, m, n, k = torch.bfloat16, 65536 * 32 + 7, 8, 32
    packed, dec = make_weight("int4_sym", 32, (n, k), dtype, seed=1)
    g = torch.Generator(device="cuda").manual_seed(2)
    width = n // 2 if act == "swiglu" else n
    x = torch.randn(m, k, device="cuda", generator=g).to(dtype).requires_grad_(True)
    b = torch.randn(n, device="cuda", generator=g).to(dtype).requires_grad_(True)
    dy = torch.randn(m, width, device="cuda", generator=g).to(dtype)
    out = compressed_linear(x, packed, dec, bias=b, activation=act)
    dx, db = torch.autograd.grad(out, (x, b), dy)
    ref = plain(x.detach(), dec(packed), b.detach(), act, None, dy)
    assert_within(out.detach(), ref[0], ref[1], "y")
    assert_within(dx, ref[2], ref[3], "dx")
    assert_within(db, ref[4], ref[5], "dbias")
    # the sums of a column: two million terms of either sign, where the bound above allows 2 m u of their magnitudes; in chunks
    # of 32 whose sums are added in four parts each addition is off by u of a partial sum, none of which is longer than m / 4 / 32
    # chunks: (32 / 4 + 3 + m / 128 + 4) u of the magnitudes
    z = x.detach().double() @ dec(packed).double().t() + b.detach().double()
    z = z.requires_grad_(True)
    from tests.linear_utils import act64
    dz = torch.autograd.grad(act64(z, act), z, dy.double())[0] if act else dy.double()
    u, half = 2.0 ** -24, torch.finfo(dtype).eps / 2
    if act == "relu":  # a sum whose sign is not settled may count or not
        ez = 2 * (k + 2) * u * (x.detach().double().abs() @ dec(packed).double().abs().t() + b.detach().double().abs())
        open_signs = torch.where(z.detach().abs() <= ez, dy.double().abs(), torch.zeros_like(z.detach())).sum(0)
    else:
        open_signs = torch.zeros(n, dtype=torch.float64, device="cuda")
    if act == "swiglu":
        return
    want = dz.sum(0)
    off = open_signs + (32 / 4 + 3 + m / 128 + 4) * u * dz.abs().sum(0)
    assert_within(db, want, off + half * (want.abs() + off))
