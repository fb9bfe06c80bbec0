"""GPU: a fused Linear under forward mode and function transforms answers as the Linear that it was."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from tests.linear_utils import make_weight

pytestmark = pytest.mark.gpu


def _pair():
    """(a compressed Linear, the same one fused)."""
    import copy
    from torch.nn.utils import parametrize
    from nncf_amd.linear import fuse_compressed_linears
    packed, dec = make_weight("int4_sym", 32, (48, 64), torch.bfloat16)
    torch.manual_seed(0)
    mod = torch.nn.Linear(64, 48, dtype=torch.bfloat16, device="cuda")
    mod.weight = torch.nn.Parameter(packed, requires_grad=False)
    parametrize.register_parametrization(mod, "weight", dec, unsafe=True)
    mod.requires_grad_(False)
    fused = copy.deepcopy(mod)
    assert fuse_compressed_linears(fused) == 1
    return mod, fused


def _x(m, seed):
    return torch.randn(m, 64, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()


def test_forward_mode():
    mod, fused = _pair()
    x, t = _x(5, 1), _x(5, 2)
    with fwd.dual_level():
        want, got = (fwd.unpack_dual(m(fwd.make_dual(x, t))) for m in (mod, fused))
        assert got.tangent is not None
        assert torch.equal(got.primal, want.primal) and torch.equal(got.tangent, want.tangent)
        assert fwd.unpack_dual(fused(x)).tangent is None  # (no tangent: the operator answers)


def test_function_transforms():
    """What the decompressor answers under a transform stays as it is (it takes no transform that wraps the tensors it makes)."""
    mod, fused = _pair()
    x, t = _x(6, 3), _x(6, 4)
    runs = (lambda m: torch.func.jvp(m, (x,), (t,)), lambda m: torch.func.grad(lambda v: m(v).float().square().sum())(x),
            lambda m: torch.vmap(m)(x.view(2, 3, 64)))
    for run in runs:
        try:
            want = run(mod)
        except RuntimeError:
            with pytest.raises(RuntimeError):
                run(fused)
        else:
            got = run(fused)
            assert torch.equal(got, want)


def test_products_of_hessians_by_vectors_need_the_library_product():
    """A gradient can be taken once; a second time it is refused, not wrong."""
    mod, fused = _pair()
    x = _x(3, 5).requires_grad_(True)
    g = torch.autograd.grad(fused(x).float().square().sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()
