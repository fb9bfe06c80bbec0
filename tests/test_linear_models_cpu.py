"""CPU: which modules of a compressed model `fuse_compressed_linears` takes over, and when their forward hands a call back.  The
decompressors run on the CPU here; `compressed_linear` is not reached (its arguments are on no GPU)."""
import copy

import pytest
import torch
from torch import nn
from torch.nn.utils import parametrize

from nncf_amd import decompressors as dcmp


@pytest.fixture(autouse=True)
def decompressed_on_the_cpu(monkeypatch):
    def decompress(codes, mode, n_groups, group_size, scale, zero_point, out_dtype, scale_kind=None):
        assert mode == "int8_sym"
        return (codes.to(torch.float16).view(n_groups, group_size) * scale.view(-1, 1)).to(out_dtype).flatten()
    monkeypatch.setattr(dcmp, "decompress", decompress)


def _compressed(mod, seed=0, cls=dcmp.INT8SymmetricWeightsDecompressor):
    """`mod`, an nn.Linear, with its weight as int8 codes behind a decompressor."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-128, 128, mod.weight.shape, dtype=torch.int8, generator=g)
    mod.weight = nn.Parameter(codes, requires_grad=False)
    dec = cls(torch.rand(codes.shape[0], 1, generator=g) * 0.01 + 0.001, result_dtype=torch.bfloat16)
    parametrize.register_parametrization(mod, "weight", dec, unsafe=True)
    return mod.requires_grad_(False)


def _linear(cls=nn.Linear, **kw):
    torch.manual_seed(0)
    return _compressed(cls(16, 8, dtype=torch.bfloat16, **kw))


class _Scaled(nn.Linear):
    def forward(self, x):
        return 2 * super().forward(x)


class _Renamed(nn.Linear):
    pass


def _x(rows=5):
    return torch.randn(rows, 16, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)


def test_a_subclass_with_its_own_forward_keeps_it():
    from nncf_amd.linear import fuse_compressed_linears
    model = nn.Sequential(_linear(_Scaled))
    want = model(_x())
    assert fuse_compressed_linears(model) == 0
    assert torch.equal(model(_x()), want)


def test_a_replaced_instance_forward_is_kept():
    from nncf_amd.linear import fuse_compressed_linears
    mod = _linear()
    before = mod.forward
    mod.forward = lambda x: before(x) + 1000
    want = mod(_x())
    assert fuse_compressed_linears(mod) == 0
    assert torch.equal(mod(_x()), want)


def test_linears_that_answer_as_linears_are_fused():
    from nncf_amd.linear import fuse_compressed_linears
    model = nn.Sequential(_linear(), _linear(_Renamed), _linear(_Scaled), nn.Linear(8, 8))
    assert fuse_compressed_linears(model) == 2
    assert fuse_compressed_linears(model) == 2  # once more: the same two
    assert fuse_compressed_linears(copy.deepcopy(model)) == 2


@pytest.mark.parametrize("cls", [nn.Linear, _Renamed])
def test_a_call_that_is_handed_back_gives_what_it_gave(cls):
    from nncf_amd.linear import fuse_compressed_linears
    mod = _linear(cls)
    want = mod(_x())
    assert fuse_compressed_linears(mod) == 1
    assert torch.equal(mod(_x()), want)  # (on the CPU: the library product)


class _AsOnGpu(torch.Tensor):
    is_cuda = property(lambda self: True)


class _Adapter(nn.Module):
    def forward(self, w):
        return w + 0.25


@pytest.fixture
def reached(monkeypatch):
    """Calls that reach `compressed_linear` are counted and answered by the plain product of the codes' decompressor alone."""
    from nncf_amd import linear
    calls = []

    def plain(x, packed, decompressor, bias=None, activation=None, residual=None):
        calls.append(1)
        return nn.functional.linear(x.as_subclass(torch.Tensor), decompressor(packed), bias)
    monkeypatch.setattr(linear, "compressed_linear", plain)
    return calls


def test_a_fused_linear_calls_the_product(reached):
    from nncf_amd.linear import fuse_compressed_linears
    mod = _linear()
    want = mod(_x())
    fuse_compressed_linears(mod)
    assert torch.equal(mod(_x().as_subclass(_AsOnGpu)), want) and len(reached) == 1


def test_a_parametrization_added_to_a_fused_weight_counts(reached):
    from nncf_amd.linear import fuse_compressed_linears
    mod = _linear()
    fuse_compressed_linears(mod)
    parametrize.register_parametrization(mod, "weight", _Adapter())
    x = _x()
    want = nn.functional.linear(x, mod.weight, mod.bias)
    assert torch.equal(mod(x.as_subclass(_AsOnGpu)).as_subclass(torch.Tensor), want) and not reached


def test_a_fused_linear_survives_the_loss_of_its_parametrization(reached):
    from nncf_amd.linear import fuse_compressed_linears
    mod = _linear()
    want = mod(_x())
    weight = mod.weight.detach().clone()
    fuse_compressed_linears(mod)
    mod._modules.pop("parametrizations")
    mod.__class__ = nn.Linear
    mod.weight = nn.Parameter(weight, requires_grad=False)
    assert torch.equal(mod(_x()), want) and not reached


def test_scales_that_were_cast_keep_the_library_product(reached):
    """`model.float()` casts the decompressor's scales, whose products the kernels do not make."""
    from nncf_amd.linear import fuse_compressed_linears, weight_dtype_of
    mod = _linear(bias=False)
    fuse_compressed_linears(mod)
    mod.float()
    want = mod(_x())
    assert torch.equal(mod(_x().as_subclass(_AsOnGpu)).as_subclass(torch.Tensor), want) and not reached
    plain = dcmp.INT8SymmetricWeightsDecompressor(torch.ones(8, 1))
    assert weight_dtype_of(plain) == torch.float16 and weight_dtype_of(plain.float()) == torch.float32


class _Doubled(dcmp.INT8SymmetricWeightsDecompressor):
    def forward(self, x):
        return 2 * super().forward(x)


class _Other(dcmp.BaseWeightsDecompressor):
    result_dtype = torch.bfloat16

    def __init__(self, scale, result_dtype):
        super().__init__()

    def forward(self, x):
        return x.to(torch.bfloat16)


@pytest.mark.parametrize("cls", [_Doubled, _Other])
def test_a_decompressor_with_a_forward_of_its_own_keeps_it(cls, reached):
    from nncf_amd.linear import fuse_compressed_linears
    torch.manual_seed(0)
    mod = _compressed(nn.Linear(16, 8, dtype=torch.bfloat16), cls=cls)
    want = mod(_x())
    assert fuse_compressed_linears(mod) == 0
    assert torch.equal(mod(_x().as_subclass(_AsOnGpu)).as_subclass(torch.Tensor), want) and not reached


def test_hooks_of_a_decompressor_run(reached):
    from nncf_amd.linear import fuse_compressed_linears
    mod = _linear()
    plain = mod(_x())
    fuse_compressed_linears(mod)
    handle = mod.parametrizations.weight[0].register_forward_hook(lambda m, args, out: 2 * out)
    want = nn.functional.linear(_x(), mod.weight, mod.bias)
    assert torch.equal(mod(_x().as_subclass(_AsOnGpu)).as_subclass(torch.Tensor), want) and not reached and not torch.equal(want, plain)
    handle.remove()
    assert torch.equal(mod(_x().as_subclass(_AsOnGpu)), plain) and len(reached) == 1


def test_the_product_refuses_a_decompressor_with_a_forward_of_its_own():
    from nncf_amd.errors import InternalError
    from nncf_amd.linear import packed_weight
    codes, x = torch.ones(8, 16, dtype=torch.int8), torch.ones(3, 16, dtype=torch.bfloat16)
    kind = type("_Named", (dcmp.INT8SymmetricWeightsDecompressor,), {})
    assert packed_weight(codes, kind(torch.ones(8, 1), torch.bfloat16), x, 2, "here").k == 16
    with pytest.raises(InternalError):
        packed_weight(codes, _Doubled(torch.ones(8, 1), torch.bfloat16), x, 2, "here")
