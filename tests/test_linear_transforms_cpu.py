"""CPU: inputs that carry a forward-mode tangent, or come from a function transform, are refused by the operators (a result
without its tangent would be a wrong derivative, silently) and handed back to the library product by a fused Linear."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from nncf_amd import _lib
from nncf_amd import decompressors as dcmp
from nncf_amd.errors import InternalError
from tests.test_linear_models_cpu import _AsOnGpu, _linear, _x, decompressed_on_the_cpu, reached  # noqa: F401


@pytest.fixture
def anywhere(monkeypatch):
    """The operators' host code with tensors that are on no GPU, up to the first call of the library, which fails the test."""
    def library():
        raise AssertionError("reached the library")
    monkeypatch.setattr(_lib, "require_gpu", lambda t, what: None)
    monkeypatch.setattr(_lib, "on_device_of", lambda t: __import__("contextlib").nullcontext())
    monkeypatch.setattr(_lib, "lib", library)


def _calls():
    from nncf_amd.experts import ExpertRouting, combine_experts, expert_linear, route_experts
    from nncf_amd.linear import compressed_linear
    dtype = torch.bfloat16
    dec = dcmp.INT8SymmetricWeightsDecompressor(torch.ones(8, 1), result_dtype=dtype)
    codes = torch.ones(8, 16, dtype=torch.int8)
    stack = dcmp.INT8SymmetricWeightsDecompressor(torch.ones(2, 8, 1), result_dtype=dtype)
    ints = torch.zeros(6, dtype=torch.int32)
    x = torch.ones(3, 16, dtype=dtype)

    def routing(weights=torch.ones(3, 2)):
        return ExpertRouting(weights, ints.view(3, 2), ints.view(3, 2), ints, ints[:3])

    stacked = torch.ones(2, 8, 16, dtype=torch.int8)
    return {"x": (x, lambda t: compressed_linear(t, codes, dec)),
            "bias": (torch.ones(8, dtype=dtype), lambda t: compressed_linear(x, codes, dec, bias=t)),
            "residual": (torch.ones(3, 8, dtype=dtype), lambda t: compressed_linear(x, codes, dec, residual=t)),
            "logits": (torch.ones(3, 2), lambda t: route_experts(t, 2)),
            "rows": (x, lambda t: expert_linear(t, stacked, stack, routing())),
            "answers": (torch.ones(6, 8, dtype=dtype), lambda t: combine_experts(t, routing())),
            "weights": (torch.ones(3, 2), lambda t: combine_experts(torch.ones(6, 8, dtype=dtype), routing(t)))}


@pytest.mark.parametrize("which", ["x", "bias", "residual", "logits", "rows", "answers", "weights"])
@pytest.mark.parametrize("grad", [False, True])
def test_a_tangent_is_refused(which, grad, anywhere):
    value, call = _calls()[which]
    with fwd.dual_level():
        dual = fwd.make_dual(value.clone().requires_grad_(grad), torch.ones_like(value))
        with pytest.raises(InternalError, match="forward-mode"):
            call(dual)
        with torch.no_grad(), pytest.raises(InternalError, match="forward-mode"):
            call(dual)
        with pytest.raises(AssertionError, match="reached the library"):  # without a tangent the level changes nothing
            call(value)


@pytest.mark.parametrize("which", ["x", "bias", "residual", "logits", "rows", "answers", "weights"])
def test_function_transforms_are_refused(which, anywhere):
    value, call = _calls()[which]
    for run in (lambda: torch.func.jvp(call, (value,), (torch.ones_like(value),)),
                lambda: torch.func.grad(lambda t: call(t).sum())(value), lambda: torch.vmap(call)(value[None])):
        with pytest.raises(InternalError, match="function transforms"):
            run()


@pytest.mark.parametrize("where", ["x", "bias"])
def test_a_fused_linear_hands_tangents_to_the_library_product(where, reached):  # noqa: F811
    from nncf_amd.linear import fuse_compressed_linears
    mod = _linear()
    with fwd.dual_level():
        x = _x()
        if where == "x":
            x = fwd.make_dual(x.as_subclass(_AsOnGpu), torch.ones_like(x).as_subclass(_AsOnGpu))
        else:
            bias = mod.bias.detach()
            del mod.bias
            mod.bias = fwd.make_dual(bias, torch.ones_like(bias))
            x = x.as_subclass(_AsOnGpu)
        want = fwd.unpack_dual(mod(x))
        fuse_compressed_linears(mod)
        got = fwd.unpack_dual(mod(x))
        assert got.tangent is not None and not reached
        assert torch.equal(got.primal.as_subclass(torch.Tensor), want.primal.as_subclass(torch.Tensor))
        assert torch.equal(got.tangent.as_subclass(torch.Tensor), want.tangent.as_subclass(torch.Tensor))


def _stand_ins(monkeypatch):
    """The operators' forward passes by plain values of the right shapes, so that their backward passes can be asked."""
    from nncf_amd import experts, linear
    monkeypatch.setattr(linear, "_forward", lambda x, w, *rest: (torch.zeros(x.shape[0], w.n, dtype=x.dtype), None))
    monkeypatch.setattr(experts, "_expert_forward", lambda x, w, slots, *rest: (torch.zeros(slots.shape[0], w.n, dtype=x.dtype), None))
    monkeypatch.setattr(experts, "_combine", lambda y, weights, places, dtype: torch.zeros(places.shape[0], y.shape[1], dtype=dtype))
    monkeypatch.setattr(experts, "_route", lambda logits, top_k, *rest: (torch.zeros(logits.shape[0], top_k), torch.zeros(21, dtype=torch.int32)))


@pytest.mark.parametrize("which", ["x", "bias", "logits", "rows", "answers", "weights"])
def test_a_tangent_of_the_incoming_gradient_is_refused(which, anywhere, monkeypatch):
    value, call = _calls()[which]
    _stand_ins(monkeypatch)
    leaf = value.clone().requires_grad_(True)
    out = call(leaf)
    out = out.weights if which == "logits" else out
    with fwd.dual_level():
        dout = fwd.make_dual(torch.ones_like(out).detach(), torch.ones_like(out).detach())
        with pytest.raises(InternalError, match="forward-mode"):
            torch.autograd.grad(out, leaf, dout)
