"""GPU: calls from several host threads at once, and routings that leave every token out (nncf_amd.linear, nncf_amd.experts)."""
import threading

import pytest
import torch

from tests.linear_utils import make_weight

pytestmark = pytest.mark.gpu


def test_threads_call_at_once():
    """Four threads with streams of their own, every way of the product, forward and backward: what each gives alone."""
    from nncf_amd.linear import compressed_linear
    dtype = torch.float16
    weights = [make_weight(mode, -1 if mode.startswith("int8") else 32, (520, 1024), dtype, seed=i)
               for i, mode in enumerate(("int8_asym", "nf4", "mxfp4", "int4_asym"))]
    xs = [torch.randn(m, 1024, generator=torch.Generator().manual_seed(m)).to(dtype).cuda() for m in (1, 40, 130, 700)]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []
    start = threading.Barrier(4)

    def work(i):
        try:
            start.wait(timeout=60)
            with torch.cuda.stream(torch.cuda.Stream()):
                out = []
                for j in range(8):
                    w, x = weights[(i + j) % 4], xs[(i + j // 2) % 4].clone().requires_grad_(True)
                    y = compressed_linear(x, *w, activation="silu")
                    out.append((y.detach(), torch.autograd.grad(y, x, torch.ones_like(y))[0]))
                torch.cuda.current_stream().synchronize()
                got[i] = out
        except Exception as e:  # (a thread's exception would be lost)
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=100)
    assert not errors, errors
    for i in range(4):
        for j in range(8):
            w, x = weights[(i + j) % 4], xs[(i + j // 2) % 4].clone().requires_grad_(True)
            y = compressed_linear(x, *w, activation="silu")
            assert torch.equal(got[i][j][0], y.detach())
            assert torch.equal(got[i][j][1], torch.autograd.grad(y, x, torch.ones_like(y))[0])


@pytest.mark.parametrize("tokens", [1, 40, 300, 3000])
@pytest.mark.parametrize("mode", ["int4_sym", "int8_asym"])
def test_a_batch_of_padding_only(tokens, mode):
    """No token has an expert: zeros forward and backward, whatever the padded rows hold."""
    from nncf_amd.experts import combine_experts, expert_linear, route_experts
    dtype, nan = torch.bfloat16, float("nan")
    packed, dec = make_weight(mode, -1 if mode == "int8_asym" else 32, (6, 96, 192), dtype)
    logits = torch.full((tokens, 6), nan, device="cuda", requires_grad=True)
    r = route_experts(logits, 2, token_mask=torch.zeros(tokens, dtype=torch.bool, device="cuda"))
    for gather in (True, False):
        x = torch.full((tokens if gather else 2 * tokens, 192), nan, dtype=dtype, device="cuda", requires_grad=True)
        y = expert_linear(x, packed, dec, r, gather=gather, activation="swiglu")
        out = combine_experts(y, r)
        assert not y.any() and not out.any()
        dx, dl = torch.autograd.grad(out, (x, logits), torch.full_like(out, 2.0), retain_graph=True)
        assert not dx.any() and not dl.any()
        assert not torch.autograd.grad(y, x, torch.full_like(y, nan))[0].any()
