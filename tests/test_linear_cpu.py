"""CPU: argument checks of the products with compressed weights and of the expert routing, at the C entry points and in the host
code, without a GPU."""
import pytest
import torch


def test_entry_points_refuse_bad_arguments():
    from nncf_amd import _lib
    L = _lib.lib()
    B, N = 2, None

    def linear(dtype=B, ldx=64, m=4, n=48, k=64, mode=3, gs=32, act=0, x=N, codes=N):
        return L.nncf_amd_compressed_linear(x, dtype, ldx, m, n, k, codes, mode, gs, N, N, N, act, N, 0, N, 48, N, N, 0, N)

    assert linear(dtype=0) == _lib.ERR_DTYPE
    assert linear(mode=6) == _lib.ERR_MODE and linear(mode=-1) == _lib.ERR_MODE
    assert linear(gs=48) == _lib.ERR_GROUP_SIZE and linear(gs=0) == _lib.ERR_GROUP_SIZE
    assert linear(n=0) == _lib.ERR_BAD_ARG and linear(m=-1) == _lib.ERR_BAD_ARG and linear(act=9) == _lib.ERR_BAD_ARG
    assert linear(n=47, act=5) == _lib.ERR_BAD_ARG
    assert linear(n=3, k=3, gs=3) == _lib.ERR_BAD_ARG  # an odd number of nibbles
    assert linear() == _lib.ERR_BAD_ARG  # null weight
    assert linear(m=0) == _lib.OK  # no rows: nothing is read
    one = 4096
    full = lambda ws, nbytes: L.nncf_amd_compressed_linear(one, B, 64, 400, 48, 64, one, 3, 32, one, N, N, 0, N, 0, one, 48, N, ws, nbytes, N)
    assert full(N, 0) == _lib.ERR_WORKSPACE and full(one, 16) == _lib.ERR_WORKSPACE
    assert L.nncf_amd_compressed_linear(one, B, 63, 4, 48, 64, one, 3, 32, one, N, N, 0, N, 0, one, 48, N, N, 0, N) == _lib.ERR_BAD_ARG
    assert L.nncf_amd_compressed_linear(one, B, 64, 4, 48, 64, one, 2, 32, one, N, N, 0, N, 0, one, 48, N, N, 0, N) == _lib.ERR_BAD_ARG  # no zero points

    def expert(offsets=one, slots=N, sources=8, rows=8, topk=2, experts=4):
        return L.nncf_amd_expert_linear(one, B, 64, sources, slots, topk, offsets, experts, rows, 48, 64, one, 3, 32, one, N, 0, one, 48, N, N, 0, N)

    assert expert(offsets=N) == _lib.ERR_BAD_ARG and expert(sources=4) == _lib.ERR_BAD_ARG and expert(topk=0) == _lib.ERR_BAD_ARG
    assert expert(experts=0) == _lib.ERR_BAD_ARG and expert(rows=0, sources=0) == _lib.OK
    assert L.nncf_amd_linear_grad_input(one, B, 48, N, 2, 8, 48, 64, one, 3, 32, one, N, one, 64, 0, N, 0, N) == _lib.ERR_BAD_ARG
    assert L.nncf_amd_linear_grad_input(one, B, 48, N, 1, 8, 48, 64, one, 3, 32, one, N, one, 64, 0, N, 0, N) == _lib.ERR_WORKSPACE
    assert L.nncf_amd_activation_grad(one, B, 48, N, 8, 48, 1, one, 64, N, N, 0, N) == _lib.ERR_BAD_ARG  # no sums for the slope
    assert L.nncf_amd_activation_grad(one, B, 48, N, 8, 48, 0, N, 0, one, N, 0, N) == _lib.ERR_WORKSPACE
    assert L.nncf_amd_activation_grad_workspace(33, 48) == 2 * 48 * 4

    def route(dtype=0, tokens=4, experts=8, topk=2, ldl=8):
        return L.nncf_amd_route_experts(N, dtype, ldl, tokens, experts, topk, 1, N, N, N, N, N, N, N, 0, N)

    assert route(dtype=5) == _lib.ERR_DTYPE and route(topk=9) == _lib.ERR_BAD_ARG and route(topk=0) == _lib.ERR_BAD_ARG
    assert route(ldl=7) == _lib.ERR_BAD_ARG and route() == _lib.ERR_BAD_ARG
    assert route(experts=1025, ldl=1025) == _lib.ERR_UNSUPPORTED and route(experts=100, ldl=100, topk=65) == _lib.ERR_UNSUPPORTED
    assert L.nncf_amd_route_experts_workspace(0, 8, 2) == 0 and L.nncf_amd_route_experts_workspace(4, 8, 2) == 0
    assert L.nncf_amd_route_experts_workspace(100000, 8, 2) > 0
    assert L.nncf_amd_combine_experts(N, 0, 8, 8, N, N, 4, 2, 8, N, 0, N) == _lib.ERR_DTYPE
    assert L.nncf_amd_combine_experts(N, 2, 8, 8, N, N, 4, 2, 8, N, 2, N) == _lib.ERR_BAD_ARG
    assert L.nncf_amd_combine_experts(N, 2, 8, 0, N, N, 0, 2, 8, N, 2, N) == _lib.OK
    assert L.nncf_amd_combine_experts_grad(N, 2, N, 8, N, N, N, 4, 2, 8, N, N, N) == _lib.ERR_BAD_ARG


def test_host_code_refuses_cpu_tensors():
    from nncf_amd import errors
    from nncf_amd.experts import combine_experts, expert_linear, route_experts
    from nncf_amd.linear import compressed_linear
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    for call in (lambda: compressed_linear(x, x, None), lambda: route_experts(x, 2), lambda: expert_linear(x, x, None, None),
                 lambda: combine_experts(x, None)):
        with pytest.raises(errors.UnsupportedBackendError):
            call()


def test_rows_of_copies_only_where_strides_ask_for_it():
    from nncf_amd.linear import rows_of
    x = torch.arange(60.0).reshape(6, 10)
    t, ld = rows_of(x[:, 2:7], 5)
    assert ld == 10 and t.data_ptr() == x[:, 2:].data_ptr()
    for bad in (x[:, ::2], x.t()[:5].t(), x[:1, :5].expand(6, 5), x.t()[:, :5]):
        t, ld = rows_of(bad, 5)
        assert ld == 5 or bad.stride(1) == 1
        assert torch.equal(t, bad.reshape(-1, 5)) and t.stride(1) == 1 and (t.shape[0] == 1 or t.stride(0) >= 5)
    t, ld = rows_of(x[:1, :5], 5)
    assert ld == 5
    assert rows_of(torch.zeros(3, 0, 5), 5)[0].shape == (0, 5)


def test_fuse_leaves_plain_models_alone():
    from nncf_amd.linear import fuse_compressed_linears
    assert fuse_compressed_linears(torch.nn.Sequential(torch.nn.Linear(4, 4))) == 0
