"""GPU: expert routing, products grouped by expert and the weighted sum (nncf_amd.experts) against plain forms in 64 bits; the
bounds of the products are derived in tests/linear_utils.py."""
import pytest
import torch

from tests.linear_utils import assert_within, make_weight, plain

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def order(logits, topk, mask=None):
    """Experts by falling logit (NaN below everything, ties to the lower number) and the plan, with torch's stable sorts."""
    x = logits.double()
    tokens, experts = x.shape
    isnan = torch.isnan(x)
    key = torch.where(isnan, torch.full_like(x, float("inf")), -x)
    ids = torch.argsort(key, dim=1, stable=True)
    # -inf and NaN share the key +inf: put the NaN ones behind
    ids = torch.stack([torch.cat((r[~n[r]], r[n[r]])) for r, n in zip(ids, isnan)]) if bool(isnan.any()) else ids
    ids = ids[:, :topk]
    if mask is not None:
        ids = torch.where(mask[:, None], ids, torch.full_like(ids, -1))
    flat = ids.reshape(-1)
    perm = torch.argsort(torch.where(flat < 0, torch.full_like(flat, experts), flat), stable=True)
    counts = torch.bincount(flat[flat >= 0], minlength=experts)
    offsets = torch.cat((counts.new_zeros(1), counts.cumsum(0)))
    rows = torch.empty_like(perm)
    rows[perm] = torch.arange(perm.numel(), device=perm.device)
    rows = torch.where(flat < 0, torch.full_like(rows, -1), rows)
    slots = torch.where(torch.arange(perm.numel(), device=perm.device) < offsets[-1], perm, torch.full_like(perm, -1))
    return ids, rows.reshape(tokens, topk), slots, offsets


def check_plan(r, logits, topk, mask=None):
    ids, rows, slots, offsets = order(logits, topk, mask)
    for got, want in ((r.experts, ids), (r.rows, rows), (r.slots, slots), (r.offsets, offsets)):
        assert got.dtype == torch.int32 and torch.equal(got, want.int())
    return ids


def plain_weights(x64, ids, renormalize):
    chosen = x64.gather(1, ids.clamp(min=0))
    w = torch.softmax(chosen, 1) if renormalize else torch.softmax(x64, 1).gather(1, ids.clamp(min=0))
    return torch.where((x64 == -float("inf")).all(1, keepdim=True) | (ids < 0), torch.zeros_like(w), w)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,experts,topk", [(1, 1, 1), (1, 8, 2), (5, 8, 8), (513, 8, 2), (2049, 7, 3), (4100, 8, 8), (300, 9, 4),
                                                 (256, 32, 32), (257, 33, 5), (129, 64, 6), (5000, 64, 6), (77, 100, 8), (65, 128, 64),
                                                 (1000, 200, 8), (33, 300, 8), (700, 512, 2), (40, 1000, 64), (20000, 16, 1)])
def test_route(tokens, experts, topk, dtype):
    from nncf_amd.experts import route_experts
    g = torch.Generator(device="cpu").manual_seed(tokens + experts)
    logits = torch.randn(tokens, experts, generator=g).to(dtype).cuda()  # 16-bit types: many ties
    mask = (torch.rand(tokens, generator=g) < 0.7).cuda()
    x64 = logits.double()
    for m in (None, mask, torch.zeros_like(mask)):
        for renormalize in (True, False):
            r = route_experts(logits, topk, renormalize=renormalize, token_mask=m)
            ids = check_plan(r, logits, topk, m)
            want = plain_weights(x64, ids, renormalize)
            # differences of logits, exp (2 steps), a sum of up to `experts` terms and a quotient
            assert_within(r.weights, want, want * (2 * x64.abs().max() + experts + 16) * 2 * U)


def test_route_ties_infinities_and_nan():
    from nncf_amd.experts import route_experts
    inf, nan = float("inf"), float("nan")
    rows = [[1, 1, 1, 1], [0.0, -0.0, 0.0, -0.0], [-inf, 2, -inf, 1], [-inf, -inf, -inf, -inf], [nan, 1, 2, 3], [nan, nan, nan, nan],
            [nan, -inf, nan, -inf], [-inf, nan, 5, -inf], [-inf, -inf, 0, -inf], [3e38, -3e38, 3e38, 1]]
    x = torch.tensor(rows, dtype=torch.float32, device="cuda")
    for renormalize in (True, False):
        for topk in (1, 2, 3, 4):
            r = route_experts(x, topk, renormalize=renormalize)
            ids = check_plan(r, x, topk)
            want = plain_weights(x.double(), ids, renormalize)
            # fp32: a few steps of exp, a sum of four terms, a quotient (not-a-number in the plain form: here as well)
            torch.testing.assert_close(r.weights.double(), want, rtol=0, atol=1e-6, equal_nan=True)
            assert bool((r.weights[3] == 0).all())  # nothing to choose
    for v in (inf,):  # an infinite logit: its place is right, the weights of the row are not numbers
        r = route_experts(torch.tensor([[0, v, 1, 2]], device="cuda"), 2)
        assert r.experts.tolist() == [[1, 3]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,experts,topk", [(1, 8, 2), (700, 8, 2), (129, 33, 5), (300, 64, 6), (31, 200, 8), (9, 1000, 17)])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_gradient(tokens, experts, topk, renormalize, dtype):
    from nncf_amd.experts import route_experts
    g = torch.Generator(device="cpu").manual_seed(experts)
    logits = torch.randn(tokens, experts, generator=g).to(dtype).cuda()
    dw = torch.randn(tokens, topk, generator=g).cuda()
    mask = (torch.rand(tokens, generator=g) < 0.8).cuda()
    logits[0, : experts // 2] = -float("inf")
    for m in (None, mask):
        leaf = logits.clone().requires_grad_(True)
        r = route_experts(leaf, topk, renormalize=renormalize, token_mask=m)
        assert not r.experts.requires_grad and not r.offsets.requires_grad
        got = torch.autograd.grad(r.weights, leaf, dw)[0]
        assert got.dtype == dtype
        x = logits.double()
        ids = order(logits, topk, m)[0]
        w, dw64 = plain_weights(x, ids, renormalize), dw.double()
        dot, mag = (w * dw64).sum(1, keepdim=True), (w * dw64).abs().sum(1, keepdim=True)
        at = ids.clamp(min=0)
        if renormalize:
            want = torch.zeros_like(x).scatter(1, at, w * (dw64 - dot))
            size = torch.zeros_like(x).scatter(1, at, w * (dw64.abs() + mag))
        else:
            p = torch.softmax(x, 1)
            want = torch.zeros_like(x).scatter(1, at, w * dw64) - p * dot
            size = torch.zeros_like(x).scatter(1, at, (w * dw64).abs()) + p * mag
        if m is not None:
            want, size = want * m[:, None], size * m[:, None]
        rel = (2 * 5 + experts + 2 * topk + 32) * 2 * U  # weights as above, a sum over topk, a few products
        bound = size * rel + (want.abs() + size * rel) * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
        assert_within(got, want, bound)


def test_route_gradient_against_differences():
    from nncf_amd.experts import route_experts
    g = torch.Generator(device="cpu").manual_seed(3)
    x = torch.randn(50, 16, generator=g, dtype=torch.float64)
    v, dw = torch.randn(50, 16, generator=g, dtype=torch.float64), torch.randn(50, 4, generator=g, dtype=torch.float64)
    x32 = x.float().cuda().requires_grad_(True)
    ids = order(x.float(), 4)[0]
    for renormalize in (True, False):
        dx = torch.autograd.grad(route_experts(x32, 4, renormalize=renormalize).weights, x32, dw.float().cuda())[0].double().cpu()
        f = lambda t: (plain_weights(x.float().double() + t * v, ids, renormalize) * dw).sum()
        h = 1e-6
        diff = ((f(h) - f(-h)) / (2 * h)).item()
        assert abs((dx * v).sum().item() - diff) <= 1e-5 * (dx.abs() * v.abs()).sum().item()


def test_route_strided_logits_and_no_tokens():
    from nncf_amd.experts import combine_experts, expert_linear, route_experts
    g = torch.Generator(device="cpu").manual_seed(1)
    wide = torch.randn(90, 40, generator=g).cuda()
    for x in (wide[:, :8], wide[:, 3:11], wide[:, ::4], wide[:8].t()):
        a, b = route_experts(x, 2), route_experts(x.contiguous(), 2)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    r = route_experts(wide[:0, :8], 2)
    assert r.weights.shape == (0, 2) and r.slots.shape == (0,) and r.offsets.tolist() == [0] * 9
    packed, dec = make_weight("int4_sym", 32, (8, 48, 64), torch.bfloat16)
    y = expert_linear(torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"), packed, dec, r)
    assert y.shape == (0, 48) and combine_experts(y, r).shape == (0, 48)


def routing_of(tokens, experts, topk, seed=0, kind="spread", mask=False):
    from nncf_amd.experts import route_experts
    g = torch.Generator(device="cpu").manual_seed(seed)
    logits = torch.randn(tokens, experts, generator=g)
    if kind == "one":
        logits[:, 0] += 50  # every token to expert 0 first
    if kind == "last":
        logits[:, : experts // 2] -= 50  # experts without a token
    m = (torch.rand(tokens, generator=g) < 0.6).cuda() if mask else None
    return route_experts(logits.cuda(), topk, token_mask=m)


def grouped(x, w, r, topk, gather, act=None, dy=None):
    """The plain grouped product by experts in 64 bits with its bounds; rows without a slot are zero."""
    experts, n, k = w.shape
    rows = r.slots.numel()
    width = n // 2 if act == "swiglu" else n
    y = torch.zeros(rows, width, dtype=torch.float64, device="cuda")
    by = torch.zeros_like(y)
    dx, bdx = (torch.zeros(rows, k, dtype=torch.float64, device="cuda") for _ in range(2))
    ends, slots = r.offsets.tolist(), r.slots.long()
    for e in range(experts):
        lo, hi = ends[e], ends[e + 1]
        if lo < hi:
            xe = x[slots[lo:hi] // topk] if gather else x[lo:hi]
            out = plain(xe, w[e], None, act, None, None if dy is None else dy[lo:hi])
            y[lo:hi], by[lo:hi] = out[0], out[1]
            if dy is not None:
                dx[lo:hi], bdx[lo:hi] = out[2], out[3]
    return y, by, dx, bdx


CASES = [("int4_sym", 32, 4, 2, 48, 64), ("int4_asym", 128, 8, 2, 130, 256), ("nf4", 64, 8, 3, 64, 320), ("mxfp4", 32, 3, 1, 258, 96),
         ("int8_asym", -1, 5, 2, 34, 100), ("int8_sym", -1, 70, 2, 16, 64), ("int4_sym", 20, 2, 2, 6, 60)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens", [1, 5, 40, 333])
@pytest.mark.parametrize("mode,gs,experts,topk,n,k", CASES)
def test_expert_linear(mode, gs, experts, topk, n, k, tokens, dtype):
    from nncf_amd.experts import expert_linear
    packed, dec = make_weight(mode, gs, (experts, n, k), dtype, seed=tokens)
    w = dec(packed)
    g = torch.Generator(device="cpu").manual_seed(tokens)
    for kind, mask in (("spread", False), ("one", False), ("last", True)):
        r = routing_of(tokens, experts, topk, seed=n, kind=kind, mask=mask)
        for gather in (True, False):
            x = torch.randn(tokens if gather else tokens * topk, k, generator=g).to(dtype).cuda()
            y, by, _, _ = grouped(x, w, r, topk, gather)
            got = expert_linear(x, packed, dec, r, gather=gather)
            assert_within(got, y, by, (kind, gather))
            live = int(r.offsets[-1])
            assert bool((got[live:] == 0).all())


@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu", "swiglu", None])
@pytest.mark.parametrize("tokens", [3, 200])
@pytest.mark.parametrize("mode,gs,experts,topk,n,k", CASES[:4])
def test_expert_gradients(mode, gs, experts, topk, n, k, tokens, act):
    from nncf_amd.experts import expert_linear
    dtype = torch.bfloat16
    packed, dec = make_weight(mode, gs, (experts, n, k), dtype, seed=tokens)
    w = dec(packed)
    g = torch.Generator(device="cpu").manual_seed(tokens)
    width = n // 2 if act == "swiglu" else n
    r = routing_of(tokens, experts, topk, seed=n, mask=True)
    dy = torch.randn(tokens * topk, width, generator=g).to(dtype).cuda()
    for gather in (True, False):
        x = torch.randn(tokens if gather else tokens * topk, k, generator=g).to(dtype).cuda()
        y, by, dx, bdx = grouped(x, w, r, topk, gather, act, dy)
        x.requires_grad_(True)
        out = expert_linear(x, packed, dec, r, gather=gather, activation=act)
        assert_within(out.detach(), y, by)
        got = torch.autograd.grad(out, x, dy)[0]
        if gather:  # rows of a token are added in fp32; the bounds already hold one rounding each
            at = r.rows.long()
            pick = lambda t: torch.where((at >= 0)[:, :, None], t[at.clamp(min=0)], torch.zeros((), dtype=t.dtype, device="cuda")).sum(1)
            size = pick(dx.abs())
            dx, bdx = pick(dx), pick(bdx)
            bdx = bdx + size * topk * 2 * U + dx.abs() * torch.finfo(dtype).eps / 2
        assert_within(got, dx, bdx)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,experts,topk,n", [(1, 8, 2, 64), (5, 8, 2, 4096), (300, 8, 1, 100), (77, 16, 8, 33), (1000, 4, 3, 520),
                                                   (70000, 4, 2, 8)])
@pytest.mark.parametrize("mask", [False, True])
def test_combine(tokens, experts, topk, n, mask, dtype):
    from nncf_amd.experts import combine_experts
    r = routing_of(tokens, experts, topk, seed=tokens, mask=mask)
    g = torch.Generator(device="cpu").manual_seed(n)
    y = torch.randn(tokens * topk, n, generator=g).to(dtype).cuda()
    dout = torch.randn(tokens, n, generator=g).to(dtype).cuda()
    at = r.rows.long()
    has = (at >= 0)[:, :, None]
    picked = torch.where(has, y.double()[at.clamp(min=0)], torch.zeros((), dtype=torch.float64, device="cuda"))
    w = r.weights.double()[:, :, None]
    eps = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    want, size = (picked * w).sum(1), (picked * w).abs().sum(1)
    sum_err = size * 2 * (topk + 1) * U
    assert_within(combine_experts(y, r), want, sum_err + (want.abs() + sum_err) * eps + tiny)
    leaf, wl = y.clone().requires_grad_(True), r.weights.clone().requires_grad_(True)
    out = combine_experts(leaf, r._replace(weights=wl))
    dy, dw = torch.autograd.grad(out, (leaf, wl), dout)
    want_w = (picked * dout.double()[:, None]).sum(2)
    assert_within(dw, want_w, (picked * dout.double()[:, None]).abs().sum(2) * 2 * (n + 1) * U)
    want_y = torch.zeros_like(y, dtype=torch.float64)
    flat = at.reshape(-1)
    values = (dout.double()[:, None] * w).reshape(-1, n)
    want_y[flat[flat >= 0]] = values[flat >= 0]
    assert_within(dy, want_y, want_y.abs() * (2 * U + eps) + tiny)
    only = torch.autograd.grad(combine_experts(y, r._replace(weights=wl)), wl, dout)[0]
    assert torch.equal(only, dw)
    only = torch.autograd.grad(combine_experts(leaf, r), leaf, dout)[0]
    assert torch.equal(only, dy)


@pytest.mark.parametrize("mode,gs", [("mxfp4", 32), ("nf4", 32), ("int4_sym", 64), ("int8_asym", -1)])
@pytest.mark.parametrize("tokens", [1, 6, 150])
def test_layer_from_weights_to_gradients(mode, gs, tokens):
    """compress_experts and the whole layer, forward and backward, against the plain layer in 64 bits on the decompressed
    weights with the roundings between the operators where they are."""
    from nncf_amd.experts import compress_experts
    dtype, experts, hidden, inter, topk = torch.bfloat16, 6, 128, 192, 2
    torch.manual_seed(tokens)
    gu = (torch.randn(experts, 2 * inter, hidden, device="cuda") * 0.1).to(dtype)
    down = (torch.randn(experts, hidden, inter, device="cuda") * 0.1).to(dtype)
    layer = compress_experts(gu, down, __import__("nncf_amd").WeightCompressionConfig(mode, gs), topk)
    w1, w2 = layer.gate_up_decompressor(layer.gate_up), layer.down_decompressor(layer.down)
    assert w1.shape == gu.shape and w2.shape == down.shape
    h = torch.randn(tokens, hidden, device="cuda").to(dtype)
    logits = torch.randn(tokens, experts, device="cuda")
    mask = torch.arange(tokens, device="cuda") % 3 != 2
    hl, ll = h.clone().requires_grad_(True), logits.clone().requires_grad_(True)
    out = layer(hl, ll, mask)
    dout = torch.randn(tokens, hidden, device="cuda").to(dtype)
    dh, dl = torch.autograd.grad(out, (hl, ll), dout)
    h64, l64 = h.double().requires_grad_(True), logits.double().requires_grad_(True)
    ids = order(logits, topk)[0]
    wt = torch.softmax(l64.gather(1, ids), 1) * mask[:, None]
    z = torch.einsum("th,tjnh->tjn", h64, w1.double()[ids])
    a = torch.nn.functional.silu(z[..., :inter]) * z[..., inter:]
    ref = (torch.einsum("tji,tjhi->tjh", a, w2.double()[ids]) * wt[:, :, None]).sum(1)
    rh, rl = torch.autograd.grad(ref, (h64, l64), dout.double())
    eps = torch.finfo(dtype).eps / 2
    # roundings on the way: inner and rows forward, rows, inner, dz and z backward, the result: each half a step of values
    # whose size (norm) the products carry on; ten of them at the products' norms (rows of weights are no larger than the
    # largest singular value allows) stay below 40 half steps of the result's norm
    for got, want in ((out.detach(), ref.detach()), (dh, rh), (dl, rl)):
        assert (got.double() - want).norm() <= 40 * eps * want.norm()
    assert bool((out[~mask] == 0).all()) and bool((dh[~mask] == 0).all()) and bool((dl[~mask] == 0).all())


@pytest.mark.parametrize("tokens", [4, 300])
def test_layer_in_a_graph_with_other_routings(tokens):
    """A captured layer replayed with other tokens, whose groups have other sizes, against eager calls."""
    from nncf_amd.experts import compress_experts
    import nncf_amd
    torch.manual_seed(0)
    layer = compress_experts((torch.randn(8, 256, 128, device="cuda") * 0.1).bfloat16(), (torch.randn(8, 128, 128, device="cuda") * 0.1).bfloat16(),
                             nncf_amd.WeightCompressionConfig("mxfp4", 32), 2)
    hs = [torch.randn(tokens, 128, device="cuda").bfloat16() for _ in range(4)]
    ls = [torch.randn(tokens, 8, device="cuda") + torch.arange(8, device="cuda") * (i - 1.5) for i in range(4)]
    want = [layer(h, l) for h, l in zip(hs, ls)]
    h, l = hs[0].clone(), ls[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(h, l)
    for i in (2, 1, 3, 0, 3):
        h.copy_(hs[i])
        l.copy_(ls[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])
        assert torch.equal(layer(hs[i], ls[i]), want[i])


def test_refusals():
    from nncf_amd.errors import InternalError
    from nncf_amd.experts import combine_experts, compress_experts, expert_linear, route_experts
    import nncf_amd
    x = torch.zeros(6, 64, dtype=torch.bfloat16, device="cuda")
    logits = torch.zeros(6, 4, device="cuda")
    r = route_experts(logits, 2)
    packed, dec = make_weight("int4_sym", 32, (4, 48, 64), torch.bfloat16)
    for bad in (logits[0], logits.long(), logits[:, :0]):
        with pytest.raises((InternalError, ValueError)):
            route_experts(bad, 1)
    for k in (0, 5):
        with pytest.raises(ValueError):
            route_experts(logits, k)
    for mask in (torch.ones(5, dtype=torch.bool, device="cuda"), torch.ones(6, device="cuda"), torch.ones(6, dtype=torch.bool)):
        with pytest.raises(InternalError):
            route_experts(logits, 2, token_mask=mask)
    with pytest.raises(InternalError):
        expert_linear(x, packed, dec, r, gather=False)
    for bad in (x[:5], x[:, :32], x.float(), x[None]):
        with pytest.raises(InternalError):
            expert_linear(bad, packed, dec, r)
    with pytest.raises(InternalError):
        expert_linear(x, packed, dec, tuple(r))
    with pytest.raises(InternalError):
        expert_linear(x, packed, dec, r._replace(offsets=r.offsets[:-1]))
    with pytest.raises(InternalError):
        expert_linear(x, packed, dec, r._replace(slots=r.slots.long()))
    with pytest.raises(InternalError):
        expert_linear(x, *make_weight("int4_sym", 32, (48, 64), torch.bfloat16), r)
    for bad in (x, x[:, :0], torch.zeros(12, 64, device="cuda")):
        with pytest.raises(InternalError):
            combine_experts(bad, r)
    with pytest.raises(InternalError):
        compress_experts(torch.zeros(2, 64, 32, device="cuda").bfloat16(), torch.zeros(2, 32, 64, device="cuda").bfloat16(),
                         nncf_amd.WeightCompressionConfig("int4_sym", 32), 2)


def test_a_routing_with_foreign_numbers_reaches_no_foreign_memory():
    """Offsets, slots and rows outside the buffers are held to their ends; every access stays inside by the kernels' own checks."""
    from nncf_amd.experts import combine_experts, expert_linear, route_experts
    packed, dec = make_weight("int4_sym", 32, (4, 48, 64), torch.bfloat16)
    x = torch.randn(6, 64, device="cuda").bfloat16()
    r = route_experts(torch.randn(6, 4, device="cuda"), 2)
    for off in ([0, 3, -5, 100, 12], [0, 2 ** 31 - 1, 0, 0, 0], [-7, -7, -7, -7, -7]):
        bad = r._replace(offsets=torch.tensor(off, dtype=torch.int32, device="cuda"))
        assert expert_linear(x, packed, dec, bad).shape == (12, 48)
    bad = r._replace(slots=torch.full_like(r.slots, 2 ** 31 - 1), rows=torch.full_like(r.rows, 10 ** 6))
    y = expert_linear(x, packed, dec, bad)
    assert bool((combine_experts(y, bad) == 0).all())
    torch.cuda.synchronize()
