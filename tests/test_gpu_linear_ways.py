"""GPU: products with compressed weights at sizes where each way of computing them is taken (strips on the codes, tiles on the
codes, a decompressed copy; with and without blocks that share k), against the plain product in 64 bits."""
import pytest
import torch

from tests.linear_utils import FOUR, assert_within, make_weight, plain

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def _rows(m, k, dtype, seed):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return torch.randn(m, k, generator=g).to(dtype).cuda()


def _check(x, packed, dec, act=None, bias=None, residual=None):
    from nncf_amd.linear import compressed_linear
    got = compressed_linear(x, packed, dec, bias=bias, activation=act, residual=residual)
    y, by = plain(x, dec(packed), bias, act, residual)
    assert_within(got, y, by, (tuple(x.shape), act))
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 16, 33, 64, 65, 97, 128, 129, 200, 257, 520, 900])
@pytest.mark.parametrize("mode,gs,n,k", [("int4_sym", 128, 1000, 4096), ("int4_asym", 64, 518, 4160), ("nf4", 32, 640, 2080),
                                         ("mxfp4", 32, 1024, 2112), ("int8_asym", -1, 777, 2048), ("int8_sym", -1, 512, 4032),
                                         ("int4_asym", -1, 260, 4096), ("nf4", 64, 130, 8192), ("int4_asym", 32, 131, 2112)])
def test_every_way_by_rows(mode, gs, n, k, m, dtype):
    packed, dec = make_weight(mode, gs, (n, k), dtype, seed=m + n)
    _check(_rows(m, k, dtype, m), packed, dec)


@pytest.mark.parametrize("m", [3, 90, 200, 700])
@pytest.mark.parametrize("act", ["swiglu", "gelu", "silu", None])
@pytest.mark.parametrize("mode,gs,n,k", [("int4_asym", 128, 1032, 2048), ("mxfp4", 32, 518, 4096), ("int8_sym", -1, 640, 2048)])
def test_epilogue_where_blocks_share_k(mode, gs, n, k, act, m):
    dtype = torch.bfloat16
    packed, dec = make_weight(mode, gs, (n, k), dtype, seed=m)
    width = n // 2 if act == "swiglu" else n
    g = torch.Generator(device="cpu").manual_seed(m)
    bias, residual = torch.randn(n, generator=g).to(dtype).cuda(), torch.randn(m, width, generator=g).to(dtype).cuda()
    _check(_rows(m, k, dtype, m) * 0.1, packed, dec, act, bias, residual)


@pytest.mark.parametrize("act", ["swiglu", "gelu", None])
@pytest.mark.parametrize("m", [40, 130, 300])
@pytest.mark.parametrize("mode,gs,n,k", [("int4_sym", 64, 20000, 256), ("nf4", 32, 17666, 192), ("int8_asym", -1, 18000, 320)])
def test_tiles_that_fill_the_device(mode, gs, n, k, m, act):
    """Tiles enough that no blocks share k: the epilogue in the product's own kernel, the last tile ragged."""
    dtype = torch.float16
    packed, dec = make_weight(mode, gs, (n, k), dtype, seed=m)
    width = n // 2 if act == "swiglu" else n
    g = torch.Generator(device="cpu").manual_seed(m)
    bias, residual = torch.randn(n, generator=g).to(dtype).cuda(), torch.randn(m, width, generator=g).to(dtype).cuda()
    _check(_rows(m, k, dtype, m) * 0.1, packed, dec, act, bias, residual)


@pytest.mark.parametrize("m", [2, 100, 300])
def test_strided_and_misaligned_rows(m):
    """Rows further apart than they are long, rows that no vector load may touch, and results into the middle of a matrix."""
    from nncf_amd.linear import compressed_linear
    packed, dec = make_weight("int4_sym", 128, (1000, 4096), torch.bfloat16, seed=1)
    x = _rows(m, 4096, torch.bfloat16, m)
    want = compressed_linear(x, packed, dec)
    y, by = plain(x, dec(packed))
    assert_within(want, y, by)
    for pad, shift in ((8, 0), (64, 8), (3, 1), (5, 0)):
        wide = torch.empty(m, 4096 + pad, dtype=x.dtype, device="cuda")
        wide[:, shift:shift + 4096] = x
        assert torch.equal(compressed_linear(wide[:, shift:shift + 4096], packed, dec), want)


@pytest.mark.parametrize("m", [97, 257])
def test_train_where_the_forward_pass_runs_on_the_codes(m):
    """The slopes are kept by the kernel that joins the parts of k (or by the tiles' own): the gradients see them."""
    from nncf_amd.linear import compressed_linear
    dtype, n, k = torch.bfloat16, 520, 2048
    for mode, act in (("int4_asym", "gelu"), ("nf4", "swiglu"), ("int8_sym", "silu")):
        packed, dec = make_weight(mode, -1 if mode == "int8_sym" else 64, (n, k), dtype, seed=m)
        x = (_rows(m, k, dtype, m) * 0.1).requires_grad_()
        bias = torch.randn(n, generator=torch.Generator().manual_seed(m)).to(dtype).cuda().requires_grad_()
        y = compressed_linear(x, packed, dec, bias=bias, activation=act)
        dy = _rows(m, y.shape[-1], dtype, m + 1)
        y.backward(dy)
        ref = plain(x.detach(), dec(packed), bias.detach(), act, None, dy)
        assert_within(y.detach(), ref[0], ref[1], "y")
        assert_within(x.grad, ref[2], ref[3], "dx")
        assert_within(bias.grad, ref[4], ref[5], "dbias")


@pytest.mark.parametrize("mode", FOUR + ("int8_asym",))
@pytest.mark.parametrize("skew", ["even", "one", "edges"])
@pytest.mark.parametrize("gather,act", [(True, None), (False, "swiglu")])
def test_experts_on_tiles(mode, skew, gather, act):
    """Groups of 0, 1, 127, 128, 129 and several hundred rows over tiles of 128 and 256, rows behind the last group."""
    from nncf_amd.experts import expert_linear, route_experts
    dtype, experts, n, k = torch.bfloat16, 6, 516, 1024
    sizes = {"even": [110] * 6, "one": [0, 0, 640, 0, 3, 0], "edges": [127, 128, 129, 0, 1, 257]}[skew]
    tokens = sum(sizes) + 9
    logits = torch.full((tokens, experts), -8.0)
    at = 0
    for e, size in enumerate(sizes):
        logits[at:at + size, e] = 1.0
        at += size
    perm = torch.randperm(tokens, generator=torch.Generator().manual_seed(5))
    mask = torch.arange(tokens) < at
    r = route_experts(logits[perm].cuda(), 1, token_mask=mask[perm].cuda())
    off = r.offsets.tolist()
    assert [b - a for a, b in zip(off, off[1:])] == sizes
    packed, dec = make_weight(mode, -1 if mode == "int8_asym" else 32, (experts, n, k), dtype, seed=7)
    w = dec(packed)
    x = _rows(tokens, k, dtype, 3)
    y = expert_linear(x, packed, dec, r, gather=gather, activation=act)
    source = r.slots.long() if gather else torch.arange(tokens, device="cuda")
    for e in range(experts):
        if off[e] == off[e + 1]:
            continue
        want, by = plain(x[source[off[e]:off[e + 1]]], w[e], None, act)
        assert_within(y[off[e]:off[e + 1]], want, by, (e, sizes[e]))
    assert not y[off[-1]:].any()


def test_offsets_beyond_31_bits():
    """A stack whose codes, values and parameters lie more than 2^31 bytes and elements behind its start."""
    from nncf_amd import decompressors as D
    from nncf_amd.experts import expert_linear, route_experts
    dtype, experts, n, k = torch.bfloat16, 80, 8192, 8192
    codes = torch.randint(0, 256, (experts * n * k // 2, 1), dtype=torch.uint8, device="cuda")
    scale = (torch.rand(experts, n, k // 64, 1, device="cuda") * 0.02 + 0.002).half()
    dec = D.INT4SymmetricWeightsDecompressor(scale, compressed_weight_shape=(experts, n, k // 64, 64), result_shape=(experts, n, k),
                                             result_dtype=dtype)
    one = D.INT4SymmetricWeightsDecompressor(scale[-1], compressed_weight_shape=(n, k // 64, 64), result_shape=(n, k), result_dtype=dtype)
    w = one(codes.reshape(experts, -1)[-1].reshape(-1, 1))
    for tokens in (2, 150):
        logits = torch.zeros(tokens, experts, device="cuda")
        logits[:, -1] = 1
        x = _rows(tokens, k, dtype, tokens)
        y = expert_linear(x, codes, dec, route_experts(logits, 1))
        want, by = plain(x, w[:512])
        assert_within(y[:, :512], want, by)
        want, by = plain(x, w[-512:])
        assert_within(y[:, -512:], want, by)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["gelu", "silu", "swiglu"])
@pytest.mark.parametrize("m", [1, 60, 333])
def test_bias_gradient_is_rounded_once(m, act, dtype):
    """Between dy and dbias nothing is rounded to 16 bits: the slopes are those of the fp32 sums and are kept as they are.  With
    u = 2^-24: a sum z of K products is off by ez <= 2 (K + 2) u sum|x w| (and the bias), a slope by at most 1.2 ez and by 32 u
    (1 + |z|) of its arithmetic (swiglu: that of silu times the other half, which is off by its own ez), and m of them times dy
    are added up in fp32: 2 (m + 2) u of their magnitudes.  Then dbias is rounded, half a step."""
    from nncf_amd.linear import compressed_linear
    from tests.linear_utils import act64
    n, k, u, half = 320, 256, 2.0 ** -24, torch.finfo(dtype).eps / 2
    packed, dec = make_weight("int4_sym", 64, (n, k), dtype, seed=m)
    x, bias = _rows(m, k, dtype, m) * 0.3, _rows(1, n, dtype, m + 1)[0].requires_grad_()
    y = compressed_linear(x, packed, dec, bias=bias, activation=act)
    dy = _rows(m, y.shape[-1], dtype, m + 2)
    y.backward(dy)
    w, d = dec(packed).double(), dy.double()
    z = (x.double() @ w.t() + bias.detach().double()).requires_grad_()
    dz = torch.autograd.grad(act64(z, act), z, d)[0]
    z = z.detach()
    ez = 2 * (k + 2) * u * (x.double().abs() @ w.abs().t() + bias.detach().double().abs())
    if act == "swiglu":
        (a, b), (ea, eb) = z.chunk(2, -1), ez.chunk(2, -1)
        off = torch.cat((d.abs() * (1.2 * (ea * b.abs() + eb) + 32 * u * (1 + a.abs()) * b.abs()),
                         d.abs() * (1.2 * ea + 32 * u * (1 + a.abs()) * (1 + a.abs()))), -1)
    else:
        off = d.abs() * (1.2 * ez + 32 * u * (1 + z.abs()))
    off = off.sum(0) + 2 * (m + 2) * u * (dz.abs() + off).sum(0)
    want = dz.sum(0)
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    assert_within(bias.grad, want, off + half * (want.abs() + off) + tiny)


def test_a_call_leaves_nothing_allocated():
    """Without the collector of cycles: what a call and its gradients allocate is freed when its results are."""
    import gc
    from nncf_amd.experts import combine_experts, expert_linear, route_experts
    from nncf_amd.linear import compressed_linear
    dtype = torch.bfloat16
    one, many = make_weight("int4_sym", 64, (256, 512), dtype), make_weight("nf4", 32, (4, 256, 512), dtype)

    def step(m):
        x, bias = _rows(m, 512, dtype, m).requires_grad_(), torch.zeros(256, dtype=dtype, device="cuda", requires_grad=True)
        compressed_linear(x, *one, bias=bias, activation="gelu").sum().backward()
        logits = torch.randn(m, 4, device="cuda", requires_grad=True)
        r = route_experts(logits, 2)
        combine_experts(expert_linear(x, *many, r, activation="swiglu"), r).float().sum().backward()

    for m in (1, 100):
        step(m)
    gc.collect()
    gc.disable()
    try:
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        for m in (1, 100, 1, 100):
            step(m)
        torch.cuda.synchronize()
        assert torch.cuda.memory_allocated() == before
    finally:
        gc.enable()


@pytest.mark.parametrize("m", [4, 90, 300])
def test_a_captured_training_step_follows_its_inputs(m):
    """Forward and gradients in one graph: five replays with other inputs, eager work of the same operators between them, and a
    second graph of the same step captured beside the first."""
    from nncf_amd.experts import combine_experts, expert_linear, route_experts
    from nncf_amd.linear import compressed_linear
    dtype = torch.bfloat16
    one, many = make_weight("int4_asym", 64, (512, 512), dtype, seed=1), make_weight("mxfp4", 32, (4, 256, 512), dtype, seed=2)

    def step(x, bias, logits, dy):
        h = compressed_linear(x, *one, bias=bias, activation="gelu")
        r = route_experts(logits, 2)
        y = combine_experts(expert_linear(h, *many, r, activation="swiglu"), r)
        return (y,) + torch.autograd.grad(y, (x, bias, logits), dy)

    def inputs(seed):
        return [(_rows(m, 512, dtype, seed) * 0.1).requires_grad_(), _rows(1, 512, dtype, seed + 1)[0].requires_grad_(),
                _rows(m, 4, torch.float32, seed + 2).requires_grad_(), _rows(m, 128, dtype, seed + 3)]

    cases = [inputs(10 * s) for s in range(4)]
    want = [step(*c) for c in cases]
    for t in want[0]:
        assert bool(torch.isfinite(t).all())
    want = [[t.detach().clone() for t in w] for w in want]
    graphs = []
    for _ in range(2):
        static = [t.detach().clone().requires_grad_(t.requires_grad) for t in cases[0]]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*static)
        graphs.append((graph, static, out))
    for i in (1, 3, 0, 2, 2):
        for graph, static, out in graphs:
            with torch.no_grad():
                for t, c in zip(static, cases[i]):
                    t.copy_(c)
            graph.replay()
        step(*cases[(i + 1) % 4])  # eager work between the replays
        torch.cuda.synchronize()
        for graph, static, out in graphs:
            for a, b in zip(out, want[i]):
                assert torch.equal(a, b)


def test_two_graphs_replayed_at_once():
    """Each capture has its own workspace: replays on two streams at the same time give what each gives alone."""
    from nncf_amd.linear import compressed_linear
    packed, dec = make_weight("nf4", 64, (1024, 4096), torch.bfloat16, seed=4)
    xs = [_rows(m, 4096, torch.bfloat16, m) for m in (97, 200, 12)]
    want = [compressed_linear(x, packed, dec) for x in xs]
    graphs, outs = [], []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(compressed_linear(x, packed, dec))
        graphs.append((graph, torch.cuda.Stream()))
    for _ in range(5):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
