"""The few-token MoE layer against its definition in 64 bits.

Bounds are per element and worst case. A sum of n products in fp32 is off by at most n * 2^-24 of the sum of the absolute products; a
rounding to the storage type by half a step, finfo.eps / 2 of the value; the 16-bit kernels' fast exponential and reciprocal by 2^-19.
With U = |x| |W1| + |b1|, L = 1.13 >= the slope of every activation:
    du = (d + 2) 2^-24 U            dh = slope terms of du + (2^-19 + rounding) |h|
    dy = sum_j |g| (dh |W2| + (F + k + 4) 2^-24 (|h| |W2| + |b2|)) + eps/2 |y|
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
PLAIN, SECOND, FIRST, OSS = 0, 1, 2, 3
SILU, GELU, TANH, RELU, IDENT = 0, 1, 2, 3, 4
ALPHA, LIMIT = 1.702, 7.0
SLOPE = 1.13


def act64(code, z):
    if code == SILU:
        return z * torch.sigmoid(z)
    if code == GELU:
        return torch.nn.functional.gelu(z)
    if code == TANH:
        return torch.nn.functional.gelu(z, approximate="tanh")
    return z.clamp(min=0) if code == RELU else z


def reference(x, up, down, gates, ids, layout, act, up_b=None, down_b=None, alpha=ALPHA, limit=LIMIT):
    """(y, bound) in 64 bits on the CPU."""
    dtype = x.dtype
    half = torch.finfo(dtype).eps / 2
    fast = 0.0 if dtype == torch.float32 else 2.0 ** -19
    x, up, down, ids = x.cpu().double(), up.cpu().double(), down.cpu().double(), ids.cpu()
    T, k = ids.shape
    E, F, d_out = down.shape
    gates = torch.ones(T, k, dtype=torch.float64) if gates is None else gates.cpu().double()
    up_b = torch.zeros(E, up.size(2), dtype=torch.float64) if up_b is None else up_b.cpu().double()
    down_b = torch.zeros(E, d_out, dtype=torch.float64) if down_b is None else down_b.cpu().double()
    y, err = torch.zeros(T, d_out, dtype=torch.float64), torch.zeros(T, d_out, dtype=torch.float64)
    for e in range(E):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        if not t.numel():
            continue
        u = x[t] @ up[e] + up_b[e]
        du = (x.size(1) + 2) * 2.0 ** -24 * (x[t].abs() @ up[e].abs() + up_b[e].abs())
        if layout == PLAIN:
            h, dh = act64(act, u), SLOPE * du
        elif layout == OSS:
            g, dg = u[:, ::2].clamp(max=limit), du[:, ::2]
            v, dv = u[:, 1::2].clamp(-limit, limit) + 1, du[:, 1::2]
            a = g * torch.sigmoid(alpha * g)
            h, dh = v * a, SLOPE * dg * v.abs() + dv * a.abs()
        else:
            (g, v), (dg, dv) = u.chunk(2, 1), du.chunk(2, 1)
            if layout == SECOND:
                (g, v), (dg, dv) = (v, g), (dv, dg)
            h, dh = act64(act, g) * v, SLOPE * dg * v.abs() + dv * act64(act, g).abs()
        dh = dh + (fast + 2.0 ** -21 + (half if dtype != torch.float32 else 0.0)) * h.abs()
        if dtype == torch.float16:
            dh = dh + 2.0 ** -25          # below the smallest normal number the step no longer shrinks
        s = gates[t, j].unsqueeze(1)
        y.index_add_(0, t, s * (h @ down[e] + down_b[e]))
        err.index_add_(0, t, s.abs() * (dh @ down[e].abs() + (F + k + 4) * 2.0 ** -24 * (h.abs() @ down[e].abs() + down_b[e].abs())))
    return y, err + half * (y.abs() + err) + (2.0 ** -25 if dtype == torch.float16 else 0.0)


def check(got, y, bound):
    got = got.double().cpu()
    assert got.shape == y.shape and torch.isfinite(got).all()
    worst = ((got - y).abs() - bound).max().item() if got.numel() else -1.0
    assert worst <= 0, "off by %g more than the bound (%g)" % (worst, bound.max().item())


def weights(g, E, rows, cols, dtype, order):
    w = torch.randn((E, cols, rows) if order == "out_in" else (E, rows, cols), generator=g) * rows ** -0.5
    w = w.to(dtype).cuda()
    return w.transpose(1, 2) if order == "out_in" else w


def problem(T, d, F, E, k, dtype, layout=FIRST, order="out_in", bias=False, d_out=None, seed=0):
    g = torch.Generator().manual_seed(seed + 17 * T + d + F + E + k)
    n_up = F if layout == PLAIN else 2 * F
    d_out = d_out or d
    p = dict(x=torch.randn(T, d, generator=g).to(dtype).cuda(), up=weights(g, E, d, n_up, dtype, order),
             down=weights(g, E, F, d_out, dtype, order),
             ids=torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).cuda() if T else torch.zeros(0, k, dtype=torch.int64).cuda(),
             gates=torch.rand(T, k, generator=g).to(dtype).cuda())
    p["up_b"] = torch.randn(E, n_up, generator=g).to(dtype).cuda() if bias else None
    p["down_b"] = torch.randn(E, d_out, generator=g).to(dtype).cuda() if bias else None
    return p


def run(p, layout, act=SILU, **kw):
    import scattermoe_b200 as sm
    return sm.few_token_mlp(p["x"], p["up"], p["down"], p["gates"], p["ids"], layout, act, up_biases=p["up_b"],
                            down_biases=p["down_b"], **kw)


def verify(p, layout, act=SILU, **kw):
    got = run(p, layout, act, **kw)
    y, bound = reference(p["x"], p["up"], p["down"], p["gates"], p["ids"], layout, act, p["up_b"], p["down_b"], **kw)
    check(got, y, bound)
    return got


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("order", ["out_in", "in_out"])
@pytest.mark.parametrize("layout", [PLAIN, SECOND, FIRST, OSS])
def test_layouts_orders_types(dtype, order, layout):
    for bias in (False, True):
        verify(problem(7, 128, 96, 8, 2, DT[dtype], layout, order, bias), layout)


@pytest.mark.parametrize("act", [SILU, GELU, TANH, RELU, IDENT])
@pytest.mark.parametrize("layout", [PLAIN, FIRST])
def test_activation_functions(act, layout):
    for dtype in (torch.bfloat16, torch.float32):
        verify(problem(5, 64, 64, 4, 2, dtype, layout), layout, act)


# sizes around every boundary of the kernels: one token, groups of 8 and of 32 slots of one expert, K of one or many pieces,
# widths that end inside a tile, rows that are not 16-byte aligned (the CUDA-core kernels)
@pytest.mark.parametrize("T,d,F,E,k", [
    (1, 64, 64, 1, 1), (1, 1536, 512, 64, 8), (1, 2048, 768, 128, 8), (2, 8, 8, 2, 1), (3, 24, 40, 5, 3), (8, 256, 200, 3, 1),
    (9, 136, 72, 2, 2), (17, 520, 264, 4, 2), (33, 64, 48, 1, 1), (64, 192, 128, 2, 2), (65, 72, 56, 3, 3), (128, 128, 64, 1, 1),
    (128, 64, 64, 16, 8), (5, 1000, 1208, 12, 3), (16, 2880, 720, 8, 4), (2, 4096, 1792, 2, 2), (4, 50, 30, 3, 2), (11, 1001, 427, 13, 3),
    (1, 7, 3, 2, 2), (6, 4104, 136, 300, 8), (3, 64, 64, 1024, 8)])
@pytest.mark.parametrize("dtype,order", [("bf16", "out_in"), ("fp16", "in_out"), ("fp32", "out_in")])
def test_sizes(T, d, F, E, k, dtype, order):
    verify(problem(T, d, F, E, k, DT[dtype], OSS if order == "in_out" else SECOND, order, bias=True), OSS if order == "in_out" else SECOND)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_output_width_differs_and_no_gates(dtype):
    p = problem(6, 96, 80, 4, 2, DT[dtype], PLAIN, d_out=152)
    verify(p, PLAIN)
    p["gates"] = None
    verify(p, PLAIN)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("order", ["out_in", "in_out"])
def test_empty_rows_and_what_they_hold(dtype, order):
    """Ids outside [0, E) contribute nothing; a row without experts is zero even where its input is not a number."""
    p = problem(9, 64, 72, 5, 3, DT[dtype], FIRST, order, bias=True)
    p["ids"][2, 1] = -1
    p["ids"][4] = torch.tensor([5, -7, 1 << 40])
    p["ids"][8] = -1
    clean = p["x"].clone()
    p["x"][4], p["x"][8] = float("nan"), float("inf")
    got = run(p, FIRST)
    assert (got[4] == 0).all() and (got[8] == 0).all()
    y, bound = reference(clean, p["up"], p["down"], p["gates"], p["ids"], FIRST, SILU, p["up_b"], p["down_b"])
    check(got, y, bound)
    p["ids"][:] = -1
    assert (run(p, FIRST) == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_same_expert_twice_and_all_on_one(dtype):
    p = problem(40, 64, 64, 4, 2, DT[dtype], FIRST)
    p["ids"][:, 1] = p["ids"][:, 0]
    verify(p, FIRST)
    p["ids"][:] = 3
    got = verify(p, FIRST)
    assert torch.equal(got, run(p, FIRST))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_nan_stays_in_its_row(dtype):
    p = problem(12, 64, 64, 2, 2, DT[dtype], FIRST)
    want = run(p, FIRST)
    p["x"][5, 3] = float("nan")
    got = run(p, FIRST)
    assert got[5].isnan().all()
    keep = torch.arange(12, device="cuda") != 5
    assert torch.equal(got[keep], want[keep])


def test_bit_equal_from_call_to_call():
    p = problem(48, 256, 192, 16, 8, torch.bfloat16, FIRST)
    first = run(p, FIRST)
    for _ in range(5):
        assert torch.equal(first, run(p, FIRST))


def test_strides():
    """Views: a token slice, gates and ids that are columns of wider tensors, weights that are slices of a larger store."""
    p = problem(6, 64, 64, 4, 2, torch.bfloat16, FIRST)
    want = run(p, FIRST)
    wide = torch.randn(6, 200, device="cuda").bfloat16()
    wide[:, 64:128] = p["x"]
    store = torch.randn(9, 128, 96, device="cuda").bfloat16()
    store[2:6, :, 16:80] = p["up"].transpose(1, 2)
    q = dict(p, x=wide[:, 64:128], up=store[2:6, :, 16:80].transpose(1, 2),
             gates=torch.cat([p["gates"], p["gates"]], 1)[:, :2], ids=torch.stack([p["ids"], p["ids"]], 2)[..., 0])
    assert torch.equal(run(q, FIRST), want)
    q = dict(p, ids=p["ids"].int(), gates=p["gates"].t().contiguous().t())
    assert torch.equal(run(q, FIRST), want)
    q = dict(p, gates=p["gates"].float())
    assert torch.equal(run(q, FIRST), want)
    # odd offsets: rows and weights that no 16-byte access can read
    odd = torch.randn(6, 65, device="cuda").bfloat16()
    odd[:, 1:] = p["x"]
    q = dict(p, x=odd[:, 1:])
    y, bound = reference(p["x"], p["up"], p["down"], p["gates"], p["ids"], FIRST, SILU)
    check(run(q, FIRST), y, bound)


def test_zero_tokens():
    assert run(problem(0, 64, 64, 4, 2, torch.bfloat16, FIRST), FIRST).shape == (0, 64)


def test_streams_and_graphs():
    """Another stream than the tensors' own, and two captured calls replayed in turn with new inputs."""
    ps = [problem(5 + i, 128, 96, 8, 2, torch.bfloat16, FIRST, seed=i) for i in range(2)]
    want = [run(p, FIRST) for p in ps]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [run(p, FIRST) for p in ps]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for p in ps:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(p, FIRST))
        graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    ps[0]["x"].copy_(ps[0]["x"].flip(0))
    ps[0]["ids"].copy_(ps[0]["ids"].flip(0))
    graphs[0].replay()
    graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], run(ps[0], FIRST)) and torch.equal(outs[1], want[1])


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,d,F,E,k", [(1, 64, 64, 4, 2), (7, 200, 72, 33, 8), (24, 512, 64, 128, 8), (3, 65, 40, 5, 5),
                                       (2, 64, 64, 1024, 32), (128, 64, 32, 16, 1)])
@pytest.mark.parametrize("mode,renorm", [("softmax_topk", True), ("softmax_topk", False), ("topk_softmax", True)])
def test_whole_layer(dtype, T, d, F, E, k, mode, renorm):
    import scattermoe_b200 as sm
    p = problem(T, d, F, E, k, DT[dtype], FIRST)
    g = torch.Generator().manual_seed(T + E)
    wr = (torch.randn(E, d, generator=g) * d ** -0.5).to(DT[dtype]).cuda()
    br = torch.randn(E, generator=g).to(DT[dtype]).cuda()
    y, gates, ids = sm.few_token_moe(p["x"], wr, p["up"], p["down"], k, FIRST, SILU, mode=mode, renormalize=renorm, router_bias=br)
    x64, w64 = p["x"].cpu().double(), wr.cpu().double()
    z = x64 @ w64.t() + br.cpu().double()
    dz = ((d + 2) * 2.0 ** -24 * (x64.abs() @ w64.abs().t() + br.cpu().double().abs())).max(1, keepdim=True).values
    # the ids are the k largest in descending order: each selected logit is the j-th largest up to the error of the logits
    best = torch.sort(z, 1, descending=True).values[:, :k]
    ids_c = ids.cpu()
    assert ((torch.gather(z, 1, ids_c) - best).abs() <= 2 * dz).all()
    assert all(len(set(row.tolist())) == k for row in ids_c)
    top = torch.gather(z, 1, ids_c)
    ref = torch.softmax(top, 1) if (mode == "topk_softmax" or renorm) else torch.exp(top - torch.logsumexp(z, 1, keepdim=True))
    # a softmax value moves by at most a factor exp(+-2 dz); expf, the sum of up to E terms and the division add their roundings
    assert ((gates.cpu().double() - ref).abs() <= ref * (2.1 * dz + (E + 8) * 2.0 ** -24)).all()
    want, bound = reference(p["x"], p["up"], p["down"], gates, ids, FIRST, SILU)
    check(y, want, bound)


def test_router_ties_and_special_values():
    """Equal logits go to the lower id; -inf is never preferred; the same rules as route_topk."""
    import scattermoe_b200 as sm
    p = problem(3, 64, 64, 40, 4, torch.float32, FIRST)
    p["x"][:] = 0
    br = torch.zeros(40, device="cuda")
    br[7] = br[33] = 1.0
    br[0] = float("-inf")
    _, gates, ids = sm.few_token_moe(p["x"], torch.zeros(40, 64, device="cuda"), p["up"], p["down"], 4, FIRST, SILU, router_bias=br)
    assert ids.tolist() == [[7, 33, 1, 2]] * 3
    g2, ids2, _ = sm.route_topk(br.repeat(3, 1), 4)
    assert torch.equal(ids, ids2) and torch.allclose(gates, g2, rtol=2e-7, atol=0)


@pytest.mark.parametrize("bias", [False, True])
def test_module_decode_matches_forward(bias):
    """MLP.decode / GLUMLP.decode give what forward gives, up to the roundings of both."""
    import scattermoe_b200 as sm
    for m in (sm.mlp.GLUMLP(128, 96, 8, 2, bias=bias), sm.mlp.MLP(128, 96, 8, 2, bias=bias, activation=torch.nn.GELU())):
        m = m.cuda().bfloat16()
        x = torch.randn(2, 5, 128, device="cuda").bfloat16()
        p, idx = torch.topk(torch.softmax(torch.randn(2, 5, 8, device="cuda"), -1), 2)
        p = p.bfloat16()
        with torch.no_grad():
            a, b = m.decode(x, p, idx), m(x, p, idx)
        assert a.shape == b.shape
        layout, act = m.act_layout, (SILU if m.up_factor == 2 else GELU)
        y, bound = reference(x.view(10, 128), m.experts.weight.detach().permute(0, 2, 1), m.output_experts.weight.detach().permute(0, 2, 1),
                             p.view(10, 2), idx.view(10, 2), layout, act, m.experts.bias, m.output_experts.bias)
        check(a.view(10, 128), y, bound)


def test_which_kernels_run(monkeypatch):
    """16-bit operands run on the streaming kernels; forced onto the CUDA cores they give the same layer; what the streaming kernels
    cannot address is refused when they are asked for."""
    from scattermoe_b200.kernels import ops
    for order, layout in (("out_in", SECOND), ("in_out", FIRST), ("out_in", OSS), ("in_out", OSS), ("in_out", PLAIN)):
        p = problem(19, 192, 136, 6, 2, torch.float16, layout, order, bias=True, d_out=151 if order == "out_in" else 152)
        for path in ("tc", "simt"):
            monkeypatch.setattr(ops, "FORCE_PATH", path)
            verify(p, layout)
            assert ops.last_path_was_tensor_core() == (path == "tc")
    monkeypatch.setattr(ops, "FORCE_PATH", "tc")
    with pytest.raises(RuntimeError, match="no tensor-core kernel"):
        run(problem(3, 50, 30, 4, 2, torch.bfloat16, FIRST), FIRST)


def test_compiles():
    """torch.compile traces the calls as one graph each."""
    import scattermoe_b200 as sm
    p = problem(6, 64, 64, 4, 2, torch.bfloat16, FIRST)
    wr = torch.randn(4, 64, device="cuda").bfloat16()
    f = torch.compile(lambda x: sm.few_token_mlp(x, p["up"], p["down"], p["gates"], p["ids"], FIRST, SILU), backend="aot_eager", fullgraph=True)
    g = torch.compile(lambda x: sm.few_token_moe(x, wr, p["up"], p["down"], 2, FIRST, SILU), backend="aot_eager", fullgraph=True)
    with torch.no_grad():
        assert torch.equal(f(p["x"]), run(p, FIRST))
        for a, b in zip(g(p["x"]), sm.few_token_moe(p["x"], wr, p["up"], p["down"], 2, FIRST, SILU)):
            assert torch.equal(a, b)


def test_refusals():
    import scattermoe_b200 as sm
    p = problem(4, 64, 64, 4, 2, torch.bfloat16, FIRST)
    big = problem(129, 64, 64, 4, 2, torch.bfloat16, FIRST)
    with pytest.raises(AssertionError, match="at most 128 tokens"):
        run(big, FIRST)
    slots = problem(120, 64, 64, 16, 9, torch.bfloat16, FIRST)
    with pytest.raises(AssertionError, match="slots"):
        run(slots, FIRST)
    with pytest.raises(RuntimeError, match="no backward"):
        run(dict(p, x=p["x"].clone().requires_grad_()), FIRST)
    with torch.no_grad():
        run(dict(p, x=p["x"].clone().requires_grad_()), FIRST)
    with pytest.raises(RuntimeError, match="are on cpu|is on cpu"):
        run(dict(p, ids=p["ids"].cpu()), FIRST)
    with pytest.raises(RuntimeError, match="no backward"):
        sm.mlp.GLUMLP(64, 64, 4, 2).cuda()
        sm.few_token_mlp(p["x"].float(), p["up"].float().requires_grad_(), p["down"].float(), None, p["ids"], FIRST, SILU)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("order", ["out_in", "in_out"])
@pytest.mark.parametrize("T,k,F", [(1, 8, 64), (1, 32, 128), (2, 16, 8), (8, 4, 64), (8, 8, 128), (9, 3, 72), (16, 2, 64), (16, 8, 128)])
def test_few_tokens_that_name_an_expert_many_times(dtype, order, T, k, F):
    """Jobs of more slots than there are tokens beside short sums over K: a stage has to hold the rows of them all. Three experts, so
    that neighbouring stages are in flight; then one."""
    for d_out in (64, 2416):
        p = problem(T, 64, F, 40, k, DT[dtype], FIRST, order, d_out=d_out)
        g = torch.Generator().manual_seed(T * k + F)
        p["ids"] = torch.randint(3, 6, (T, k), generator=g).cuda()
        verify(p, FIRST)
        p["ids"][:] = 7
        got = verify(p, FIRST)
        assert torch.equal(got, run(p, FIRST))
