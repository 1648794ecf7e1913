"""Low-rank adapters beside a shared projection against their definition in 64 bits.

Bounds are per element and worst case: a sum of n products in fp32 is off by at most n * 2^-24 of the sum of the absolute products, a
rounding to the storage type by half a step (finfo.eps / 2 of the value). The rank-sized rows h and g are rounded once to the storage
type where the tensor cores multiply them; `half` stands for that rounding in 16 bits and for 0 in fp32.
    h = s A x:   dh = (C + 2) 2^-24 s |A||x| + half |h|
    y = W x + b + B h:   dy = (C + r + 2) 2^-24 (|W||x| + |b| + |B||h|) + |B| dh + eps/2 |y|
    dA = sum g x^T:   dg |x| + (rows + 1) 2^-24 |g||x| + eps/2 |dA|
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U = 2.0 ** -24
TINY = 2.0 ** -24      # the step of fp16 below its normal range


def reference(p, dy=None):
    """{name: (value, bound)} in 64 bits on the CPU."""
    dtype = p["x"].dtype
    eps = torch.finfo(dtype).eps / 2
    half = 0.0 if dtype == torch.float32 else eps
    tiny = TINY if dtype == torch.float16 else 0.0
    x, w, a, b = (p[n].detach().cpu().double() for n in ("x", "weight", "a", "b"))
    ids = p["ids"].cpu().flatten()
    x = x.reshape(-1, x.shape[-1])
    n, r, C = a.shape
    O = w.size(0)
    T = x.size(0)
    bias = p["bias"].detach().cpu().double() if p["bias"] is not None else torch.zeros(O, dtype=torch.float64)
    s = p["scaling"].cpu().double() if isinstance(p["scaling"], torch.Tensor) else torch.full((n,), float(p["scaling"]), dtype=torch.float64)
    rnd = lambda v, e: e + eps * (v.abs() + e) + tiny  # noqa: E731
    y, e_y = x @ w.t() + bias, (C + r + 2) * U * (x.abs() @ w.abs().t() + bias.abs())
    out = {}
    if dy is not None:
        dy = dy.cpu().double().reshape(T, O)
        dx, e_dx = dy @ w, (O + r + 2) * U * (dy.abs() @ w.abs())
        da, e_da, db, e_db = torch.zeros_like(a), torch.zeros_like(a), torch.zeros_like(b), torch.zeros_like(b)
    for e in range(n):
        t = torch.nonzero(ids == e).flatten()
        if not t.numel():
            continue
        h = s[e] * (x[t] @ a[e].t())
        dh = (C + 2) * U * s[e].abs() * (x[t].abs() @ a[e].abs().t()) + half * h.abs() + tiny
        y[t] += h @ b[e].t()
        e_y[t] += (C + r + 2) * U * (h.abs() @ b[e].abs().t()) + dh @ b[e].abs().t()
        if dy is not None:
            g = s[e] * (dy[t] @ b[e])
            dg = (O + 2) * U * s[e].abs() * (dy[t].abs() @ b[e].abs()) + half * g.abs() + tiny
            dx[t] += g @ a[e]
            e_dx[t] += (O + r + 2) * U * (g.abs() @ a[e].abs()) + dg @ a[e].abs()
            da[e], db[e] = g.t() @ x[t], dy[t].t() @ h
            e_da[e] = dg.t() @ x[t].abs() + (t.numel() + 1) * U * (g.abs().t() @ x[t].abs())
            e_db[e] = dy[t].abs().t() @ dh + (t.numel() + 1) * U * (dy[t].abs().t() @ h.abs())
    out["y"] = (y, rnd(y, e_y))
    if dy is not None:
        out["x"], out["a"], out["b"] = (dx, rnd(dx, e_dx)), (da, rnd(da, e_da)), (db, rnd(db, e_db))
        dw, dbias = dy.t() @ x, dy.sum(0)
        out["weight"] = (dw, rnd(dw, (T + 1) * U * (dy.abs().t() @ x.abs())))
        out["bias"] = (dbias, rnd(dbias, (T + 1) * U * dy.abs().sum(0)))
    return out


def check(name, got, want):
    v, bound = want
    got = got.detach().double().cpu().reshape(v.shape)
    assert torch.isfinite(got).all(), name
    worst = ((got - v).abs() - bound).max().item() if v.numel() else -1.0
    assert worst <= 0, "%s is off by %g more than the bound (largest bound %g)" % (name, worst, bound.max().item())


def problem(T, C, O, r, n, dtype, order="segments", bias=False, bare=0.0, scaling="tensor", seed=0):
    g = torch.Generator().manual_seed(seed + T + 3 * C + 5 * O + 7 * r + n)
    p = dict(x=torch.randn(T, C, generator=g).to(dtype).cuda(), weight=(torch.randn(O, C, generator=g) * C ** -0.5).to(dtype).cuda(),
             a=(torch.randn(n, r, C, generator=g) * C ** -0.5).to(dtype).cuda(), b=(torch.randn(n, O, r, generator=g) * r ** -0.5).to(dtype).cuda(),
             bias=torch.randn(O, generator=g).to(dtype).cuda() if bias else None)
    ids = torch.randint(0, n, (T,), generator=g)
    ids[torch.rand(T, generator=g) < bare] = -1
    if order == "segments":
        ids = torch.sort(ids).values.roll(T // 3)
    p["ids"] = ids.cuda()
    p["scaling"] = (torch.rand(n, generator=g) + 0.5).cuda() if scaling == "tensor" else scaling
    return p


def call(p):
    import scattermoe_b200 as sm
    return sm.adapter_linear(p["x"], p["weight"], p["a"], p["b"], p["ids"], scaling=p["scaling"], bias=p["bias"])


LEAVES = ("x", "weight", "a", "b", "bias")


def train(p, names=LEAVES, seed=1):
    names = [n for n in names if p[n] is not None]
    q = dict(p, **{n: p[n].clone().requires_grad_() for n in names})
    y = call(q)
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(seed)).to(y.dtype).cuda()
    grads = torch.autograd.grad(y, [q[n] for n in names], dy)
    return y, dy, dict(zip(names, grads))


def verify(p, names=LEAVES):
    y, dy, grads = train(p, names)
    want = reference(p, dy)
    check("y", y, want["y"])
    for n, v in grads.items():
        assert v.shape == p[n].shape and v.dtype == p[n].dtype
        check("gradient of " + n, v, want[n])


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("order", ["segments", "shuffled"])
@pytest.mark.parametrize("bias", [False, True])
def test_forward_and_gradients(dtype, order, bias):
    verify(problem(200, 192, 136, 16, 4, DT[dtype], order, bias, bare=0.1))


# one row, tiles of rows that end early, many adapters with one row each, ranks around the multiples of 16 and 64, widths that are no
# multiple of 8 (CUDA cores) or of a tile
@pytest.mark.parametrize("T,C,O,r,n", [
    (1, 64, 64, 16, 1), (1, 4096, 512, 16, 32), (2, 8, 8, 1, 2), (31, 256, 264, 8, 31), (32, 72, 520, 24, 3), (33, 1000, 200, 17, 5),
    (64, 128, 1000, 64, 64), (65, 136, 128, 65, 2), (127, 256, 256, 33, 127), (128, 512, 384, 32, 9), (129, 2048, 256, 128, 2),
    (300, 264, 776, 5, 70), (513, 128, 512, 256, 3), (1030, 320, 264, 16, 2), (700, 200, 123, 5, 3), (77, 33, 65, 3, 4)])
@pytest.mark.parametrize("dtype,order", [("bf16", "segments"), ("fp16", "shuffled"), ("fp32", "shuffled")])
def test_sizes(T, C, O, r, n, dtype, order):
    verify(problem(T, C, O, r, n, DT[dtype], order, bias=T % 2 == 1, bare=0.05))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("T", [5, 300])
def test_rows_without_adapter_and_adapters_without_rows(dtype, T):
    p = problem(T, 128, 192, 16, 6, DT[dtype], "shuffled")
    p["ids"][p["ids"] == 4] = 2
    p["ids"][0], p["ids"][1], p["ids"][2] = -1, 6, 1 << 40
    verify(p)
    _, _, grads = train(p)
    assert (grads["a"][4] == 0).all() and (grads["b"][4] == 0).all()
    p["ids"][:] = -1
    verify(p)
    _, _, grads = train(p)
    assert (grads["a"] == 0).all() and (grads["b"] == 0).all()


@pytest.mark.parametrize("T", [6, 260])
def test_an_adapter_that_is_not_a_number_stays_with_its_rows(T):
    """A row only meets its own adapter: Inf and NaN in another one, or in another row, do not reach it."""
    p = problem(T, 128, 160, 16, 3, torch.bfloat16, "shuffled", bare=0.2)
    want = call(p)
    p["a"][1], p["b"][2, 5] = float("nan"), float("inf")
    p["x"][3] = float("inf")
    got = call(p)
    keep = p["ids"] != 1
    keep[3] = False
    cols = torch.arange(160, device="cuda") != 5
    assert torch.equal(got[keep & (p["ids"] != 2)], want[keep & (p["ids"] != 2)])
    assert torch.equal(got[keep & (p["ids"] == 2)][:, cols], want[keep & (p["ids"] == 2)][:, cols])
    bare = (p["ids"] < 0) & keep
    assert torch.equal(got[bare], want[bare])


def test_gradients_of_a_subset():
    """Only what is asked for: a frozen projection, frozen adapters, a fixed input."""
    p = problem(150, 128, 96, 16, 3, torch.bfloat16, bias=True)
    for names in (("a", "b"), ("x",), ("b",), ("a",), ("weight",), ("bias",), ("x", "bias"), ("weight", "bias")):
        verify(p, names)


def test_gradients_against_differences():
    """fp32, central differences of a scalar of the output along random directions. The function is a polynomial of degree two in the
    adapters and linear in the rest, so the difference itself is exact; fp32 sums of about 40000 terms leave 1e-4 of their size."""
    p = problem(40, 24, 20, 4, 3, torch.float32, "shuffled", bias=True, bare=0.1)
    y, dy, grads = train(p)
    for n in LEAVES:
        v = torch.randn(p[n].shape, generator=torch.Generator().manual_seed(5)).cuda()
        f = [(call(dict(p, **{n: p[n] + s * v})).double() * dy.double()).sum() for s in (0.5, -0.5)]
        want, got = (f[0] - f[1]).item(), (grads[n].double() * v.double()).sum().item()
        scale = (grads[n].double() * v.double()).abs().sum().item()
        assert abs(want - got) <= 1e-4 * scale, (n, want, got)


def test_leading_shape_strides_scalars():
    p = problem(60, 64, 96, 8, 4, torch.bfloat16, "shuffled", bias=True, scaling=0.5)
    want = call(p)
    q = dict(p, x=p["x"].view(3, 20, 64), ids=p["ids"].view(3, 20).int(), scaling=torch.full((4,), 0.5, device="cuda", dtype=torch.bfloat16))
    assert torch.equal(call(q).view(60, 96), want)
    wide = torch.randn(60, 200, device="cuda").bfloat16()
    wide[:, 8:72] = p["x"]
    store = torch.randn(64, 104, device="cuda").bfloat16()
    store[:, 8:] = p["weight"].t()
    q = dict(p, x=wide[:, 8:72], weight=store[:, 8:].t(), a=p["a"].transpose(1, 2).contiguous().transpose(1, 2),
             b=p["b"].transpose(1, 2).contiguous().transpose(1, 2))
    y, dy, grads = train(q)
    ref = reference(p, dy)
    check("y", y, ref["y"])
    for n, v in grads.items():
        check(n, v, ref[n])
    odd = torch.randn(60, 65, device="cuda").bfloat16()
    odd[:, 1:] = p["x"]
    check("y", call(dict(p, x=odd[:, 1:])), reference(p)["y"])
    every_other = torch.zeros(120, 64, device="cuda").bfloat16()
    every_other[::2] = p["x"]
    assert torch.equal(call(dict(p, x=every_other[::2])), want)
    # an output gradient that is a broadcast view
    x = p["x"].clone().requires_grad_()
    (g,) = torch.autograd.grad(call(dict(p, x=x)).sum(), [x])
    check("x", g, reference(p, torch.ones(60, 96))["x"])


def test_bit_equal_from_call_to_call():
    p = problem(1500, 256, 256, 16, 5, torch.bfloat16, "shuffled", bias=True)
    y, _, grads = train(p)
    for _ in range(3):
        y2, _, g2 = train(p)
        assert torch.equal(y, y2) and all(torch.equal(grads[n], g2[n]) for n in grads)


def test_zero_rows():
    p = problem(4, 64, 96, 8, 3, torch.bfloat16)
    p = dict(p, x=p["x"][:0], ids=p["ids"][:0])
    y, _, grads = train(p, ("x", "a", "b"))
    assert y.shape == (0, 96) and grads["x"].shape == (0, 64)
    assert (grads["a"] == 0).all() and (grads["b"] == 0).all()


def test_streams_and_graphs():
    for T in (9, 400):
        ps = [problem(T + i, 128, 192, 16, 4, torch.bfloat16, "shuffled", seed=i) for i in range(2)]
        want = [call(p) for p in ps]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = [call(p) for p in ps]
        torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        graphs, outs = [], []
        for p in ps:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(call(p))
            graphs.append(graph)
        for _ in range(3):
            for graph in graphs:
                graph.replay()
        ps[0]["ids"].copy_(ps[0]["ids"].flip(0))
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], call(ps[0])) and torch.equal(outs[1], want[1])


def test_training_step_in_a_graph():
    """Forward and backward captured once and replayed on new data give the eager gradients."""
    p = problem(300, 128, 192, 16, 4, torch.bfloat16, "shuffled", bias=True)
    q = dict(p, **{n: p[n].clone().requires_grad_() for n in ("x", "a", "b")})
    dy = torch.randn(300, 192, device="cuda").bfloat16()
    leaves = [q[n] for n in ("x", "a", "b")]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(call(q), leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = torch.autograd.grad(call(q), leaves, dy)
    with torch.no_grad():
        q["x"].copy_(q["x"].flip(0))
    q["ids"].copy_(q["ids"].flip(0))
    graph.replay()
    torch.cuda.synchronize()
    want = torch.autograd.grad(call(q), leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_module():
    import scattermoe_b200 as sm
    m = sm.AdapterLinear(64, 96, 5, 8, bias=True, alpha=16).cuda().bfloat16()
    x = torch.randn(2, 7, 64, device="cuda").bfloat16()
    ids = torch.randint(-1, 5, (2, 7), device="cuda")
    # new adapters change nothing
    p = dict(x=x, weight=m.weight, a=m.lora_a, b=m.lora_b, bias=m.bias, ids=ids, scaling=m.scaling.float())
    check("y", m(x, ids), reference(p)["y"])
    with torch.no_grad():
        m.lora_b.normal_()
    m(x, ids).float().square().sum().backward()
    assert m.weight.grad is None and m.bias.grad is None and m.lora_a.grad is not None and m.lora_b.grad is not None


def test_a_decode_step_runs_both_operators():
    """A block as a server runs it: an adapted projection, the MoE layer with its router, an adapted shared expert beside it, on one
    padded batch; each stage against its definition on the stage's own input."""
    import scattermoe_b200 as sm
    from test_gpu_few_token import FIRST, SILU
    from test_gpu_few_token import check as check_layer
    from test_gpu_few_token import problem as layer_problem
    from test_gpu_few_token import reference as layer_reference
    T, d = 9, 128
    lay = layer_problem(T, d, 96, 8, 2, torch.bfloat16, FIRST)
    proj, shared = problem(T, d, d, 16, 4, torch.bfloat16, "shuffled", seed=1), problem(T, d, d, 8, 4, torch.bfloat16, "shuffled", seed=2)
    ids = torch.tensor([0, 1, 1, 3, 2, -1, 0, -1, -1], device="cuda")
    router = torch.randn(8, d, device="cuda").bfloat16()
    with torch.no_grad():
        x = call(dict(proj, x=lay["x"], ids=ids))
        y, gates, experts = sm.few_token_moe(x, router, lay["up"], lay["down"], 2, FIRST, SILU)
        z = call(dict(shared, x=x, ids=ids))
        out = y + z
    check("projection", x, reference(dict(proj, x=lay["x"], ids=ids))["y"])
    check_layer(y, *layer_reference(x, lay["up"], lay["down"], gates, experts, FIRST, SILU))
    check("shared expert", z, reference(dict(shared, x=x, ids=ids))["y"])
    assert out.shape == (T, d) and torch.isfinite(out).all()


@pytest.mark.parametrize("T", [20, 400])
def test_which_kernels_run(T, monkeypatch):
    """16-bit operands run on the tensor cores; forced onto the CUDA cores they give the same step; widths no 16-byte access can read
    are refused when the tensor cores are asked for."""
    from scattermoe_b200.kernels import ops
    p = problem(T, 192, 264, 24, 5, torch.float16, "shuffled", bias=True, bare=0.1)
    for path in ("tc", "simt"):
        monkeypatch.setattr(ops, "FORCE_PATH", path)
        call(p)
        assert ops.last_path_was_tensor_core() == (path == "tc")
        verify(p, ("x", "a", "b", "bias"))
    monkeypatch.setattr(ops, "FORCE_PATH", "tc")
    with pytest.raises(RuntimeError, match="no tensor-core kernel"):
        call(problem(T, 33, 64, 8, 3, torch.bfloat16))


def test_compiles():
    """torch.compile traces forward and backward as one graph."""
    import scattermoe_b200 as sm
    p = problem(200, 128, 96, 16, 3, torch.bfloat16, "shuffled", bias=True)
    q = dict(p, **{n: p[n].clone().requires_grad_() for n in ("x", "a", "b")})
    f = torch.compile(lambda x, a, b: sm.adapter_linear(x, p["weight"], a, b, p["ids"], scaling=p["scaling"], bias=p["bias"]),
                      backend="aot_eager", fullgraph=True)
    dy = torch.randn(200, 96, device="cuda").bfloat16()
    leaves = [q[n] for n in ("x", "a", "b")]
    got, want = f(*leaves), call(q)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, leaves, dy), torch.autograd.grad(want, leaves, dy)):
        assert torch.equal(a, b)


def test_refusals():
    import scattermoe_b200 as sm
    p = problem(4, 64, 96, 8, 3, torch.bfloat16)
    with pytest.raises(RuntimeError, match="constant"):
        call(dict(p, scaling=torch.ones(3, device="cuda", requires_grad=True)))
    with pytest.raises(RuntimeError, match="is on cpu"):
        call(dict(p, ids=p["ids"].cpu()))
    with pytest.raises(RuntimeError, match="are torch.bfloat16|is torch.float32"):
        call(dict(p, a=p["a"].float()))
    with pytest.raises(AssertionError):
        call(dict(p, ids=p["ids"][:3]))
    with pytest.raises(AssertionError, match="rank"):
        sm.adapter_linear(p["x"], p["weight"], torch.zeros(3, 257, 64, device="cuda").bfloat16(),
                          torch.zeros(3, 96, 257, device="cuda").bfloat16(), p["ids"])
