"""The few-token MoE layer on values that are not numbers, on small gates and on wide outputs. Bounds as in test_gpu_few_token.py."""
import pytest
import torch

from test_gpu_few_token import DT, FIRST, IDENT, OSS, PLAIN, RELU, SECOND, SILU, check, problem, reference, run, verify

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("order", ["out_in", "in_out"])
@pytest.mark.parametrize("layout,act", [(PLAIN, SILU), (PLAIN, RELU), (PLAIN, IDENT), (SECOND, SILU), (SECOND, RELU), (FIRST, SILU),
                                        (FIRST, RELU), (OSS, SILU)])
def test_nan_comes_out_where_it_went_in(dtype, order, layout, act):
    """A NaN in a token, a weight or a bias makes the rows that meet it NaN, whatever clamps and comparisons the activation has (the
    larger and the smaller of a NaN and a limit are NaN); the other rows keep their bits."""
    p = problem(12, 64, 64, 4, 2, DT[dtype], layout, order, bias=True)
    p["ids"] = torch.stack([torch.arange(12) % 4, (torch.arange(12) + 1) % 4], 1).cuda()      # tokens t with t % 4 in (1, 2) miss expert 0
    want = run(p, layout, act)
    assert torch.isfinite(want).all()
    met = ((p["ids"] == 0).any(1)).cpu()
    x = p["x"].clone()
    x[5, 3] = NAN
    got = run(dict(p, x=x), layout, act)
    keep = torch.arange(12) != 5
    assert got[5].isnan().all() and torch.equal(got[keep], want[keep])
    F = p["down"].size(1)
    # a hidden value's one or two columns, by weight and by bias
    for col in ([3] if layout == PLAIN else ([6, 7] if layout == OSS else [3, F + 3])):
        for name, at in (("up", (0, 9, col)), ("up_b", (0, col))):
            w = p[name].clone(memory_format=torch.preserve_format)
            w[at] = NAN
            assert w.stride() == p[name].stride()
            got = run(dict(p, **{name: w}), layout, act)
            assert got[met].isnan().all(), (name, col)
            assert torch.equal(got[~met], want[~met]), (name, col)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_infinities_meet_the_clamps(dtype):
    """The interleaved layout clamps an infinite gate or up column to the limit, as the definition does."""
    p = problem(6, 64, 32, 3, 2, DT[dtype], OSS, bias=True)
    for col in (6, 7):
        for v in (INF, -INF):
            q = dict(p, up_b=p["up_b"].clone())
            q["up_b"][:, col] = v
            if col == 6 and v < 0:      # the gate has no lower limit: -inf times sigmoid(-inf) is not a number
                assert run(q, OSS).isnan().all()
                continue
            # the reference's error terms follow |b|, which is infinite here: a bias far past the limit is the same layer
            far = dict(p, up_b=p["up_b"].clone())
            far["up_b"][:, col] = 1000.0 if v > 0 else -1000.0
            assert torch.equal(run(q, OSS), run(far, OSS))


@pytest.mark.parametrize("order", ["out_in", "in_out"])
@pytest.mark.parametrize("layout", [PLAIN, FIRST, OSS])
def test_small_gates(order, layout):
    """Gates of 2^-18 on outputs of ordinary size, in fp16. A hidden row that carried the whole gate would lie below fp16's normal range,
    where a rounding is off by 2^-25 whatever the value. It carries at least 1/16: the bound has half a step of the hidden value, and
    16 x 2^-25 where that is less."""
    p = problem(9, 96, 64, 5, 2, torch.float16, layout, order)
    p["down"] = p["down"] * 512
    p["gates"] = torch.full((9, 2), 2.0 ** -18, device="cuda")
    for _ in range(2):
        y, bound = reference(p["x"], p["up"], p["down"], p["gates"], p["ids"], layout, SILU)
        columns = p["down"].cpu().double().abs().sum(1)                      # (E, d_out)
        bound = bound + 2.0 ** -21 * (p["gates"].cpu().double().unsqueeze(2) * columns[p["ids"].cpu()]).sum(1)
        check(run(p, layout), y, bound)
        p["gates"] = p["gates"] * torch.rand(9, 2, generator=torch.Generator().manual_seed(3)).cuda()


@pytest.mark.parametrize("order", ["out_in", "in_out"])
@pytest.mark.parametrize("gate", [1 / 16, 0.1, 0.5])
def test_gates_leave_headroom(order, gate):
    """Hidden values past fp16's largest, 65504, whose gated values are not: finite and right, as the gate's power of two goes in front
    of the rounding."""
    p = problem(9, 96, 64, 5, 1, torch.float16, PLAIN, order)
    h = p["x"].cpu().double() @ p["up"].cpu().double()[0]
    p["x"] = (p["x"].float() * 80000 / h.abs().max().item() ** 0.5 / 256).half()
    p["up"] = (p["up"].float() * 256 / h.abs().max().item() ** 0.5).half()       # hidden values of up to about 80000
    p["down"] = p["down"] / 16
    p["gates"] = torch.full((9, 1), gate, device="cuda")
    y, bound = reference(p["x"], p["up"], p["down"], p["gates"], p["ids"], PLAIN, IDENT)
    check(run(p, PLAIN, IDENT), y, bound)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("order", ["out_in", "in_out"])
@pytest.mark.parametrize("d_out", [4736, 4744, 5120, 7168, 9480])
def test_wide_outputs(dtype, order, d_out):
    """More output columns than one tile per block of the down-projection."""
    p = problem(5, 64, 72, 4, 2, DT[dtype], SECOND, order, bias=True, d_out=d_out)
    p["ids"][3] = -1
    got = run(p, SECOND)
    assert (got[3] == 0).all()
    check(got, *reference(p["x"], p["up"], p["down"], p["gates"], p["ids"], SECOND, SILU, p["up_b"], p["down_b"]))


@pytest.mark.parametrize("order", ["out_in", "in_out"])
def test_experts_that_share_a_matrix(order, monkeypatch):
    """Broadcast views: one matrix for all experts (stride 0), one row of inputs for all tokens, one bias. The streaming kernels' tensor
    maps take no stride of zero, so the layer runs on CUDA cores and says so when the tensor cores are asked for."""
    from scattermoe_b200.kernels import ops
    p = problem(7, 64, 72, 5, 2, torch.bfloat16, FIRST, order, bias=True)
    q = dict(p, x=p["x"][:1].expand(7, 64), up_b=p["up_b"][:1].expand(5, -1), down_b=p["down_b"][:1].expand(5, -1))
    verify(q, FIRST)
    assert ops.last_path_was_tensor_core()
    for names in (("up",), ("down",), ("up", "down")):
        r = dict(q, **{n: q[n][:1].expand(5, -1, -1) for n in names})
        verify(r, FIRST)
        assert not ops.last_path_was_tensor_core()
    one = {n: p[n][:1].expand(1, -1, -1) for n in ("up", "down")}      # a single expert has no stride to speak of
    verify(dict(p, **one, up_b=None, down_b=None, ids=torch.zeros_like(p["ids"])), FIRST)
    assert ops.last_path_was_tensor_core()
    monkeypatch.setattr(ops, "FORCE_PATH", "tc")
    with pytest.raises(RuntimeError, match="no tensor-core kernel"):
        run(dict(q, up=q["up"][:1].expand(5, -1, -1)), FIRST)
