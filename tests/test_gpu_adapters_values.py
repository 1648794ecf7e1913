"""Low-rank adapters: long sums, values that are not numbers in both directions, zero rows, and what the tensor-core switch covers.
Bounds as in test_gpu_adapters.py."""
import pytest
import torch

from test_gpu_adapters import LEAVES, U, call, check, problem, reference, train, verify

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("order", ["one", "two"])
def test_gradients_of_many_rows_in_fp32(order):
    """65536 rows whose products are all 1 + 2^-12: added one after the other in fp32 every product loses its 2^-12 once the sum has
    passed 2^13. Sums of up to 128 rows, added up, are off by at most (128 + rows / 128) 2^-24 of the sum."""
    T = 65536
    ids = torch.zeros(T, dtype=torch.int64, device="cuda")
    if order == "two":
        ids[::2] = 1
    n = int(ids.max()) + 1
    rows = T // n
    v = 1 + 2.0 ** -12
    p = dict(x=torch.full((T, 8), v, device="cuda"), weight=torch.zeros(4, 8, device="cuda"), a=torch.zeros(n, 1, 8, device="cuda"),
             b=torch.zeros(n, 4, 1, device="cuda"), bias=None, ids=ids, scaling=1.0)
    p["a"][:, 0, 0] = 1.0      # h = x[:, 0]
    p["b"][:, 0] = 1.0         # g = dy[:, 0]
    q = dict(p, a=p["a"].clone().requires_grad_(), b=p["b"].clone().requires_grad_())
    d_a, d_b = torch.autograd.grad(call(q), [q["a"], q["b"]], torch.ones(T, 4, device="cuda"))
    want, bound = rows * v, (128 + rows / 128) * U * rows * v
    for name, d in (("a", d_a), ("b", d_b)):
        assert (d.double() - want).abs().max().item() <= bound, (name, (d.double() - want).abs().max().item(), bound)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T", [40, 300])
@pytest.mark.parametrize("r,stored", [(16, "rank"), (16, "columns"), (12, "rank")])
def test_what_is_not_a_number_stays_with_its_adapter(dtype, T, r, stored):
    """Inf and NaN in one adapter's matrices or in one row of x or dy reach that adapter's rows and gradients alone, in both directions and
    however the matrices are stored (16-byte pieces of the rank, of the columns, or single elements)."""
    from test_gpu_adapters import DT
    p = problem(T, 128, 160, r, 4, DT[dtype], "shuffled", bare=0.1)
    p["ids"][:4] = torch.tensor([0, 1, 2, 3], device="cuda")
    dy = torch.randn(T, 160, generator=torch.Generator().manual_seed(2)).to(DT[dtype]).cuda()

    def step(p, dy):
        q = dict(p, b=p["b"].transpose(1, 2).contiguous().transpose(1, 2)) if stored == "columns" else dict(p)
        q = dict(q, **{n: q[n].detach().requires_grad_() for n in ("x", "a", "b")})
        y = call(q)
        return y.detach(), *torch.autograd.grad(y, [q["x"], q["a"], q["b"]], dy)

    want = step(p, dy)
    assert all(torch.isfinite(w).all() for w in want)
    others = p["ids"] != 2
    ads = torch.tensor([0, 1, 3], device="cuda")

    def same(got, rows):
        y, dx, da, db = got
        assert torch.equal(y[rows], want[0][rows]) and torch.equal(dx[rows], want[1][rows])
        assert torch.equal(da[ads], want[2][ads]) and torch.equal(db[ads], want[3][ads])

    for name in ("a", "b"):
        for v in (NAN, INF, -INF):
            q = dict(p, **{name: p[name].clone()})
            q[name][2, 3, 5] = v
            got = step(q, dy)
            same(got, others)
            mine = ~others
            if name == "a":      # every rank row of x is finite: h, y, dB of the adapter and column 5 of its dx are not
                assert not torch.isfinite(got[0][mine]).any(1).any() and not torch.isfinite(got[1][mine][:, 5]).any()
                assert torch.equal(got[1][mine][:, :5], want[1][mine][:, :5])
            else:                # column 3 of y, and all of dx and dA
                assert not torch.isfinite(got[0][mine][:, 3]).any() and torch.equal(got[0][mine][:, :3], want[0][mine][:, :3])
                assert not torch.isfinite(got[1][mine]).any(1).any() and not torch.isfinite(got[2][2]).any(1).all()
    for v in (NAN, INF):         # one row, of adapter 2
        q = dict(p, x=p["x"].clone())
        q["x"][2, 7] = v
        rows = torch.arange(T, device="cuda") != 2
        got = step(q, dy)
        assert torch.equal(got[0][rows], want[0][rows]) and torch.equal(got[1], want[1])
        assert torch.equal(got[2][ads], want[2][ads]) and torch.equal(got[3][ads], want[3][ads])
        bad = dy.clone()
        bad[2, 9] = v
        got = step(p, bad)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1][rows], want[1][rows])
        assert torch.equal(got[2][ads], want[2][ads]) and torch.equal(got[3][ads], want[3][ads])


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_zero_rows_with_every_gradient(dtype):
    from test_gpu_adapters import DT
    p = problem(4, 64, 96, 8, 3, DT[dtype], bias=True)
    p = dict(p, x=p["x"][:0], ids=p["ids"][:0])
    for names in (LEAVES, ("bias",), ("weight",), ("a",), ("weight", "bias")):
        y, _, grads = train(p, names)
        assert y.shape == (0, 96)
        for n, g in grads.items():
            assert g.shape == p[n].shape and (g == 0).all(), n


def test_asking_for_tensor_cores_covers_every_product(monkeypatch):
    """Forced onto the tensor cores, a step whose output gradient no 16-byte access can read is refused by each of its products (the
    product alone used to be), and one they can read runs; the shrink of up to 256 rows of an input-major A is a CUDA-core kernel by
    choice and is not refused."""
    from scattermoe_b200.kernels import ops
    p = problem(400, 192, 264, 24, 5, torch.float16, "shuffled", bias=True)
    odd = torch.randn(400, 265, device="cuda").half()[:, 1:]
    monkeypatch.setattr(ops, "FORCE_PATH", "tc")
    for T in (200, 400):
        verify(dict(p, x=p["x"][:T], ids=p["ids"][:T]))
    for name in ("x", "a", "b", "weight"):
        q = dict(p, **{name: p[name].clone().requires_grad_()})
        y = call(q)
        with pytest.raises(RuntimeError, match="no tensor-core kernel"):
            torch.autograd.grad(y, [q[name]], odd)
    monkeypatch.setattr(ops, "FORCE_PATH", None)
    for name in ("x", "a", "b", "weight"):
        q = dict(p, **{name: p[name].clone().requires_grad_()})
        (g,) = torch.autograd.grad(call(q), [q[name]], odd)
        check(name, g, reference(p, odd)[name])
