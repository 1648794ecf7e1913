"""Low-rank adapters: long sums.
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
