"""NaN passes through the clamped interleaved SwiGLU and ReLU of the grouped path (stand-alone kernels and fused epilogues), forward and
backward, as it does in torch.clamp and torch.relu."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
PLAIN, SECOND, FIRST, OSS = 0, 1, 2, 3
SILU, RELU = 0, 3


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("layout,act", [(PLAIN, SILU), (PLAIN, RELU), (SECOND, RELU), (FIRST, RELU), (FIRST, SILU), (OSS, SILU)])
@pytest.mark.parametrize("F", [64, 33])
def test_stand_alone(dtype, layout, act, F):
    from scattermoe_b200 import activation
    g = torch.Generator().manual_seed(F)
    up = torch.randn(5, F if layout == PLAIN else 2 * F, generator=g).to(DT[dtype]).cuda()
    dh = torch.randn(5, F, generator=g).to(DT[dtype]).cuda()

    def step(up):
        up = up.detach().requires_grad_()
        h = activation.fused_activation(up, layout, act)
        return h.detach(), torch.autograd.grad(h, up, dh)[0]

    want_h, want_d = step(up)
    for half in range(1 if layout == PLAIN else 2):
        col = 3 if layout == PLAIN else (2 * 3 + half if layout == OSS else half * F + 3)
        other = None if layout == PLAIN else (2 * 3 + 1 - half if layout == OSS else (1 - half) * F + 3)
        bad = up.clone()
        bad[2, col] = float("nan")
        h, d = step(bad)
        assert h[2, 3].isnan()
        keep = torch.ones_like(h, dtype=torch.bool)
        keep[2, 3] = False
        assert torch.equal(h[keep], want_h[keep])
        keep = torch.ones_like(d, dtype=torch.bool)
        keep[2, col] = False
        if other is not None:      # the product's other factor is not a number, so its gradient is not
            assert d[2, other].isnan()
            keep[2, other] = False
        assert torch.equal(d[keep], want_d[keep])


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("layout,act", [(PLAIN, RELU), (FIRST, RELU), (SECOND, SILU), (OSS, SILU)])
def test_expert_mlp(dtype, layout, act):
    """One token with a NaN: its row of the output and of the input's gradient and its gates' gradients, no other row's."""
    import scattermoe_b200 as sm
    T, d, F, E, k = 300, 128, 96, 4, 2
    g = torch.Generator().manual_seed(layout)
    dt = DT[dtype]
    x = torch.randn(T, d, generator=g).to(dt).cuda()
    up = (torch.randn(E, F if layout == PLAIN else 2 * F, d, generator=g) * d ** -0.5).to(dt).cuda().transpose(1, 2)
    down = (torch.randn(E, d, F, generator=g) * F ** -0.5).to(dt).cuda().transpose(1, 2)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).cuda()
    gates = torch.rand(T, k, generator=g).to(dt).cuda()
    dy = torch.randn(T, d, generator=g).to(dt).cuda()

    def step(x, grad):
        x, p = x.detach().requires_grad_(grad), gates.detach().requires_grad_(grad)
        with torch.set_grad_enabled(grad):
            y = sm.expert_mlp(x, up, down, p, k, *sm.flatten_sort_count(ids, E), layout, act)
        return (y.detach(), *torch.autograd.grad(y, [x, p], dy)) if grad else (y,)

    bad = x.clone()
    bad[7, 5] = float("nan")
    keep = torch.arange(T) != 7
    for grad in (True, False):
        want, got = step(x, grad), step(bad, grad)
        assert got[0][7].isnan().all()
        for a, b in zip(got, want):
            assert torch.equal(a[keep], b[keep])
        if grad:
            assert got[2][7].isnan().all()
