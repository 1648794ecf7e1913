"""The whole few-token layer and the adapters captured, replayed with new data, and run on two streams at once."""
import pytest
import torch

from test_gpu_adapters import call
from test_gpu_adapters import problem as adapter_problem
from test_gpu_few_token import FIRST, SILU, problem

pytestmark = pytest.mark.gpu


def layer(p, wr):
    import scattermoe_b200 as sm
    return sm.few_token_moe(p["x"], wr, p["up"], p["down"], 2, FIRST, SILU, router_bias=None)


def make(seed, order="out_in", T=24):
    p = problem(T, 256, 192, 16, 2, torch.bfloat16, FIRST, order, seed=seed)
    return p, torch.randn(16, 256, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()


@pytest.mark.parametrize("order", ["out_in", "in_out"])
def test_router_and_layer_replayed(order):
    """The router, the up- and the down-projection overlap: replays with new tokens give what calls on them give."""
    (p, wr), (q, wq) = make(0, order), make(1, order)
    layer(p, wr)
    graphs = []
    for a, w in ((p, wr), (q, wq)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(a, w)
        graphs.append((graph, out))
    for seed in range(4):
        for i, a in enumerate((p, q)):
            a["x"].copy_(torch.randn(24, 256, generator=torch.Generator().manual_seed(10 * seed + i)).bfloat16())
        for _ in range(3):
            for graph, _ in graphs:
                graph.replay()
        torch.cuda.synchronize()
        for (_, out), a, w in zip(graphs, (p, q), (wr, wq)):
            for got, want in zip(out, layer(a, w)):
                assert torch.equal(got, want)


def test_two_streams_at_once():
    """Calls on two streams share nothing: the results of both are those of calls one after the other."""
    (p, wr), (q, wq) = make(0), make(1, "in_out")
    a, b = adapter_problem(40, 256, 256, 16, 4, torch.bfloat16, "shuffled"), adapter_problem(300, 256, 256, 16, 4, torch.bfloat16, "shuffled")
    jobs = [lambda: layer(p, wr), lambda: (call(a),), lambda: layer(q, wq), lambda: (call(b),)]
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                results.append([job() for job in (jobs if i == 0 else jobs[::-1])][::1 if i == 0 else -1])
    torch.cuda.synchronize()
    for got in results:
        for g, w in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(g, w))


def test_more_than_one_device_is_not_assumed():
    """A call made while another stream of the device is current leaves the current device and stream as they were."""
    p, wr = make(2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        layer(p, wr)
        assert torch.cuda.current_stream() == s and torch.cuda.current_device() == p["x"].device.index
    torch.cuda.synchronize()
