"""A context's work and another stream's on the same memory, ordered on the device."""
import numpy as np
import pytest
import torch

from rgpu_amd import gpu as G

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    g = G.Gpu(0)
    yield g
    g.close()


@pytest.mark.parametrize("default", [False, True])
def test_work_of_two_streams_in_turn(gpu, default):
    stream = torch.cuda.default_stream() if default else torch.cuda.Stream()
    n = 1 << 20
    with torch.cuda.stream(stream):
        big = torch.ones(4096, 4096, device="cuda")
        x, y, seen = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"), []
    torch.cuda.synchronize()
    wx, wy = gpu.wrap(x.data_ptr(), (n,), owner=x), gpu.wrap(y.data_ptr(), (n,), owner=y)
    for k in range(4):
        with torch.cuda.stream(stream):
            for _ in range(10):  # so that x is late
                big @ big
            x.fill_(k + 1.0)
        gpu.order_after(stream.cuda_stream)
        for _ in range(20):  # so that y is late
            gpu.map("scale", wx, wy, 2.0)
        gpu.map("offset", wy, wy, 1.0)
        gpu.order_before(stream.cuda_stream)
        with torch.cuda.stream(stream):
            seen.append(y + 1)
            x.fill_(-5.0)
            y.fill_(-7.0)
    torch.cuda.synchronize()
    for k, z in enumerate(seen):
        assert bool((z == 2 * (k + 1) + 2).all())


def test_a_captured_stream_is_refused(gpu):
    x = torch.zeros(64, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stream = torch.cuda.current_stream().cuda_stream
        x.add_(1)
        for call in (gpu.order_after, gpu.order_before):
            with pytest.raises(G.RtError) as e:
                call(stream)
            assert e.value.status == "RT_ERR_INVALID"
        x.add_(1)
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(x.cpu().numpy(), np.full(64, 2.0 * (k + 1), np.float32))
        gpu.sync()
