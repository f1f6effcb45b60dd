"""The layer operators and their scratch when the backend's stream is captured, or replaced by another."""
import numpy as np
import pytest
import torch

from ferro_b200 import kinds as K

pytestmark = pytest.mark.gpu


@pytest.fixture()
def be():
    from ferro_b200.backend import CudaBackend
    return CudaBackend(0)


@pytest.mark.parametrize("current", ["the captured stream", "another stream"])
def test_a_captured_call_takes_scratch_of_the_graph_whatever_stream_is_current(be, current):
    """What counts is whether the backend's own stream is captured: the graph's launches must not point into the scratch
    of eager calls, which a later, larger call gives back."""
    t, k, e, c = 20000, 4, 64, 96
    r = np.random.default_rng(1)
    ids, g = be.alloc_i64_from_host(r.integers(0, e, t * k)), be.alloc_from_host(r.standard_normal((t, c)))

    def go():
        plan = be.moe_sort_dev(ids, t, k, e)
        dx, db = be.dropout_backward_dev(g, 0.2, 1, 2, t, c, want_dbias=True)
        return [plan.place.t, plan.order.t, plan.offsets.t, dx.t, db.t]

    want = go()
    be.synchronize()
    eager, used = be._scratch.data_ptr(), []
    lib, real = be.lib, be.lib.fb_dropout_bwd

    class Seen:
        def __getattr__(self, name):
            return getattr(lib, name)

        def fb_dropout_bwd(self, *a):
            used.append(a[-2])
            return real(*a)

    be.lib = Seen()
    other = torch.cuda.Stream(device=be.device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=be.stream):
        if current == "another stream":
            with torch.cuda.stream(other):
                outs = go()
        else:
            outs = go()
    be.lib = lib
    assert used and used[0] != eager
    # a larger eager call drops the eager scratch; its memory is written over by whoever gets it next
    size = be._scratch.numel()
    big = be.alloc_from_host(np.zeros(1 << 24, np.float32))
    be.dropout_backward_dev(big, 0.5, 1, 2, 1 << 12, 1 << 12, want_dbias=True)
    be.synchronize()
    assert be._scratch.numel() > size
    for o in outs:
        o.zero_()
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_a_captured_reduction_takes_scratch_of_the_graph(be):
    """The same of the entries whose scratch comes from the shared workspace."""
    rows, cols = 4096, 1024
    r = np.random.default_rng(2)
    x, g, w = (be.alloc_from_host(r.standard_normal(n)) for n in (rows * cols, rows * cols, cols))

    def go():
        y, mean, rstd = be.layer_norm_stats_dev(x, w, None, rows, cols, 1e-5)
        dx, dw, db = be.layer_norm_backward_dev(g, w, rows, cols, x=x, mean=mean, rstd=rstd)
        return [y.t, dx.t, dw.t, db.t, be.sum_dim_dev(g, (rows, cols), 0).t, be.reduce_dev(K.RED_SUM, x).t]

    want = go()
    be.synchronize()
    eager = be._ws
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=be.stream):
        outs = go()
    assert be._ws is eager and be._ws_of_capture.data_ptr() != eager.data_ptr()
    eager.fill_(0xFF)
    for o in outs:
        o.zero_()
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    assert bool((eager == 0xFF).all())  # the graph wrote nothing there
