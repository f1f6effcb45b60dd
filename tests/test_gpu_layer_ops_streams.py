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


def norm_and_sort(be, seed):
    """A large backward whose column sums go through the workspace, a bias gradient and a sort that go through the scratch."""
    rows, cols, e = 65536, 1024, 64
    with torch.cuda.stream(be.stream):
        gen = torch.Generator(device=be.device).manual_seed(seed)
        from ferro_b200.backend import DeviceBuffer
        x, g, w = (DeviceBuffer(torch.randn(n, device=be.device, generator=gen)) for n in (rows * cols, rows * cols, cols))
        ids = DeviceBuffer(torch.randint(0, e, (rows,), device=be.device, generator=gen))

    def go():
        y, mean, rstd = be.layer_norm_stats_dev(x, w, None, rows, cols, 1e-5)
        dx, dw, db = be.layer_norm_backward_dev(g, w, rows, cols, x=x, mean=mean, rstd=rstd)
        _, bias = be.dropout_backward_dev(g, 0.3, 5, 6, rows, cols, want_dx=False, want_dbias=True)
        plan = be.moe_sort_dev(ids, rows, 1, e)
        return [dx.t, dw.t, db.t, bias.t, plan.place.t, plan.offsets.t]

    return go


def test_a_replaced_stream_keeps_order_and_shares_no_scratch(be):
    """Calls on the new stream while backwards on the old one are in flight, without a wait on the host: they read what the
    old stream wrote and disturb none of its partial sums."""
    first, second = norm_and_sort(be, 1), norm_and_sort(be, 2)
    want = [first(), second()]
    be.synchronize()
    home, away = be.stream, torch.cuda.Stream(device=be.device)
    for _ in range(3):
        got = [None, None]
        for _ in range(4):
            got[0] = first()
        ws, scratch = be._ws.data_ptr(), be._scratch.data_ptr()
        held = be._ws, be._scratch  # so that their addresses are not given out again
        x = got[0][0]
        be.stream = away
        assert be._ws is None and be._scratch is None
        got[1] = second()
        from ferro_b200.backend import BinaryKind, DeviceBuffer
        twice = be.binary_dev(BinaryKind.Add, DeviceBuffer(x), DeviceBuffer(x))  # written by the old stream
        assert be._ws.data_ptr() != ws and be._scratch.data_ptr() != scratch
        be.stream = home
        again = first()
        torch.cuda.synchronize()
        assert torch.equal(twice.t, 2 * want[0][0])
        for a, b in [(got[0], want[0]), (got[1], want[1]), (again, want[0])]:
            assert all(torch.equal(p, q) for p, q in zip(a, b))
        del held
    be.check_experts()


def test_a_bad_expert_seen_on_a_replaced_stream_is_reported(be):
    busy = norm_and_sort(be, 3)
    ids = be.alloc_i64_from_host([0, 1, 7, 1])
    for _ in range(40):
        busy()
    be.moe_sort_dev(ids, 4, 1, 4)
    be.stream = torch.cuda.Stream(device=be.device)
    with pytest.raises(Exception, match="assignment 2 "):
        be.check_experts()
    be.check_experts()  # said once
    # the first calls of a backend, on a stream set before anything else
    from ferro_b200.backend import CudaBackend
    b = CudaBackend(0)
    b.stream = torch.cuda.Stream(device=b.device)
    b.moe_sort_dev(b.alloc_i64_from_host([0, 9]), 2, 1, 4)
    with pytest.raises(Exception, match="assignment 1 "):
        b.check_experts()


def test_a_stream_set_within_a_capture(be):
    """The backend moved to a stream that is being captured, and back, with work of its own stream in flight: nothing is
    waited for across the capture's border, the graph has scratch of its own."""
    go = norm_and_sort(be, 4)
    want = go()
    be.synchronize()
    home, graph, side = be.stream, torch.cuda.CUDAGraph(), torch.cuda.Stream(device=be.device)
    with torch.cuda.graph(graph, stream=side):
        be.stream = side
        outs = go()
        be.stream = home
    assert be._ws is None and be._scratch is None
    eager = go()
    be.synchronize()
    for o in outs:
        o.zero_()
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and torch.equal(c, b) for a, b, c in zip(outs, want, eager))
    be.check_experts()


def test_a_bad_expert_seen_before_a_move_into_a_capture_is_reported(be):
    """A captured stream waits for nothing outside its graph: what the former stream still holds is kept in mind and waited
    for by the stream that follows."""
    busy = norm_and_sort(be, 5)
    ids = be.alloc_i64_from_host([0, 1, 7, 1])
    good = be.alloc_i64_from_host([0, 1, 2, 1])
    side, third = torch.cuda.Stream(device=be.device), torch.cuda.Stream(device=be.device)
    busy()
    be.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side, capture_error_mode="relaxed"):  # the eager calls below need memory
        for _ in range(40):
            busy()
        be.moe_sort_dev(ids, 4, 1, 4)  # on the backend's stream, outside the graph
        be.stream = side
        plan = be.moe_sort_dev(good, 4, 1, 4)
        be.stream = third
    with pytest.raises(Exception, match="assignment 2 "):
        be.check_experts()
    graph.replay()
    torch.cuda.synchronize()
    assert plan.place.t.tolist() == [0, 1, 3, 2]
    be.check_experts()
