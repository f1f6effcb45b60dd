"""Rotary positions, dropout, gate and expert rows past 32-bit element numbers, in a capture that nothing warmed up, and
from two streams at once."""
import subprocess
import sys
import textwrap

import numpy as np
import pytest
import torch

import layer_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    from ferro_b200.backend import CudaBackend
    return CudaBackend(0)


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def filled(be, n, value):
    from ferro_b200.backend import DeviceBuffer
    with torch.cuda.stream(be.stream):
        return DeviceBuffer(torch.full((n,), value, device=be.device))


def part(be, buf, start, n):
    be.synchronize()
    return buf.t[start:start + n].cpu().numpy()


def test_dropout_past_32_bits(be):
    rows, cols, p, seed, off = 1047554, 4100, 0.25, 12345, 2 ** 33
    n = rows * cols
    assert n > 2 ** 32
    x = filled(be, n, 3.0)
    bias = np.arange(cols, dtype=np.float32)
    B = be.alloc_from_host(bias)
    be.dropout_dev(x, B, None, p, seed, off, rows, cols, out=x)
    for start in (0, 2 ** 31 - 2000, 2 ** 32 - 2000, n - 4000):
        start -= start % 4
        e = start + np.arange(4000, dtype=np.int64)
        keep = ref.drop_keep(4000, p, seed, off + start // 4)
        want = np.where(keep, (3.0 + bias[e % cols].astype(np.float64)) / 0.75, 0)
        assert (np.abs(part(be, x, start, 4000) - want) <= 4 * ref.EPS * np.abs(want)).all(), start
    g = x
    with torch.cuda.stream(be.stream):
        g.t.fill_(1.0)
    dx, db = be.dropout_backward_dev(g, p, seed, off, rows, cols, want_dbias=True, dx=g)
    for start in (0, 2 ** 32 - 2000, n - 4000):
        start -= start % 4
        keep = ref.drop_keep(4000, p, seed, off + start // 4)
        assert ((part(be, dx, start, 4000) != 0) == keep).all(), start
    kept = be.copy_to_host(db).astype(np.float64) * 0.75 / rows  # share of a column's elements that stay
    assert np.abs(kept - 0.75).max() < 6 * np.sqrt(0.25 * 0.75 / rows)  # six standard deviations, 4100 columns


def test_rope_past_32_bits_in_place(be):
    s, h, d = 1048577, 32, 128
    n = s * h * d
    assert n > 2 ** 32
    x = filled(be, n, 1.0)
    for layout in ("half", "interleaved"):
        plan = be.rope_plan(d, layout=layout)
        with torch.cuda.stream(be.stream):
            x.t.fill_(1.0)
        be.rope_dev(x, (1, s, h, d), plan, start=7, out=x)
        for t in (0, s // 2, s - 1):
            ang = ref.rope_angles(np.array([[t + 7]]), ref.rope_theta(d))
            one = np.ones((1, 1, h, d))
            got = part(be, x, t * h * d, h * d).reshape(1, 1, h, d)
            assert (np.abs(got - ref.rope(one, ang, layout)) <= ref.rope_bound(one, d, layout)).all(), (layout, t)


def test_rows_past_32_bits(be):
    from ferro_b200.backend import MoePlan
    cols, slots = 2 ** 30 + 4, 5
    x = filled(be, 2 * cols, 2.0)
    with torch.cuda.stream(be.stream):
        x.t[cols:].fill_(3.0)
    xs = filled(be, slots * cols, 9.0)
    plan = MoePlan(be.alloc_i64_from_host([4, 0]), None, None, 2, 1, slots)
    be.moe_dispatch_dev(x, plan, cols, out=xs)
    for row, want in ((0, 3.0), (1, 9.0), (3, 9.0), (4, 2.0)):
        for at in (0, cols - 1000):
            assert (part(be, xs, row * cols + at, 1000) == want).all(), row
    w = be.alloc_from_host([0.5, 2.0])
    be.moe_combine_dev(xs, w, plan, cols, out=x)
    for row, want in ((0, 1.0), (1, 6.0)):
        for at in (0, cols - 1000):
            assert (part(be, x, row * cols + at, 1000) == want).all(), row
    dys, dw = be.moe_combine_backward_dev(x, xs, w, plan, cols, dys=xs)
    assert (part(be, dys, 4 * cols + cols - 1000, 1000) == 0.5).all() and (part(be, dys, 0, 1000) == 12.0).all()
    got = be.copy_to_host(dw)
    # sums of 2^30 equal terms: at most cols / 256 + 8 additions deep in f32
    assert abs(got[0] / (2.0 * cols) - 1) < (cols / 256 + 8) * ref.EPS and abs(got[1] / (18.0 * cols) - 1) < (cols / 256 + 8) * ref.EPS
    be.moe_dispatch_backward_dev(xs, plan, cols, out=x)
    assert (part(be, x, cols - 500, 1000) == np.r_[np.full(500, 0.5), np.full(500, 12.0)]).all()


def test_gate_past_32_bits(be):
    t, e, k = 4194400, 1024, 2
    assert t * e > 2 ** 32
    l = filled(be, t * e, 0.0)
    with torch.cuda.stream(be.stream):
        v = l.t.view(t, e)
        v[-1, 700], v[-1, 3] = 5.0, 4.0
        v[-2].fill_(-float("inf"))
        v[t // 2, 1023] = 1.0
    w, ids = be.moe_gate_dev(l, t, e, k)
    got = part(be, ids, 0, k * t).reshape(t, k)
    assert got[-1].tolist() == [700, 3] and got[-2].tolist() == [-1, -1] and got[t // 2].tolist() == [1023, 0] and got[5].tolist() == [0, 1]
    dl = be.moe_gate_backward_dev(filled(be, t * k, 0.0), l, w, ids, t, e, k, renorm=False, dlogits=filled(be, t * e, 7.0))
    assert (part(be, dl, t * e - 4096, 4096) == 0).all() and (part(be, dl, 2 ** 32 - 2048, 4096) == 0).all()


def test_sort_of_many_assignments(be):
    from ferro_b200.backend import DeviceBuffer
    n, e = 3 * 2 ** 24 + 5, 200
    gen = torch.Generator(device=be.device).manual_seed(3)
    with torch.cuda.stream(be.stream):
        ids = torch.randint(-1, e, (n,), device=be.device, generator=gen)
        key = torch.where(ids < 0, e, ids)
        want = torch.sort(key, stable=True)[1]
        total = int((ids >= 0).sum())
    plan = be.moe_sort_dev(DeviceBuffer(ids), n, 1, e)
    be.synchronize()
    assert int(plan.offsets.t[-1]) == total
    assert torch.equal(plan.order.t[:total], want[:total])
    assert torch.equal(plan.place.t[want[:total]], torch.arange(total, device=be.device))
    assert bool((plan.place.t[ids < 0] == -1).all())


def test_first_calls_inside_a_capture():
    """Nothing of the library has run in the process before the capture: attribute calls and module loading happen inside
    it, the replay equals eager calls."""
    code = textwrap.dedent("""
        import torch
        from ferro_b200.backend import CudaBackend, DeviceBuffer
        be = CudaBackend(0)
        t, e, k, c = 5000, 1024, 4, 48
        with torch.cuda.stream(be.stream):
            gen = torch.Generator(device=be.device).manual_seed(1)
            buf = lambda *s: DeviceBuffer(torch.randn(*s, device=be.device, generator=gen).view(-1))
            x, logits, g = buf(t, c), buf(t, e), buf(t, c)
        plan = be.rope_plan(16)
        def step():
            q = be.rope_dev(x, (1, t, 3, 16), plan)
            z = be.dropout_dev(q, None, x, 0.3, 5, 6, t, c)
            w, ids = be.moe_gate_dev(logits, t, e, k)
            mp = be.moe_sort_dev(ids, t, k, e)
            xs = be.moe_dispatch_dev(z, mp, c)
            y = be.moe_combine_dev(xs, w, mp, c)
            dys, dw = be.moe_combine_backward_dev(g, xs, w, mp, c)
            dl = be.moe_gate_backward_dev(dw, logits, w, ids, t, e, k)
            dz = be.moe_dispatch_backward_dev(dys, mp, c)
            dq, db = be.dropout_backward_dev(dz, 0.3, 5, 6, t, c, want_dbias=True)
            return [y, dl, db, be.rope_backward_dev(dq, (1, t, 3, 16), plan), mp.place, mp.offsets]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=be.stream):
            outs = step()
        graph.replay()
        torch.cuda.synchronize()
        first = [o.t.clone() for o in outs]
        eager = step()
        be.synchronize()
        assert all(torch.equal(a, b.t) for a, b in zip(first, eager))
        print("captured ok")
    """)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=180, cwd=__file__.rsplit("/tests/", 1)[0])
    assert r.returncode == 0 and "captured ok" in r.stdout, r.stdout + r.stderr


def test_two_backends_at_once():
    """Two streams with calls in flight at the same time: scratch is each backend's own."""
    from ferro_b200.backend import CudaBackend
    pair = [CudaBackend(0), CudaBackend(0)]
    t, k, e, c = 20000, 4, 64, 96
    data = []
    for i, b in enumerate(pair):
        r = np.random.default_rng(i)
        data.append((b.alloc_i64_from_host(r.integers(0, e, t * k)), b.alloc_from_host(r.standard_normal((t, c)))))

    def go(b, ids, x):
        plan = b.moe_sort_dev(ids, t, k, e)
        xs = b.moe_dispatch_dev(x, plan, c)
        dx, db = b.dropout_backward_dev(xs, 0.2, 1, 2, t * k, c, want_dbias=True)
        return [plan.place, plan.offsets, dx, db]

    want = []
    for b, d in zip(pair, data):
        got = go(b, *d)
        b.synchronize()
        want.append([o.t.clone() for o in got])
    torch.cuda.synchronize()
    for _ in range(5):
        outs = [None, None]
        for _ in range(3):
            for i, (b, d) in enumerate(zip(pair, data)):
                outs[i] = go(b, *d)
        for b in pair:
            b.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(a.t, v) for a, v in zip(o, w))


def test_two_threads_on_one_backend():
    """Each call's launches share a scratch and stand together on the stream, whatever the other thread launches; a new
    stream gets a scratch of its own."""
    import threading
    from ferro_b200.backend import CudaBackend
    b = CudaBackend(0)
    t, k, e, c = 20000, 4, 64, 96
    data = []
    for i in range(2):
        r = np.random.default_rng(i)
        data.append((b.alloc_i64_from_host(r.integers(0, e, t * k)), b.alloc_from_host(r.standard_normal((t, c)))))

    def go(ids, g):
        plan = b.moe_sort_dev(ids, t, k, e)
        dx, db = b.dropout_backward_dev(g, 0.2, 1, 2, t, c, want_dbias=True)
        return [plan.place.t, plan.order.t, plan.offsets.t, dx.t, db.t]

    want = [go(*d) for d in data]
    b.synchronize()
    wrong = []

    def run(i):
        try:
            with torch.cuda.stream(b.stream):
                same = [torch.stack([(a == v).all() for a, v in zip(go(*data[i]), want[i])]).all()
                        for _ in range(100)]
                wrong.extend(n for n, ok in enumerate(torch.stack(same).tolist()) if not ok)
        except Exception as x:
            wrong.append(x)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for h in threads:
        h.start()
    for h in threads:
        h.join()
    assert not wrong
    b.stream = torch.cuda.Stream(device=b.device)
    got = go(*data[0])
    b.synchronize()
    assert all(torch.equal(a, v) for a, v in zip(got, want[0]))
