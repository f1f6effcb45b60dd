"""Expert rows and dropout past 32-bit element numbers with sums that come out exactly, so that no element can be missed,
taken twice or taken from another column unseen."""
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


@pytest.mark.parametrize("more", [4, 3])  # rows in 16-byte accesses, and not
def test_weight_gradient_of_long_rows_counts_every_column_once(be, more):
    """dy is 0 but for powers of two at a few columns, where the experts' rows hold 1 and 3, and 7 elsewhere: the sums are
    whole numbers below 2^24."""
    from ferro_b200.backend import MoePlan
    cols, slots = 2 ** 30 + more, 5
    at = torch.tensor([0, 1, 255, 1024, 2 ** 28 + 5, 2 ** 29 - 1, 2 ** 29, 3 * 2 ** 28, 2 ** 30 - 1, 2 ** 30, cols - 2, cols - 1])
    dy, ys = filled(be, 2 * cols, 0.0), filled(be, slots * cols, 7.0)
    plan = MoePlan(be.alloc_i64_from_host([4, 0]), None, None, 2, 1, slots)
    w = be.alloc_from_host([0.5, 2.0])
    with torch.cuda.stream(be.stream):
        where = at.to(be.device)
        value = 2.0 ** torch.arange(len(at), device=be.device, dtype=torch.float32)
        dy.t[where], dy.t[cols + where] = value, value.flip(0)
        ys.t[4 * cols + where], ys.t[where] = 1.0, 3.0
    dys, dw = be.moe_combine_backward_dev(dy, ys, w, plan, cols, dys=ys)
    total = 2.0 ** len(at) - 1
    assert be.copy_to_host(dw).tolist() == [total, 3 * total]
    be.synchronize()
    for row, factor, place in ((0, 0.5, 4), (1, 2.0, 0)):
        got = dys.t[place * cols:(place + 1) * cols]
        assert torch.equal(got[where], factor * dy.t[row * cols + where])
        assert int(torch.count_nonzero(got[:2 ** 30])) + int(torch.count_nonzero(got[2 ** 30:])) == len(at)
    assert bool((dys.t[cols:4 * cols:1 << 12] == 7.0).all())  # rows of nobody


def test_dropout_of_an_odd_width_past_32_bits(be):
    """The forward's bias by column where no row starts on a vector, and the backward's column sums: p = 1/2 makes every kept
    element exactly 2, a column's sum twice a count below 2^24."""
    rows, cols, p, seed, off = 1047555, 4101, 0.5, 987654321, 2 ** 32 - 77
    n = rows * cols
    assert n > 2 ** 32
    x = filled(be, n, 1.0)
    bias = np.arange(cols, dtype=np.float32)
    B = be.alloc_from_host(bias)
    be.dropout_dev(x, B, None, p, seed, off, rows, cols, out=x)
    be.synchronize()
    for start in (0, 2 ** 31 - 8000, 2 ** 32 - 8000, n - 16000):
        start -= start % 4
        m = min(16000, n - start)
        keep = ref.drop_keep(m, p, seed, off + start // 4)
        want = np.where(keep, 2 * (1 + bias[(start + np.arange(m, dtype=np.int64)) % cols]), 0)
        assert (x.t[start:start + m].cpu().numpy() == want).all(), start
    with torch.cuda.stream(be.stream):
        x.t.fill_(1.0)
    dx, db = be.dropout_backward_dev(x, p, seed, off, rows, cols, want_dbias=True, dx=x)
    sums = be.copy_to_host(db)
    for start in (0, 2 ** 32 - 8000, n - 16000):
        start -= start % 4
        m = min(16000, n - start)
        keep = ref.drop_keep(m, p, seed, off + start // 4)
        assert (dx.t[start:start + m].cpu().numpy() == np.where(keep, 2, 0)).all(), start
    for c in (0, 1, 1023, 1024, 4099, 4100):
        e = np.arange(rows, dtype=np.int64) * cols + c
        words = ref.philox(np.uint64(off) + (e // 4).astype(np.uint64), seed)
        kept = int((words[np.arange(rows), e % 4] >= np.uint64(2 ** 31)).sum())
        assert sums[c] == 2 * kept, c
