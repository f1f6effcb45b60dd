"""Rotary positions, dropout, the router's gate and the expert sort, without a GPU: what the entries refuse before any
launch, the table of frequencies, and the 64-bit references against published values and finite differences."""
import ctypes as C
import decimal

import numpy as np
import pytest

import layer_reference as ref
from ferro_b200 import _lib, build
from ferro_b200 import kinds as K

P = 0x100000  # an address that no refused call touches


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def says(lib, rc, code, text):
    assert rc == code, (rc, lib.fb_last_error())
    assert text.encode() in lib.fb_last_error()


# ---- frequencies -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rot,base", [(2, 10000.0), (64, 10000.0), (128, 1e6), (40, 500000.0), (256, 1.0)])
@pytest.mark.parametrize("scaling", ["plain", "linear", "base", "by_parts"])
def test_frequency_table_holds_turns_as_64_bit_fractions(lib, rot, base, scaling):
    if scaling == "base" and rot == 2:
        return
    kinds = {"plain": K.ROPE_PLAIN, "linear": K.ROPE_LINEAR, "base": K.ROPE_BASE, "by_parts": K.ROPE_BY_PARTS}
    factor, length, low, high = 8.0, 4096.0, 1.0, 32.0
    got = np.empty(rot // 2, np.int64)
    assert lib.fb_rope_turns(rot, base, kinds[scaling], factor, length, low, high, got.ctypes.data) == 0
    with decimal.localcontext() as ctx:
        ctx.prec = 60
        D = decimal.Decimal
        pi = D("3.14159265358979323846264338327950288419716939937510582097494459")
        b = D(base) * (D(factor) ** (D(rot) / D(rot - 2)) if scaling == "base" else 1)
        for i in range(rot // 2):
            theta = b ** (D(-2 * i) / D(rot))
            if scaling == "linear":
                theta /= D(factor)
            if scaling == "by_parts":
                keep = min(D(1), max(D(0), (D(length) * theta / (2 * pi) - D(low)) / (D(high) - D(low))))
                theta = theta * keep + theta / D(factor) * (1 - keep)
            want = theta / (2 * pi) * 2 ** 64
            # 80-bit powl and divisions: the exponent's rounding is multiplied by ln(1 / theta) < 16, a dozen further
            # roundings of 2^-64; one unit for the last place of the fraction
            assert abs(D(int(got[i]) % 2 ** 64) - want) <= want * D(2) ** -59 + 1, (i, got[i], want)


def test_frequency_table_refusals(lib):
    t = np.empty(64, np.int64).ctypes.data
    says(lib, lib.fb_rope_turns(3, 1e4, 0, 1, 0, 0, 0, t), 1, "even number")
    says(lib, lib.fb_rope_turns(0, 1e4, 0, 1, 0, 0, 0, t), 1, "even number")
    says(lib, lib.fb_rope_turns(64, 0.0, 0, 1, 0, 0, 0, t), 2, "base")
    says(lib, lib.fb_rope_turns(64, float("nan"), 0, 1, 0, 0, 0, t), 2, "base")
    says(lib, lib.fb_rope_turns(64, 1e4, 4, 1, 0, 0, 0, t), 2, "scaling")
    says(lib, lib.fb_rope_turns(64, 1e4, 1, 0.0, 0, 0, 0, t), 2, "factor")
    says(lib, lib.fb_rope_turns(2, 1e4, 2, 2.0, 0, 0, 0, t), 2, "one pair")
    says(lib, lib.fb_rope_turns(64, 1e4, 3, 2.0, 0.0, 1, 32, t), 2, "original_len")
    says(lib, lib.fb_rope_turns(64, 1e4, 3, 2.0, 4096.0, 32, 32, t), 2, "low < high")
    says(lib, lib.fb_rope_turns(64, 1e4, 0, 1, 0, 0, 0, None), 2, "null")


def rope_call(lib, shape=(2, 3, 4, 8), strides=None, ptr=P, length=None, offset=0, rank=4, positions=None, pos_rows=1,
              turns=P, rot=8, layout=K.ROPE_HALF, out=2 * P, out_len=None, out_strides=None, out_offset=0):
    n, st = 1, []
    for s in reversed(shape):
        st.insert(0, n)
        n *= s
    strides = strides or st
    v = _lib.ViewDesc(ptr, n if length is None else length, offset, rank, (C.c_uint64 * 16)(*shape), (C.c_int64 * 16)(*strides))
    os_ = (C.c_int64 * 4)(*out_strides) if out_strides else None
    return lib.fb_rope(None, C.byref(v), positions, pos_rows, 0, turns, rot, layout, 1.0, 0, out,
                       n if out_len is None else out_len, os_, out_offset)


def test_rope_refusals(lib):
    says(lib, rope_call(lib, layout=2), 2, "layout")
    says(lib, rope_call(lib, rank=3), 1, "rank")
    says(lib, rope_call(lib, rot=7), 1, "rot_dim")
    says(lib, rope_call(lib, rot=10), 1, "rot_dim")
    says(lib, rope_call(lib, rot=0), 1, "rot_dim")
    says(lib, rope_call(lib, positions=P, pos_rows=3), 1, "positions")
    says(lib, rope_call(lib, length=191), 1, "outside its storage")
    says(lib, rope_call(lib, offset=1), 1, "outside its storage")
    says(lib, rope_call(lib, out_len=191), 1, "outside its storage")
    says(lib, rope_call(lib, out_offset=-1), 1, "outside its storage")
    says(lib, rope_call(lib, ptr=None), 2, "null")
    says(lib, rope_call(lib, out=None), 2, "null")
    says(lib, rope_call(lib, turns=None), 2, "null")
    says(lib, rope_call(lib, out_strides=(96, 32, 0, 1)), 2, "share addresses")   # broadcast output
    says(lib, rope_call(lib, out_strides=(96, 32, 7, 1), out_len=400), 2, "share addresses")
    says(lib, rope_call(lib, out=P + 4, out_len=192), 2, "overlaps x")
    says(lib, rope_call(lib, out=P, out_strides=(8, 16, 48, 1)), 2, "overlaps x")  # same storage, another order
    says(lib, rope_call(lib, shape=(1 << 31, 1, 1, 2), strides=(2, 2, 2, 1), rot=2, out=P + (1 << 40)), 4, "2^31")
    # nothing to do: no launch, no device
    for shape in [(0, 3, 4, 8), (2, 0, 4, 8), (2, 3, 0, 8), (0, 1 << 62, 1 << 62, 8)]:
        assert rope_call(lib, shape=shape, ptr=None, out=None) == 0


def test_dropout_refusals(lib):
    for p in (-0.1, 1.1, float("nan")):
        says(lib, lib.fb_dropout_fwd(None, P, None, None, 2, 4, p, 1, 0, None, P), 2, "p must lie")
        says(lib, lib.fb_dropout_bwd(None, P, 2, 4, p, 1, 0, None, P, None, None, 0), 2, "p must lie")
    says(lib, lib.fb_dropout_fwd(None, P, None, None, 1 << 63, 4, 0.1, 1, 0, None, P), 1, "overflows")
    says(lib, lib.fb_dropout_bwd(None, P, 1 << 63, 4, 0.1, 1, 0, None, P, None, None, 0), 1, "overflows")
    says(lib, lib.fb_dropout_fwd(None, None, None, None, 2, 4, 0.1, 1, 0, None, P), 2, "null")
    says(lib, lib.fb_dropout_fwd(None, P, None, None, 2, 4, 0.1, 1, 0, None, None), 2, "null")
    says(lib, lib.fb_dropout_bwd(None, None, 2, 4, 0.1, 1, 0, None, P, None, None, 0), 2, "null")
    says(lib, lib.fb_dropout_fwd(None, P, P - 64, None, 1, 1 << 31, 0.1, 1, 0, None, P + (1 << 40)), 4, "bias")
    # outputs that overlap an input without being it
    says(lib, lib.fb_dropout_fwd(None, P, None, None, 2, 4, 0.1, 1, 0, None, P + 4), 2, "overlaps")
    says(lib, lib.fb_dropout_fwd(None, P, None, 2 * P, 2, 4, 0.1, 1, 0, None, 2 * P - 4), 2, "overlaps")
    says(lib, lib.fb_dropout_fwd(None, P, 2 * P, None, 2, 4, 0.1, 1, 0, None, 2 * P + 8), 2, "overlaps")
    says(lib, lib.fb_dropout_bwd(None, P, 2, 4, 0.1, 1, 0, None, P + 16, None, None, 0), 2, "overlaps")
    says(lib, lib.fb_dropout_bwd(None, P, 2, 4, 0.1, 1, 0, None, 2 * P, P + 16, None, 0), 2, "overlaps")
    says(lib, lib.fb_dropout_bwd(None, P, 2, 4, 0.1, 1, 0, None, 2 * P, 2 * P, None, 0), 2, "overlaps")
    need = lib.fb_dropout_bwd_workspace_bytes(100000, 64)
    assert need > 0
    says(lib, lib.fb_dropout_bwd(None, 1 << 40, 100000, 64, 0.1, 1, 0, None, 1 << 40, P, None, 0), 5, "scratch")
    says(lib, lib.fb_dropout_bwd(None, 1 << 40, 100000, 64, 0.1, 1, 0, None, 1 << 40, P, P, need - 1), 5, "scratch")
    says(lib, lib.fb_dropout_advance(None, None, 1), 2, "null")
    assert lib.fb_dropout_fwd(None, None, None, None, 0, 4, 0.1, 1, 0, None, None) == 0
    assert lib.fb_dropout_bwd(None, P, 4, 0, 0.1, 1, 0, None, P, P, None, 0) == 0
    assert lib.fb_dropout_bwd(None, P, 4, 4, 0.1, 1, 0, None, None, None, None, 0) == 0  # no output asked for


def test_expert_refusals(lib):
    for k, e in [(0, 4), (5, 4), (33, 64)]:
        says(lib, lib.fb_moe_gate_fwd(None, P, 2, e, k, 1, P, P), 1, "k ")
        says(lib, lib.fb_moe_gate_bwd(None, P, P, P, P, 2, e, k, 1, P), 1, "k ")
    for e in (0, 1025):
        says(lib, lib.fb_moe_gate_fwd(None, P, 2, e, 1, 1, P, P), 1, "experts")
        says(lib, lib.fb_moe_sort(None, P, 8, e, P, P, P, None, None, 0), 1, "experts")
    says(lib, lib.fb_moe_gate_fwd(None, P, 1 << 62, 64, 2, 1, P, P), 1, "overflows")
    for a in ([None, P, P], [P, None, P], [P, P, None]):
        says(lib, lib.fb_moe_gate_fwd(None, a[0], 2, 4, 2, 1, a[1], a[2]), 2, "null")
    says(lib, lib.fb_moe_gate_bwd(None, P, None, P, P, 2, 4, 2, 0, P), 2, "null")  # all experts' softmax needs the logits
    says(lib, lib.fb_moe_sort(None, P, 1 << 31, 4, P, P, P, None, None, 0), 4, "2^31")
    says(lib, lib.fb_moe_sort(None, None, 8, 4, P, P, P, None, None, 0), 2, "null")
    says(lib, lib.fb_moe_sort(None, P, 8, 4, None, P, P, None, None, 0), 2, "null")
    says(lib, lib.fb_moe_sort(None, P, 8, 4, P, P, None, None, None, 0), 2, "null")
    for a in ([P + 8, 2 * P, 3 * P], [P, P, 3 * P], [2 * P, 2 * P + 8, 3 * P], [2 * P, 3 * P, 3 * P - 8], [2 * P, 3 * P, P + 56]):
        says(lib, lib.fb_moe_sort(None, P, 8, 4, a[0], a[1], a[2], None, None, 0), 2, "overlaps")
    for a in ([P + 4, 3 * P], [2 * P, P], [2 * P, 2 * P + 12]):
        says(lib, lib.fb_moe_gate_fwd(None, P, 2, 4, 2, 1, a[0], a[1]), 2, "overlaps")
    for a in (P, 2 * P + 4, 3 * P, 4 * P + 24):
        says(lib, lib.fb_moe_gate_bwd(None, P, 2 * P, 3 * P, 4 * P, 2, 4, 2, 0, a), 2, "overlaps")
    need = lib.fb_moe_sort_workspace_bytes(1 << 20, 64)
    assert need > 0 and lib.fb_moe_sort_workspace_bytes(100, 64) == 0
    says(lib, lib.fb_moe_sort(None, 1 << 32, 1 << 20, 64, 1 << 33, 1 << 34, 1 << 35, None, P, need - 1), 5, "scratch")
    for k in (0, 33):
        says(lib, lib.fb_moe_dispatch_fwd(None, P, P, 2, k, 4, 2 * P, 8), 1, "k ")
        says(lib, lib.fb_moe_dispatch_bwd(None, P, P, 2, k, 4, 8, 2 * P), 1, "k ")
        says(lib, lib.fb_moe_combine_fwd(None, P, P, P, 2, k, 4, 8, 2 * P), 1, "k ")
        says(lib, lib.fb_moe_combine_bwd(None, P, P, P, P, 2, k, 4, 8, 2 * P, 3 * P), 1, "k ")
    says(lib, lib.fb_moe_dispatch_fwd(None, P, P, 1 << 62, 2, 4, 2 * P, 8), 1, "overflow")
    says(lib, lib.fb_moe_dispatch_fwd(None, P, P, 2, 2, 4, 2 * P, 1 << 62), 1, "overflow")
    says(lib, lib.fb_moe_dispatch_fwd(None, P, None, 2, 2, 4, 2 * P, 8), 2, "null")
    says(lib, lib.fb_moe_dispatch_fwd(None, P, 3 * P, 2, 2, 4, P, 8), 2, "must not")
    says(lib, lib.fb_moe_dispatch_bwd(None, None, P, 2, 2, 4, 8, P), 2, "null")
    says(lib, lib.fb_moe_dispatch_bwd(None, P, 3 * P, 2, 2, 4, 8, P + 64), 2, "must not")
    says(lib, lib.fb_moe_combine_fwd(None, P, None, P, 2, 2, 4, 8, 2 * P), 2, "null")
    says(lib, lib.fb_moe_combine_bwd(None, P, None, P, P, 2, 2, 4, 8, 2 * P, 3 * P), 2, "null")
    says(lib, lib.fb_moe_dispatch_fwd(None, P, 3 * P, 2, 2, 4, P + 28, 8), 2, "must not")
    says(lib, lib.fb_moe_dispatch_fwd(None, P, 3 * P, 2, 2, 4, 3 * P, 8), 2, "must not")
    for y in (P + 124, 2 * P, 3 * P):
        says(lib, lib.fb_moe_combine_fwd(None, P, 2 * P, 3 * P, 2, 2, 4, 8, y), 2, "must not")
    # dy, ys, weights, place -> dys, dweights: dys may be ys and nothing else
    for a in ([P, 6 * P], [2 * P + 4, 6 * P], [3 * P, 6 * P], [4 * P, 6 * P], [5 * P, P], [5 * P, 2 * P], [5 * P, 3 * P], [5 * P, 4 * P],
              [5 * P, 5 * P], [2 * P, 2 * P + 16]):
        says(lib, lib.fb_moe_combine_bwd(None, P, 2 * P, 3 * P, 4 * P, 2, 2, 4, 8, a[0], a[1]), 2, "must not")
    says(lib, lib.fb_moe_dispatch_fwd(None, P, 3 * P, 2, 2, 1 << 31, 2 * P, 8), 4, "2^31")
    # nothing to do
    assert lib.fb_moe_gate_fwd(None, None, 0, 4, 2, 1, None, None) == 0
    assert lib.fb_moe_gate_bwd(None, None, None, None, None, 0, 4, 2, 0, None) == 0
    assert lib.fb_moe_dispatch_fwd(None, None, None, 0, 2, 4, None, 0) == 0
    assert lib.fb_moe_dispatch_fwd(None, P, P, 2, 2, 4, None, 0) == 0
    assert lib.fb_moe_combine_fwd(None, None, None, None, 0, 2, 4, 0, None) == 0
    assert lib.fb_moe_combine_bwd(None, P, P, P, P, 2, 2, 4, 8, None, None) == 0


# ---- the references themselves -------------------------------------------------------------------------------------------

def test_philox_reference_gives_the_published_words():
    """Known answers of the generator's paper distribution for Philox4x32-10: all-zero and all-one counters and keys."""
    zero = ref.philox(np.zeros(1, np.uint64), 0)[0]
    assert [int(w) for w in zero] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = ref.philox_rounds([np.full(1, 0xFFFFFFFF, np.uint64)] * 4, 2 ** 64 - 1)[0]
    assert [int(w) for w in ones] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_dropout_reference_keeps_the_share_it_should():
    n, p = 1 << 18, 0.3
    kept = ref.drop_keep(n, p, 12345, 2 ** 64 - 7).mean()  # counters that wrap
    assert abs(kept - 0.7) < 5 * np.sqrt(0.3 * 0.7 / n)  # five standard deviations of the mean


def differences(f, x, up, h=1e-5):
    """Central differences of (f(x) * up).sum() in 64 bits."""
    g = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        a, b = x.copy(), x.copy()
        a[i] += h
        b[i] -= h
        g[i] = ((f(a) - f(b)) * up).sum() / (2 * h)
    return g


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_reference_gradient_against_differences(layout):
    r = np.random.default_rng(1)
    x, up = r.standard_normal((2, 3, 2, 8)), r.standard_normal((2, 3, 2, 8))
    ang = ref.rope_angles(np.array([[5, 100, 7], [0, -3, 9]]), ref.rope_theta(6))
    got = ref.rope(up, ang, layout, 1.3, inverse=True)
    assert np.abs(got - differences(lambda z: ref.rope(z, ang, layout, 1.3), x, up)).max() < 1e-8


def test_dropout_reference_gradient_against_differences():
    r = np.random.default_rng(4)
    x, b, res, up = r.standard_normal((3, 5)), r.standard_normal(5), r.standard_normal((3, 5)), r.standard_normal((3, 5))
    p, seed, off = float(np.float32(0.4)), 9, 11
    dx = ref.dropout(up, None, None, p, seed, off)[0]
    assert np.abs(dx - differences(lambda z: ref.dropout(z, b, res, p, seed, off)[0], x, up)).max() < 1e-8
    assert np.abs(dx.sum(0) - differences(lambda z: ref.dropout(x, z, res, p, seed, off)[0], b, up)).max() < 1e-8
    assert np.abs(up - differences(lambda z: ref.dropout(x, b, z, p, seed, off)[0], res, up)).max() < 1e-8


@pytest.mark.parametrize("renorm", [True, False])
def test_gate_reference_gradient_against_differences(renorm):
    r = np.random.default_rng(2)
    l = r.standard_normal((5, 7))
    l[1, [2, 5]] = -np.inf
    l[3, 1:] = -np.inf   # one expert left
    l[4, :] = -np.inf    # none
    up = r.standard_normal((5, 3))
    _, ids = ref.gate(l, 3, renorm)
    got = ref.gate_backward(up, l, ids, 3, renorm)
    want = np.zeros_like(l)
    for i in np.ndindex(*l.shape):
        if l[i] == -np.inf:
            continue
        d = 1e-5
        a, b = l.copy(), l.copy()
        a[i] += d
        b[i] -= d
        want[i] = ((ref.gate(a, 3, renorm)[0] - ref.gate(b, 3, renorm)[0]) * up).sum() / (2 * d)
    assert np.abs(got - want).max() < 1e-8
    assert (got[4] == 0).all()


def test_expert_references_agree_with_their_gradients():
    """spread and collect are each other's transpose; weight_gradient is collect's derivative in the weights."""
    r = np.random.default_rng(3)
    t, k, e, c = 9, 2, 4, 3
    ids = r.integers(-1, e, (t, k))
    place, order, off = ref.sort_by_expert(ids, e)
    assert off[-1] == (ids >= 0).sum() == len(order)
    assert (np.sort(place[place >= 0]) == np.arange(len(order))).all()
    assert all(ids.reshape(-1)[order[off[i]:off[i + 1]]].tolist() == [i] * (off[i + 1] - off[i]) for i in range(e))
    x, up, w = r.standard_normal((t, c)), r.standard_normal((t * k, c)), r.standard_normal(t * k)
    a = (ref.spread(x, place, k, t * k, 0.0, w) * up).sum()
    assert abs(a - (x * ref.collect(up, place, t, k, w)[0]).sum()) < 1e-12
    dy = r.standard_normal((t, c))
    dw = ref.weight_gradient(dy, up, place, k)[0]
    num = differences(lambda v: ref.collect(up, place, t, k, v)[0], w, dy)
    assert np.abs(dw - num).max() < 1e-8
