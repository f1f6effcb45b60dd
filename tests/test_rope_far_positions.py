"""How far a rotary angle is off at far positions: |p| * 2^-64 + 2^-32 turns, against frequencies of 60 digits."""
import decimal
import math

import numpy as np
import pytest

import layer_reference as ref
from ferro_b200 import _lib, build

D = decimal.Decimal
PI = D("3.14159265358979323846264338327950288419716939937510582097494459")
SCALINGS = ["plain", "linear", "base", "by_parts"]
FACTOR, LENGTH, LOW, HIGH = 8.0, 4096.0, 1.0, 32.0


def turns(rot, base, scaling):
    """theta_i / 2 pi to 60 digits."""
    with decimal.localcontext() as ctx:
        ctx.prec = 60
        b = D(base) * (D(FACTOR) ** (D(rot) / D(rot - 2)) if scaling == "base" else 1)
        out = []
        for i in range(rot // 2):
            theta = b ** (D(-2 * i) / D(rot))
            if scaling == "linear":
                theta /= D(FACTOR)
            if scaling == "by_parts":
                keep = min(D(1), max(D(0), (D(LENGTH) * theta / (2 * PI) - D(LOW)) / (D(HIGH) - D(LOW))))
                theta = theta * keep + theta / D(FACTOR) * (1 - keep)
            out.append(theta / (2 * PI))
        return out


@pytest.mark.parametrize("rot,base", [(64, 10000.0), (128, 1e6), (80, 1e7), (256, 500000.0)])
@pytest.mark.parametrize("scaling", SCALINGS)
def test_a_tabled_frequency_is_off_by_less_than_its_last_place(rot, base, scaling):
    build.build()
    got = np.empty(rot // 2, np.int64)
    assert _lib.load().fb_rope_turns(rot, base, SCALINGS.index(scaling), FACTOR, LENGTH, LOW, HIGH, got.ctypes.data) == 0
    for i, t in enumerate(turns(rot, base, scaling)):
        assert abs(D(int(got[i]) % 2 ** 64) - t * 2 ** 64) < 1, i


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("scaling", SCALINGS)
@pytest.mark.parametrize("start", [2 ** 20, 2 ** 31 - 2, -2 ** 33, 2 ** 40, 2 ** 50 + 12345])
def test_far_positions_against_frequencies_of_60_digits(layout, scaling, start):
    from ferro_b200.backend import CudaBackend
    be = CudaBackend(0)
    rot, dim, s = 64, 80, 5
    r = np.random.default_rng(abs(start) % 1000)
    plan = be.rope_plan(rot, layout=layout, scaling=scaling, factor=FACTOR, original_len=LENGTH, low=LOW, high=HIGH)
    with decimal.localcontext() as ctx:
        ctx.prec = 60
        ang = np.array([[[float((D(start + p) * t) % 1) * 2 * math.pi for t in turns(rot, 10000.0, scaling)] for p in range(s)]])
    for inverse, fn in ((False, be.rope_dev), (True, be.rope_backward_dev)):
        x = r.standard_normal((1, s, 2, dim)).astype(np.float32)
        got = be.copy_to_host(fn(be.alloc_from_host(x), x.shape, plan, start=start)).reshape(x.shape)
        # the bound of a near position, which has the cut to 2^-32 turns, and 2 pi |p| 2^-64 on (|a| + |b|)
        per = 2 * math.pi * (abs(start) + s) * 2.0 ** -64
        half = ref.rope_bound(x, rot, layout)
        a, b = (slice(0, 32), slice(32, 64)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
        more = np.zeros_like(half)
        more[..., a] = more[..., b] = (np.abs(x[..., a]) + np.abs(x[..., b])) * per
        assert (np.abs(got - ref.rope(x, ang, layout, 1.0, inverse)) <= half + more).all()
