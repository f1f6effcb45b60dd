"""64-bit references, in plain numpy, of what a transformer layer with routed experts runs between its matrix products:
rotary positions, dropout from a counter-based generator, the router's gate, the expert sort and the row movement around
the experts.  Written from the formulas of include/ferro_b200.h; tests/test_layer_ops_cpu.py holds them against finite
differences and published values before the GPU tests use them."""
import math

import numpy as np

EPS = 2.0 ** -24  # one f32 rounding is off by at most this, relative


# ---- rotary positions ------------------------------------------------------------------------------------------------

def rope_theta(rot, base=10000.0, scaling="plain", factor=1.0, original_len=0.0, low=0.0, high=0.0):
    i = np.arange(rot // 2, dtype=np.float64)
    if scaling == "base":
        base = base * factor ** (rot / (rot - 2))
    theta = np.power(float(base), -2.0 * i / rot)
    if scaling == "linear":
        theta = theta / factor
    if scaling == "by_parts":
        turns = original_len * theta / (2 * math.pi)
        keep = np.clip((turns - low) / (high - low), 0.0, 1.0)
        theta = theta * keep + theta / factor * (1.0 - keep)
    return theta


def rope_angles(positions, theta):
    """positions int64 [batch, seq] -> angles [batch, seq, pairs] modulo one turn, the product taken in 80 bits (exact to
    2^-64 of the whole angle, where 64 bits lose far positions)."""
    a = np.asarray(positions).astype(np.longdouble)[..., None] * np.asarray(theta, np.longdouble)
    two_pi = 2 * np.longdouble("3.14159265358979323846264338327950288")
    return (a - np.floor(a / two_pi) * two_pi).astype(np.float64)


def rope(x, angles, layout, scale=1.0, inverse=False):
    """x [batch, seq, heads, dim] in f64; angles [batch, seq, pairs]."""
    x = np.asarray(x, np.float64)
    rot = 2 * angles.shape[-1]
    c, s = np.cos(angles)[:, :, None, :] * scale, np.sin(angles)[:, :, None, :] * (-scale if inverse else scale)
    out = x.copy()
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def rope_bound(x, rot, layout, scale=1.0):
    """How far one f32 result may be off.  The angle: its remainder of a quarter turn, at most 1/4 of a half turn, becomes a
    float, off by 2^-27 of a half turn, after 2^-31 of one was cut off: pi (2^-27 + 2^-31).  Cosine and sine from their
    series: 2^-23, two units in the last place.  Times scale, each product and the final sum: three roundings of 2^-24.
    All of it relative to (|a| + |b|) * scale."""
    x = np.abs(np.asarray(x, np.float64))
    per = math.pi * (2.0 ** -27 + 2.0 ** -31) + 2.0 ** -23 + 3 * EPS
    bound = np.zeros_like(x)
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    bound[..., a] = bound[..., b] = (x[..., a] + x[..., b]) * scale * per
    return bound


# ---- dropout ---------------------------------------------------------------------------------------------------------

def philox(counters, key):
    """Philox4x32-10 (Salmon, Moraes, Dror and Shaw, SC 2011): words [n, 4] for 64-bit counters [n]."""
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    n = np.asarray(counters, np.uint64)
    c = [n & low, n >> half, np.zeros_like(n), np.zeros_like(n)]
    return philox_rounds(c, key)


def philox_rounds(c, key):
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    k0, k1 = key & 0xFFFFFFFF, key >> 32
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> half) ^ c[1] ^ np.uint64(k0), q & low, (p >> half) ^ c[3] ^ np.uint64(k1), p & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, -1)


def drop_keep(n, p, seed, offset):
    """Which of n elements stay."""
    blocks = (n + 3) // 4
    first = np.uint64(offset % 2 ** 64)
    with np.errstate(over="ignore"):
        at = first + np.arange(blocks, dtype=np.uint64)  # wraps
    words = philox(at, seed % 2 ** 64).reshape(-1)[:n]
    return words >= np.uint64(int(np.rint(float(np.float32(p)) * 2.0 ** 32)))


def dropout(x, bias, residual, p, seed, offset):
    """(out, keep, bound): the bound counts x + bias, the factor 1 / (1 - p), the product and the final sum, a rounding
    each."""
    x = np.asarray(x, np.float64)
    keep = drop_keep(x.size, p, seed, offset).reshape(x.shape)
    p = float(np.float32(p))
    factor = 0.0 if p == 1.0 else 1.0 / (1.0 - p)
    z = x if bias is None else x + np.asarray(bias, np.float64)
    with np.errstate(invalid="ignore"):
        z = np.where(keep, z * factor, 0.0)
    out = z if residual is None else z + np.asarray(residual, np.float64)
    return out, keep, 1.0001 * EPS * (3 * np.abs(z) + np.abs(out))


# ---- gate --------------------------------------------------------------------------------------------------------------

def gate(logits, k, renorm):
    """(weights f64 [t, k], ids i64 [t, k]): descending, ties to the lowest index, NaN first, -inf never."""
    l = np.asarray(logits, np.float64)
    t, e = l.shape
    w, ids = np.zeros((t, k)), np.full((t, k), -1, np.int64)
    for r in range(t):
        order = sorted((i for i in range(e) if l[r, i] != -math.inf),
                       key=lambda i: (0 if math.isnan(l[r, i]) else 1, 0.0 if math.isnan(l[r, i]) else -l[r, i], i))
        chosen = order[:k]
        if not chosen:
            continue
        ids[r, :len(chosen)] = chosen
        pool = chosen if renorm else order
        m = l[r, chosen[0]]
        with np.errstate(invalid="ignore"):
            mass = {i: math.nan if math.isnan(l[r, i] - m) else math.exp(l[r, i] - m) for i in pool}
        total = sum(mass.values())
        w[r, :len(chosen)] = [mass[i] / total for i in chosen]
    return w, ids


def gate_rel(logits, k, renorm):
    """Relative bound on a weight: the exponent's rounding |l - m| 2^-24 and expf's 2 ulp, once for the numerator and once
    for the (positive) sum, whose additions follow at most experts / 32 + 6 deep, and the division."""
    l = np.asarray(logits, np.float64)
    fin = np.where(np.isfinite(l), l, 0.0)
    spread = min(float((fin.max() - fin.min()) if l.size else 0.0), 104.0)  # past that the f32 exponential is 0
    return 2 * (spread * EPS + 2.0 ** -22) + (l.shape[1] / 32 + 8) * EPS


def gate_backward(dw, logits, ids, k, renorm):
    l, dw = np.asarray(logits, np.float64), np.asarray(dw, np.float64)
    t, e = l.shape
    out = np.zeros((t, e))
    for r in range(t):
        real = ids[r] >= 0
        chosen = ids[r][real]
        if not len(chosen):
            continue
        pool = np.zeros(e, bool)
        if renorm:
            pool[chosen] = True
        else:
            pool = l[r] != -math.inf
        p = np.zeros(e)
        m = l[r][pool].max()
        p[pool] = np.exp(l[r][pool] - m)
        p /= p.sum()
        up = np.zeros(e)
        up[chosen] = dw[r][real]
        out[r] = p * (up - (p * up).sum())
    return out


# ---- experts -----------------------------------------------------------------------------------------------------------

def sort_by_expert(ids, experts):
    """(place, order of the rows there are, offsets)."""
    ids = np.asarray(ids, np.int64).reshape(-1)
    ok = (ids >= 0) & (ids < experts)
    order = np.flatnonzero(ok)
    order = order[np.argsort(ids[order], kind="stable")]
    place = np.full(len(ids), -1, np.int64)
    place[order] = np.arange(len(order))
    counts = np.bincount(ids[ok], minlength=experts) if experts else np.zeros(0, np.int64)
    return place, order, np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)


def spread(x, place, k, rows, fill, weights=None):
    """Rows of x at their places; rows nobody has keep `fill`."""
    out = np.full((rows, x.shape[1]), fill, np.float64)
    for a, s in enumerate(place):
        if 0 <= s < rows:
            out[s] = np.asarray(x[a // k], np.float64) * (1.0 if weights is None else float(weights[a]))
    return out


def collect(ys, place, tokens, k, weights=None):
    """(sum over a token's places, the same sum of absolute values)."""
    out, mag = np.zeros((tokens, ys.shape[1])), np.zeros((tokens, ys.shape[1]))
    for a, s in enumerate(place):
        if 0 <= s < len(ys):
            v = np.asarray(ys[s], np.float64) * (1.0 if weights is None else float(weights[a]))
            out[a // k] += v
            mag[a // k] += np.abs(v)
    return out, mag


def weight_gradient(dy, ys, place, k):
    out, mag = np.zeros(len(place)), np.zeros(len(place))
    for a, s in enumerate(place):
        if 0 <= s < len(ys):
            v = np.asarray(dy[a // k], np.float64) * np.asarray(ys[s], np.float64)
            out[a], mag[a] = v.sum(), np.abs(v).sum()
    return out, mag
