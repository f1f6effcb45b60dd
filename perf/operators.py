"""Cases that measure the operators a transformer layer with routed experts runs between its matrix products.

Four operators, forward and backward, f32 as everywhere in this library (i64 for whole numbers):

  rope     rotary positions: pairs of channels turned by position * frequency, in the interleaved and the half layout,
           on part of the head, with frequencies scaled for long contexts
  dropout  bias + dropout + residual, the mask drawn from Philox4x32-10 by element number and never stored; its gradient
           draws the same mask again
  gate     a router's choice: softmax over the experts, the k largest, weights over the chosen or over all; its gradient
  experts  token rows sorted by expert (stable), spread to their experts' rows and brought back with the weights applied;
           the gradients of both directions

`own` False computes them from elementary torch operations, True calls ferro_b200's entry points.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
_BACKEND = []


def _backend():
    """The framework's backend handle: one per process, as a program keeps it."""
    if not _BACKEND:
        from ferro_b200.backend import CudaBackend
        _BACKEND.append(CudaBackend(0))
    return _BACKEND[0]


# ---- cases ---------------------------------------------------------------------------------------------------------

def listed():
    return [
        # One new token for each of 32 sequences, every sequence at a position of its own: a generation step.
        _rope("rope one token", 32, 1, 8, 64, 64, "half", "plain", "tokens", positions="own", train=False),
        # The queries of a training step at a usual head size, forward and gradient.
        _rope("rope training", 4, 4096, 32, 128, 128, "interleaved", "plain", "tokens", positions="count", train=True),
        # Few heads out of a packed projection, part of an uncommon head size, an odd length far into a long context.
        _rope("rope long context", 3, 1021, 5, 80, 40, "half", "by_parts", "packed", positions="far", train=True),
        # The matrix of this repository's smoke run: launches and host calls count as much as bytes.
        _dropout("dropout small", 64, 4096, 0.1, bias=False, residual=True, train=True),
        # The output of a projection in a training step: bias, dropout, residual; gradient with the bias gradient.
        _dropout("dropout training", 16384, 4096, 0.1, bias=True, residual=True, train=True),
        # A width that no vector load fits, without the extras.
        _dropout("dropout odd width", 1537, 1001, 0.35, bias=True, residual=False, train=True),
        # A generation step of 32 sequences through a router of 64 experts.
        _gate("gate one token", 32, 64, 8, renorm=True, masked=False, train=False),
        # A training step's router: weights are shares of the softmax over all experts.
        _gate("gate training", 32768, 128, 8, renorm=False, masked=False, train=True),
        # Padded tokens and experts that are shut, a number of experts that is no power of two.
        _gate("gate masked", 10007, 60, 6, renorm=True, masked=True, train=True),
        # The generation step's experts: few rows, latency counts.
        _experts("experts one token", 32, 64, 8, 2048, padded=False, train=False),
        # A training step's experts, forward and gradients.
        _experts("experts training", 8192, 128, 8, 2048, padded=False, train=True),
        # Padded tokens that go to no expert, an odd width, few experts.
        _experts("experts padded", 1000, 7, 3, 1030, padded=True, train=True),
    ]


def _rope(name, batch, seq, heads, dim, rot, layout, scaling, arrangement, positions, train):
    return {"name": name, "op": "rope", "batch": batch, "seq": seq, "heads": heads, "dim": dim, "rot": rot, "layout": layout,
            "scaling": scaling, "arrangement": arrangement, "positions": positions, "train": train}


def _dropout(name, rows, cols, p, bias, residual, train):
    return {"name": name, "op": "dropout", "rows": rows, "cols": cols, "p": p, "bias": bias, "residual": residual, "train": train}


def _gate(name, tokens, experts, k, renorm, masked, train):
    return {"name": name, "op": "gate", "tokens": tokens, "experts": experts, "k": k, "renorm": renorm, "masked": masked, "train": train}


def _experts(name, tokens, experts, k, cols, padded, train):
    return {"name": name, "op": "experts", "tokens": tokens, "experts": experts, "k": k, "cols": cols, "padded": padded, "train": train}


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "dropout", "gate", "experts"])
    most = max(work(c)["bytes"] for c in listed() if c["op"] == op)
    while True:
        c = _draw_one(op, rng)
        if work(c)["bytes"] <= most:
            return c


def _draw_one(op, rng):
    train = rng.random() < 0.7
    if op == "rope":
        dim = 2 * _spread(rng, 8, 128)
        rot = dim if rng.random() < 0.5 else 2 * rng.randint(1, dim // 2)
        seq = 1 if rng.random() < 0.25 else _spread(rng, 2, 16384)
        c = _rope("", _spread(rng, 1, 256 if seq == 1 else 8), seq, _spread(rng, 1, 64), dim, rot, rng.choice(["half", "interleaved"]),
                  rng.choice(["plain", "linear", "base", "by_parts"]) if rot > 2 else "plain", rng.choice(["tokens", "packed", "heads"]),
                  rng.choice(["own", "count", "far"]), train)
    elif op == "dropout":
        cols = _spread(rng, 1, 16384)
        c = _dropout("", _spread(rng, 1, 65536), cols if rng.random() < 0.5 else max(4, cols // 64 * 64), round(rng.uniform(0.01, 0.6), 3),
                     rng.random() < 0.5, rng.random() < 0.5, train)
    elif op == "gate":
        experts = _spread(rng, 2, 512)
        c = _gate("", _spread(rng, 1, 65536), experts, rng.randint(1, min(experts, 10)), rng.random() < 0.5, rng.random() < 0.4, train)
    else:
        experts = _spread(rng, 2, 512)
        cols = _spread(rng, 32, 8192)
        c = _experts("", _spread(rng, 1, 32768), experts, rng.randint(1, min(experts, 10)), cols if rng.random() < 0.4 else max(32, cols // 32 * 32),
                     rng.random() < 0.4, train)
    del c["name"]
    return c


# What one pass has to read and write, each value once, and the operations that it cannot do without.
def work(case):
    c = case
    if c["op"] == "rope":
        n = c["batch"] * c["seq"] * c["heads"] * c["dim"]
        turned = c["batch"] * c["seq"] * c["heads"] * c["rot"]
        once = 8 * n + 8 * c["batch"] * c["seq"] * (c["positions"] == "own")
        return {"bytes": once * (2 if c["train"] else 1), "flops": 3 * turned * (2 if c["train"] else 1)}
    if c["op"] == "dropout":
        n = c["rows"] * c["cols"]
        fwd = 4 * n * (2 + c["residual"]) + 4 * c["cols"] * c["bias"]
        bwd = 8 * n + 4 * c["cols"] * c["bias"] if c["train"] else 0
        return {"bytes": fwd + bwd, "flops": n * (1 + c["residual"] + c["bias"]) + (n * (1 + c["bias"]) if c["train"] else 0)}
    if c["op"] == "gate":
        t, e, k = c["tokens"], c["experts"], c["k"]
        fwd = 4 * t * e + 12 * t * k
        bwd = 4 * t * e + 16 * t * k + (0 if c["renorm"] else 4 * t * e)
        return {"bytes": fwd + (bwd if c["train"] else 0), "flops": 4 * t * e * (2 if c["train"] else 1)}
    t, k, row = c["tokens"], c["k"], 4 * c["cols"]
    gone = _padded(c["tokens"]) if c["padded"] else 0
    s = (t - gone) * k  # rows that reach an expert
    sort = 8 * t * k * 2 + 8 * s + 8 * (c["experts"] + 1)
    fwd = row * (t + s) + row * (s + t) + 8 * t * k * 2 + 4 * t * k
    bwd = row * (s + t) + row * (t + 2 * s) + 8 * t * k * 2 + 8 * t * k
    return {"bytes": sort + fwd + (bwd if c["train"] else 0), "flops": 2 * s * c["cols"] + (4 * s * c["cols"] if c["train"] else 0)}


def _padded(tokens):
    """How many of the tokens are padding where a case has some."""
    return tokens // 8


# ---- inputs ----------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case)
    s["seed"] = seed
    {"rope": _prepare_rope, "dropout": _prepare_dropout, "gate": _prepare_gate, "experts": _prepare_experts}[case["op"]](s, gen)
    return s


def _normal(gen, *shape):
    return torch.randn(*shape, device=DEV, generator=gen)


def _empty(*shape):
    return torch.zeros(*shape, device=DEV)


# base, factor, length of the original context and the ramp's ends, as long-context settings have them
ROPE_BASE, ROPE_FACTOR, ROPE_LENGTH, ROPE_LOW, ROPE_HIGH = 10000.0, 8.0, 4096.0, 1.0, 32.0


def _rope_scale(scaling):
    """The factor on cosine and sine that goes with the frequencies' scaling by parts."""
    return 0.1 * math.log(ROPE_FACTOR) + 1.0 if scaling == "by_parts" else 1.0


def _prepare_rope(s, gen):
    b, n, h, d = s["batch"], s["seq"], s["heads"], s["dim"]
    if s["arrangement"] == "heads":  # [batch, heads, seq, dim] in memory
        shape, strides, extra = (b, h, n, d), (h * n * d, d, n * d, 1), 0
    else:  # [batch, seq, heads, dim], in a packed projection with other heads before and behind
        extra = 3 if s["arrangement"] == "packed" else 0
        shape, strides = (b, n, h + extra, d), (n * (h + extra) * d, (h + extra) * d, d, 1)
    s["strides"], s["offset"] = strides, d if extra else 0
    s["x"] = _normal(gen, *shape).reshape(-1)
    s["g"] = _normal(gen, *shape).reshape(-1) if s["train"] else None
    s["start"], s["pos"] = 0, None
    if s["positions"] == "far":
        s["start"] = 100_000 + s["seed"] % 50_000
    if s["positions"] == "own":
        s["pos"] = torch.randint(0, 32768, (b, n), device=DEV, generator=gen)
    out = (b, h, n, d) if s["arrangement"] == "heads" else (b, n, h, d)
    s["out_strides"] = (h * n * d, d, n * d, 1) if s["arrangement"] == "heads" else (n * h * d, h * d, d, 1)
    s["out"] = _empty(out)
    s["dx"] = _empty(out) if s["train"] else None
    if own:
        be = _backend()
        s["plan"] = be.rope_plan(s["rot"], base=ROPE_BASE, layout=s["layout"], scaling=s["scaling"], factor=ROPE_FACTOR, original_len=ROPE_LENGTH,
                                 low=ROPE_LOW, high=ROPE_HIGH, scale=_rope_scale(s["scaling"]))
        be.synchronize()


def _prepare_dropout(s, gen):
    r, c = s["rows"], s["cols"]
    s["x"] = _normal(gen, r, c)
    s["b"] = 0.02 * _normal(gen, c) if s["bias"] else None
    s["res"] = _normal(gen, r, c) if s["residual"] else None
    s["g"] = _normal(gen, r, c) if s["train"] else None
    s["key"] = (0x9E3779B97F4A7C15 * (s["seed"] + 1)) % 2**64
    s["counter"] = 2**32 - 1000 + 977 * (s["seed"] % 1000)  # the counters of a long run pass 32 bits
    s["out"] = _empty(r, c)
    s["dx"] = _empty(r, c) if s["train"] else None
    s["db"] = _empty(c) if s["train"] and s["bias"] else None


def _prepare_gate(s, gen):
    t, e, k = s["tokens"], s["experts"], s["k"]
    s["logits"] = 2.0 * _normal(gen, t, e)
    if s["masked"]:
        shut = torch.rand(t, e, device=DEV, generator=gen) < 0.3
        pad = torch.rand(t, 1, device=DEV, generator=gen) < 0.1
        s["logits"].masked_fill_(shut | pad, -math.inf)
    s["dw"] = _normal(gen, t, k) if s["train"] else None
    s["w"] = _empty(t, k)
    s["ids"] = torch.zeros(t, k, device=DEV, dtype=torch.int64)
    s["dlogits"] = _empty(t, e) if s["train"] else None


def _prepare_experts(s, gen):
    t, e, k, c = s["tokens"], s["experts"], s["k"], s["cols"]
    liked = 1.0 * _normal(gen, 1, e) + _normal(gen, t, e)  # some experts are liked more than others
    s["ids"] = torch.argsort(liked, dim=1)[:, :k].contiguous()
    w = torch.rand(t, k, device=DEV, generator=gen) + 0.05
    s["w"] = w / w.sum(1, keepdim=True)
    if s["padded"]:
        pad = torch.randperm(t, device=DEV, generator=gen)[:_padded(t)]
        s["ids"][pad] = -1
        s["w"][pad] = 0.0
    s["x"] = _normal(gen, t, c)
    s["ys"] = _normal(gen, t * k, c)
    s["dy"] = _normal(gen, t, c) if s["train"] else None
    s["dxs"] = _normal(gen, t * k, c) if s["train"] else None
    s["place"] = torch.full((t, k), -1, device=DEV, dtype=torch.int64)
    s["order"] = torch.full((t * k,), -1, device=DEV, dtype=torch.int64)
    s["offsets"] = torch.zeros(e + 1, device=DEV, dtype=torch.int64)
    s["xs"], s["y"] = _empty(t * k, c), _empty(t, c)
    if s["train"]:
        s["dx"], s["dys"], s["dweights"] = _empty(t, c), _empty(t * k, c), _empty(t, k)


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    op = state["op"]
    if own:
        return {"rope": _own_rope, "dropout": _own_dropout, "gate": _own_gate, "experts": _own_experts}[op](state)
    return {"rope": _plain_rope, "dropout": _plain_dropout, "gate": _plain_gate, "experts": _plain_experts}[op](state)


def _buf(t):
    from ferro_b200.backend import DeviceBuffer
    return None if t is None else DeviceBuffer(t.view(-1))


def _own_rope(s):
    from ferro_b200.backend import View
    be = _backend()
    shape = (s["batch"], s["seq"], s["heads"], s["dim"])
    pos = _buf(s["pos"])
    out = View(_buf(s["out"]), s["out_strides"])
    be.rope_dev(View(_buf(s["x"]), s["strides"], s["offset"]), shape, s["plan"], positions=pos, start=s["start"], out=out)
    if not s["train"]:
        return {"out": s["out"]}
    dx = View(_buf(s["dx"]), s["out_strides"])
    be.rope_backward_dev(View(_buf(s["g"]), s["strides"], s["offset"]), shape, s["plan"], positions=pos, start=s["start"], out=dx)
    return {"out": s["out"], "dx": s["dx"]}


def _own_dropout(s):
    be = _backend()
    r, c, p = s["rows"], s["cols"], s["p"]
    be.dropout_dev(_buf(s["x"]), _buf(s["b"]), _buf(s["res"]), p, s["key"], s["counter"], r, c, out=_buf(s["out"]))
    if not s["train"]:
        return {"out": s["out"]}
    be.dropout_backward_dev(_buf(s["g"]), p, s["key"], s["counter"], r, c, want_dbias=s["bias"], dx=_buf(s["dx"]), dbias=_buf(s["db"]))
    return {"out": s["out"], "dx": s["dx"], "db": s["db"]}


def _own_gate(s):
    be = _backend()
    t, e, k = s["tokens"], s["experts"], s["k"]
    logits, w, ids = _buf(s["logits"]), _buf(s["w"]), _buf(s["ids"])
    be.moe_gate_dev(logits, t, e, k, renorm=s["renorm"], weights=w, ids=ids)
    if not s["train"]:
        return {"w": s["w"], "ids": s["ids"]}
    be.moe_gate_backward_dev(_buf(s["dw"]), logits, w, ids, t, e, k, renorm=s["renorm"], dlogits=_buf(s["dlogits"]))
    return {"w": s["w"], "ids": s["ids"], "dlogits": s["dlogits"]}


def _own_experts(s):
    be = _backend()
    t, e, k, c = s["tokens"], s["experts"], s["k"], s["cols"]
    w, ys = _buf(s["w"]), _buf(s["ys"])
    plan = be.moe_sort_dev(_buf(s["ids"]), t, k, e, place=_buf(s["place"]), order=_buf(s["order"]), offsets=_buf(s["offsets"]))
    be.moe_dispatch_dev(_buf(s["x"]), plan, c, out=_buf(s["xs"]))
    be.moe_combine_dev(ys, w, plan, c, out=_buf(s["y"]))
    got = {"place": s["place"], "order": s["order"], "offsets": s["offsets"], "xs": s["xs"], "y": s["y"]}
    if s["train"]:
        be.moe_dispatch_backward_dev(_buf(s["dxs"]), plan, c, out=_buf(s["dx"]))
        be.moe_combine_backward_dev(_buf(s["dy"]), ys, w, plan, c, dys=_buf(s["dys"]), dweights=_buf(s["dweights"]))
        got.update(dx=s["dx"], dys=s["dys"], dweights=s["dweights"])
    return got


# ---- the plain forms -------------------------------------------------------------------------------------------------

def _logical(s, flat):
    """[batch, seq, heads, dim] as a view of the case's storage."""
    return torch.as_strided(flat, (s["batch"], s["seq"], s["heads"], s["dim"]), s["strides"], s["offset"])


def _frequencies(rot, scaling):
    """Radians a position, one for each pair of channels, in 64 bits."""
    i = torch.arange(rot // 2, device=DEV, dtype=torch.float64)
    base = ROPE_BASE * ROPE_FACTOR ** (rot / (rot - 2)) if scaling == "base" else ROPE_BASE
    f = base ** (-2.0 * i / rot)
    if scaling == "linear":
        f = f / ROPE_FACTOR
    if scaling == "by_parts":  # whole turns within the original context decide between both
        keep = ((ROPE_LENGTH * f / (2 * math.pi) - ROPE_LOW) / (ROPE_HIGH - ROPE_LOW)).clamp(0.0, 1.0)
        f = f / ROPE_FACTOR * (1 - keep) + f * keep
    return f


def _plain_rope(s):
    pos = s["pos"] if s["pos"] is not None else (torch.arange(s["seq"], device=DEV) + s["start"])[None, :]
    angle = pos.double()[:, :, None, None] * _frequencies(s["rot"], s["scaling"])  # 64 bits: positions may be far
    m = _rope_scale(s["scaling"])
    cos, sin = (angle.cos() * m).float(), (angle.sin() * m).float()
    out = _turned(s, _logical(s, s["x"]), cos, sin)
    if not s["train"]:
        return {"out": out}
    return {"out": out, "dx": _turned(s, _logical(s, s["g"]), cos, -sin)}


def _turned(s, x, cos, sin):
    rot = s["rot"]
    out = x.clone(memory_format=torch.contiguous_format)
    if s["layout"] == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        out[..., :rot // 2] = a * cos - b * sin
        out[..., rot // 2:rot] = b * cos + a * sin
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        out[..., 0:rot:2] = a * cos - b * sin
        out[..., 1:rot:2] = b * cos + a * sin
    return out.transpose(1, 2).contiguous() if s["arrangement"] == "heads" else out


def _philox(blocks, first, key):
    """Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011) at counters first, first + 1, ...: [blocks, 4] words in i64."""
    low = 0xFFFFFFFF
    n = torch.arange(blocks, device=DEV, dtype=torch.int64) + first
    c0, c1, c2, c3 = n & low, (n >> 32) & low, torch.zeros_like(n), torch.zeros_like(n)
    k0, k1 = key & low, key >> 32
    for _ in range(10):
        p, q = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((q >> 32) & low) ^ c1 ^ k0, q & low, ((p >> 32) & low) ^ c3 ^ k1, p & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], 1)


def _drop_numbers(p):
    """(smallest word that keeps its element, factor of the kept) for a probability held in f32."""
    p = float(np.float32(p))
    return int(round(p * 2.0**32)), float(np.float32(1.0 / (1.0 - p)))


def _plain_dropout(s):
    r, c = s["rows"], s["cols"]
    least, factor = _drop_numbers(s["p"])
    keep = (_philox((r * c + 3) // 4, s["counter"], s["key"]) >= least).view(-1)[:r * c].view(r, c)
    scale = keep.float() * factor
    z = s["x"] if s["b"] is None else s["x"] + s["b"]
    out = z * scale
    if s["res"] is not None:
        out = out + s["res"]
    if not s["train"]:
        return {"out": out}
    dx = s["g"] * scale
    return {"out": out, "dx": dx, "db": dx.sum(0) if s["bias"] else None}


def _plain_gate(s):
    logits, k = s["logits"], s["k"]
    best, at = torch.sort(logits, dim=1, descending=True, stable=True)  # equal ones stay in the order of their numbers
    best, ids = best[:, :k], at[:, :k]
    chosen = best > -math.inf  # what is masked is never chosen
    ids = torch.where(chosen, ids, -1)
    top = best[:, :1].clamp(min=-3.4e38)
    mass = torch.exp(best - top)
    total = mass.sum(1, keepdim=True) if s["renorm"] else torch.exp(logits - top).sum(1, keepdim=True)
    total = torch.where(total > 0, total, 1.0)
    w = mass / total
    if not s["train"]:
        return {"w": w, "ids": ids}
    dot = (w * s["dw"]).sum(1, keepdim=True)
    if s["renorm"]:
        dlogits = torch.zeros_like(logits)
        share = w * (s["dw"] - dot)
    else:
        dlogits = -torch.exp(logits - top) / total * dot
        share = w * s["dw"]
    dlogits.scatter_add_(1, at[:, :k], torch.where(chosen, share, 0.0))
    return {"w": w, "ids": ids, "dlogits": dlogits}


def _plain_experts(s):
    t, e, k = s["tokens"], s["experts"], s["k"]
    flat = s["ids"].view(-1)
    key = torch.where(flat >= 0, flat, e)  # what goes nowhere sorts behind the last expert
    rank = torch.sort(key, stable=True)[1]
    gone = flat < 0
    place = torch.empty_like(flat)
    place[rank] = torch.arange(t * k, device=DEV)
    ends = torch.searchsorted(key[rank], torch.arange(e + 1, device=DEV), right=False)
    total = (~gone).sum()
    filled = torch.arange(t * k, device=DEV) < total
    order = torch.where(filled, rank, -1)
    xs = torch.where(filled[:, None], s["x"][rank // k], 0.0)
    here = (~gone).view(t, k, 1)
    mine = torch.where(here, s["ys"][place].view(t, k, -1), 0.0)
    y = (mine * s["w"][:, :, None]).sum(1)
    got = {"place": torch.where(gone, -1, place).view(t, k), "order": order, "offsets": ends, "xs": xs, "y": y}
    if s["train"]:
        got["dx"] = torch.where(here, s["dxs"][place].view(t, k, -1), 0.0).sum(1)
        got["dys"] = torch.where(filled[:, None], s["dy"][rank // k] * s["w"].view(-1)[rank][:, None], 0.0)
        got["dweights"] = (mine * s["dy"][:, None, :]).sum(2)
    return got


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "dropout": _exact_dropout, "gate": _exact_gate, "experts": _exact_experts}[case["op"]](s)


def _exact_rope(s):
    rot, half = s["rot"], s["rot"] // 2
    base, theta = ROPE_BASE, []
    if s["scaling"] == "base":
        base *= ROPE_FACTOR ** (rot / (rot - 2))
    for i in range(half):
        f = math.pow(base, -2.0 * i / rot)
        if s["scaling"] == "linear":
            f /= ROPE_FACTOR
        elif s["scaling"] == "by_parts":
            g = min(1.0, max(0.0, (ROPE_LENGTH * f / (2 * math.pi) - ROPE_LOW) / (ROPE_HIGH - ROPE_LOW)))
            f *= g + (1 - g) / ROPE_FACTOR
        theta.append(f)
    where = s["pos"] if s["pos"] is not None else torch.arange(s["start"], s["start"] + s["seq"], device=DEV).expand(s["batch"], -1)
    turn = torch.polar(torch.full((), _rope_scale(s["scaling"]), device=DEV, dtype=torch.float64),
                       where.double()[..., None, None] * torch.tensor(theta, device=DEV, dtype=torch.float64))

    def turned(flat, by):
        v = _logical(s, flat).double()
        part = v[..., :rot]
        part = part.unflatten(-1, (2, half)).transpose(-1, -2) if s["layout"] == "half" else part.unflatten(-1, (half, 2))
        z = torch.view_as_real(torch.view_as_complex(part.contiguous()) * by)
        z = z.transpose(-1, -2) if s["layout"] == "half" else z
        v = torch.cat([z.reshape(*v.shape[:-1], rot), v[..., rot:]], -1)
        return v.permute(0, 2, 1, 3).contiguous() if s["arrangement"] == "heads" else v

    out = {"out": turned(s["x"], turn)}
    if s["train"]:
        out["dx"] = turned(s["g"], turn.conj())
    return out


def _exact_dropout(s):
    n, low = s["rows"] * s["cols"], np.uint64(0xFFFFFFFF)
    at = np.uint64(s["counter"]) + np.arange((n + 3) // 4, dtype=np.uint64)
    half = np.uint64(32)
    v = [at & low, at >> half, np.zeros_like(at), np.zeros_like(at)]
    for i in range(10):
        ka = np.uint64(((s["key"] & 0xFFFFFFFF) + i * 0x9E3779B9) & 0xFFFFFFFF)
        kb = np.uint64(((s["key"] >> 32) + i * 0xBB67AE85) & 0xFFFFFFFF)
        a, b = v[0] * np.uint64(0xD2511F53), v[2] * np.uint64(0xCD9E8D57)
        v = [(b >> half) ^ v[1] ^ ka, b & low, (a >> half) ^ v[3] ^ kb, a & low]
    words = np.stack(v, 1).reshape(-1)[:n]
    p = float(np.float32(s["p"]))
    kept = torch.from_numpy(words >= np.uint64(round(p * 2**32))).to(DEV).view(s["rows"], s["cols"])
    z = s["x"].double() + (0 if s["b"] is None else s["b"].double())
    out = torch.where(kept, z / (1.0 - p), 0.0) + (0 if s["res"] is None else s["res"].double())
    if not s["train"]:
        return {"out": out}
    dx = torch.where(kept, s["g"].double() / (1.0 - p), 0.0)
    return {"out": out, "dx": dx, "db": dx.sum(0) if s["bias"] else None}


def _exact_gate(s):
    l, k = s["logits"].double(), s["k"]
    none = torch.isinf(l).all(1, keepdim=True)
    left, member = l.clone(), torch.zeros_like(l, dtype=torch.bool)
    picks = []
    for _ in range(k):  # the greatest that is left, the lowest number among equals
        top = left.max(1, keepdim=True)[0]
        first = (left == top).int().argmax(1, keepdim=True)
        picks.append((first, top > -math.inf))
        member.scatter_(1, first, member.gather(1, first) | (top > -math.inf))
        left = left.scatter(1, first, -math.inf)
    pool = l.masked_fill(~member, -math.inf) if s["renorm"] else l
    prob = torch.softmax(pool.masked_fill(none, 0.0), 1).masked_fill(none, 0.0)
    at, real = torch.cat([p for p, _ in picks], 1), torch.cat([r for _, r in picks], 1)
    w = prob.gather(1, at) * real
    if not s["train"]:
        return {"w": w, "ids": None}
    up = torch.zeros_like(l).scatter_add_(1, at, s["dw"].double() * real)
    return {"w": w, "ids": None, "dlogits": prob * (up - (prob * up).sum(1, keepdim=True))}


def _exact_experts(s):
    t, k, c = s["tokens"], s["k"], s["cols"]
    ids = s["ids"].view(-1).cpu().numpy()
    slots = np.concatenate([np.flatnonzero(ids == e) for e in range(s["experts"])])  # assignments in the order of their rows
    m = len(slots)
    slot = torch.from_numpy(slots).to(DEV)
    tok = slot // k
    w = s["w"].view(-1)[slot].double()[:, None]

    def back(rows):
        return torch.zeros(t, c, device=DEV, dtype=torch.float64).index_add_(0, tok, rows)

    def spread(rows):
        return torch.cat([rows, torch.zeros(t * k - m, c, device=DEV, dtype=torch.float64)])

    ys = s["ys"][:m].double()
    got = {"place": None, "order": None, "offsets": None, "xs": spread(s["x"].double()[tok]), "y": back(ys * w)}
    if s["train"]:
        got["dx"] = back(s["dxs"][:m].double())
        up = s["dy"].double()[tok]
        got["dys"] = spread(up * w)
        got["dweights"] = torch.zeros(t * k, device=DEV, dtype=torch.float64).index_copy_(0, slot, (ys * up).sum(1)).view(t, k)
    return got
