"""Attention over a bounded context, as measurable cases.

A robot that runs for hours cannot keep every token it has seen.  Two things
bound its context: a sliding window with a few first tokens that stay visible
(sinks), and a K/V cache held in 8 or 4 bits.  The operators:

* ``window``: attention over dense bf16 K and V where a query at position p sees
  the keys of positions (p - window, p] and of the first ``sinks`` positions;
* ``store``: new K and V rows quantised as they are written into a microscaled
  cache (blocks of 32 values of a row share a power of two; values are e4m3 or
  e2m1), and the whole cache read back as bf16;
* ``attend``: attention of one or more new queries over such a cache;
* ``step``: both in one call, as a stream of tokens uses them (its outputs are the
  attention's and the new rows as the cache holds them then).

The plain forms are elementary torch operations in 32 bits.  ``exact`` restates
every operator in float64 and quantises by another route.
"""

import math
import os
import sys

import torch

own = False

BF16 = torch.bfloat16
F32 = torch.float32
F64 = torch.float64
D = 64                      # head dimension of every attention of the framework
BLOCK = 32                  # values that share a scale
SCALE = 1.0 / math.sqrt(D)
E_MIN, E_MAX = -110, 126    # exponents of a block's scale
LIMIT = 1.5 * 2.0 ** 127    # magnitudes above it are stored as it


# ------------------------------------------------------------------ cases ---
def listed():
    return [
        # one robot, one new token after a prefix: latency is all that counts
        _step("step_1x241", 1, 15, 5, "mxfp8", 241),
        # 32 robots far into their run, each with a window and four sinks
        _step("step_32x20000_w4096", 32, 15, 5, "mxfp4", 20000, window=4096, sinks=4),
        # the prefixes of a batch of 32 observations into the cache
        _store("store_32x241", 32, 5, "mxfp8", 0, 241),
        # four long recordings loaded at once, of uneven lengths
        _store("store_4x32768", 4, 5, "mxfp4", 0, 32768, ragged=True),
        # one long context, an odd length: a single sequence has to fill the chip
        _attend("attend_1x100003", 1, 15, 5, "mxfp4", 100003),
        # a batch of uneven ordinary contexts
        _attend("attend_32x8192", 32, 15, 5, "mxfp8", 8192, ragged=True),
        # the largest cache: sixteen long contexts
        _attend("attend_16x65536", 16, 15, 5, "mxfp4", 65536),
        # a chunk of 50 action rows of each of 32 robots over its context
        _attend("attend_32x50x1024", 32, 15, 5, "mxfp4", 1024, rows=50),
        # a long prompt fed in pieces: 1000 rows at the end of a windowed context
        _attend("attend_2x1000x8192_w2048", 2, 15, 5, "mxfp8", 8192, rows=1000, window=2048,
                sinks=4),
        # one short prompt, the smallest windowed call
        _window("window_1x241", 1, 15, 5, 241, 64, 1),
        # uneven padded prompts, a head of K and V for every query head
        _window("window_8x2000", 8, 12, 12, 2000, 500, 4, ragged=True),
        # two long prompts
        _window("window_2x16384", 2, 15, 5, 16384, 4096, 4),
    ]


def _step(name, batch, heads, kv_heads, fmt, held, rows=1, window=0, sinks=0, ragged=False):
    return dict(name=name, op="step", batch=batch, heads=heads, kv_heads=kv_heads, fmt=fmt,
                held=held, rows=rows, window=window, sinks=sinks, ragged=ragged)


def _attend(name, batch, heads, kv_heads, fmt, held, rows=1, window=0, sinks=0, ragged=False):
    """``rows`` queries, the last rows of ``held``."""
    return dict(_step(name, batch, heads, kv_heads, fmt, held, rows, window, sinks, ragged),
                op="attend")


def _store(name, batch, kv_heads, fmt, held, rows, ragged=False):
    return dict(name=name, op="store", batch=batch, kv_heads=kv_heads, fmt=fmt, held=held,
                rows=rows, ragged=ragged)


def _window(name, batch, heads, kv_heads, length, window, sinks, ragged=False):
    return dict(name=name, op="window", batch=batch, heads=heads, kv_heads=kv_heads,
                length=length, window=window, sinks=sinks, ragged=ragged)


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(15, 5), (15, 5), (12, 12), (8, 1), (16, 2), (32, 8)]


def draw(rng):
    op = rng.choice(["step", "attend", "attend", "store", "window"])
    heads, kv = rng.choice(HEADS)
    fmt = rng.choice(["mxfp4", "mxfp8"])
    ragged = rng.random() < 0.5
    batch = _log(rng, 1, 64)
    if op == "window":
        length = min(_log(rng, 1, 16384), 200000 // (batch * heads))
        window = _log(rng, 1, 4096)
        return _strip(_window("", batch, heads, kv, max(1, length), window, rng.randint(0, 8),
                              ragged))
    if op == "store":
        rows = max(1, min(_log(rng, 1, 32768), 400000 // (batch * kv)))
        held = rng.choice([0, rng.randint(0, max(0, min(2000, 200000 // (batch * kv) - 1)))])
        return _strip(_store("", batch, kv, fmt, held, rows, ragged))
    window, sinks = (_log(rng, 16, 4096), rng.randint(0, 8)) if rng.random() < 0.5 else (0, 0)
    rows = 1 if rng.random() < 0.6 else _log(rng, 2, 1000)
    held = max(rows, min(_log(rng, 1, 100000), 5000000 // (batch * kv),
                         200000000 // (batch * heads * rows)))
    make = _step if op == "step" else _attend
    return _strip(make("", batch, heads, kv, fmt, held, rows, window, sinks, ragged))


def _strip(case):
    del case["name"]
    return case


def _uneven(n, case):
    """Per sequence a number of up to ``n``: all of them, or down to half."""
    b = case["batch"]
    if not case["ragged"]:
        return [n] * b
    return [n - (i * (n // 2)) // max(1, b - 1) for i in range(b)]


def _held(case):
    return _uneven(case["held"], case)


def _rows(case):
    """New rows per sequence (a query of ``attend`` is one of the rows held)."""
    return [min(r, h) if case["op"] == "attend" else r
            for r, h in zip(_uneven(case["rows"], case), _held(case))]


def _totals(case):
    """Tokens per sequence once the new rows are in."""
    return _held(case) if case["op"] == "attend" else [h + r for h, r in
                                                       zip(_held(case), _rows(case))]


# ----------------------------------------------------------------- inputs ---
class _Gen:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.g, device="cuda", dtype=F32)

    def keys(self, batch, rows, heads):
        """Keys have a few channels far larger than the others."""
        gain = torch.exp(0.3 * self.normal(heads, D))
        gain[:, 5] *= 4.0
        gain[:, 40] *= 4.0
        return (self.normal(batch, rows, heads, D) * gain).to(BF16).view(batch, rows, heads * D)

    def values(self, batch, rows, heads):
        return self.normal(batch, rows, heads * D).to(BF16)


def _inputs(case, seed):
    g = _Gen(seed)
    b, kv = case["batch"], case["kv_heads"]
    if case["op"] == "window":
        n = case["length"]
        return dict(q=g.values(b, n, case["heads"]), k=g.keys(b, n, kv), v=g.values(b, n, kv))
    inp = dict(k_held=g.keys(b, case["held"], kv), v_held=g.values(b, case["held"], kv))
    if case["op"] != "store":
        inp["q"] = g.values(b, case["rows"], case["heads"])
    if case["op"] != "attend":
        inp.update(k=g.keys(b, case["rows"], kv), v=g.values(b, case["rows"], kv))
    return inp


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    inp = _inputs(case, seed)
    state = dict(case=case, **{n: inp[n] for n in ("q", "k", "v") if n in inp})
    if case["op"] == "window":
        state["lens"] = _i32(_uneven(case["length"], case)) if case["ragged"] else None
        if own:
            _import_own()
            state["out"] = torch.empty_like(inp["q"])
        return state
    held, rows = _held(case), _rows(case)
    state["held"] = _i32(held)
    state["counts"] = _i32(rows) if case["ragged"] else None
    if own:
        _import_own()
        from smolvla.kv_cache import KVCache
        window = case.get("window") or None
        cache = KVCache(case["batch"], case["kv_heads"], fmt=case["fmt"],
                        max_len=None if window else max(_totals(case)), window=window,
                        sinks=case.get("sinks", 0), rows=case["rows"])
        if case["held"]:
            cache.append(inp["k_held"], inp["v_held"], counts=state["held"])
        state["cache"] = cache
        return state
    # a plain program keeps the positions that a later query can still see
    if case.get("window"):
        keep = case["window"] + case["rows"]
        near = torch.arange(keep, device="cuda") + (state["held"][:, None].long() - keep)
        near = torch.where(near < case["sinks"], -1, near)
        first = torch.arange(case["sinks"], device="cuda").expand(case["batch"], -1)
        pos = torch.cat([first, near], 1)
    else:
        pos = torch.arange(case["held"], device="cuda").expand(case["batch"], -1)
    pos = torch.where(pos < state["held"][:, None], pos, -1)
    state["pos"] = pos
    at = pos.clamp(min=0)[:, :, None].expand(-1, -1, case["kv_heads"] * D)
    for name in ("k", "v"):
        state[name + "_codes"], state[name + "_exps"] = _quantise(
            torch.gather(inp[name + "_held"], 1, at), case["fmt"])
    return state


def _import_own():
    root = os.path.join(os.getcwd(), "vla-to-npu_amd")
    if root not in sys.path:
        sys.path.insert(0, root)


# ------------------------------------------------------- the plain program ---
# magnitudes of the element codes, and per format the largest one, the exponent
# of the smallest normal one and the fraction bits
FP4 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
FP8 = [(m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
       for e in range(16) for m in range(8)][:127]
FORMATS = {"mxfp4": (FP4, 6.0, 0, 1), "mxfp8": (FP8, 448.0, -6, 3)}


def _quantise(x, fmt):
    """bf16 [..., n] -> (codes uint8, one a value or two a byte; exponents int8
    of the blocks of 32)."""
    table, top, e_low, frac = FORMATS[fmt]
    x = x.float().unflatten(-1, (-1, BLOCK)).clamp(-LIMIT, LIMIT)
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True))
    mt, et = math.frexp(top)
    e = (e - et + (m > mt).int()).clamp(E_MIN, E_MAX)
    y = torch.ldexp(x.abs(), -e)
    step = torch.frexp(y)[1] - 1
    step = torch.where(y == 0, e_low, step.clamp(min=e_low)) - frac
    y = torch.ldexp(torch.round(torch.ldexp(y, -step)), step)
    at = torch.tensor(table, device=x.device)
    codes = torch.searchsorted(at, y.contiguous()).to(torch.uint8)
    codes |= torch.signbit(x).to(torch.uint8) << (3 if fmt == "mxfp4" else 7)
    codes = codes.flatten(-2)
    if fmt == "mxfp4":
        codes = codes[..., 0::2] | codes[..., 1::2] << 4
    return codes, e.squeeze(-1).to(torch.int8)


def _values(codes, exps, fmt):
    """What the codes stand for, in fp32."""
    table = torch.tensor(FORMATS[fmt][0], device=codes.device)
    if fmt == "mxfp4":
        table = torch.cat([table, -table])
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    else:
        nan = table.new_full((1,), math.nan)
        table = torch.cat([table, nan, -table, nan])
    x = table[codes.int()].unflatten(-1, (-1, BLOCK))
    return torch.ldexp(x, exps[..., None].int()).flatten(-2)


def _heads(x, heads):
    """[B, n, heads * D] -> [B, heads, n, D]"""
    return x.unflatten(-1, (heads, D)).transpose(1, 2).contiguous()


def _softmax_product(q, k, v, seen):
    """q [B, kv, G * T, D], k and v [B, kv, n, D], seen [B, 1, G * T, n]; a row
    that sees nothing gives zeros."""
    s = torch.matmul(q, k.transpose(-1, -2)) * SCALE
    s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total == 0, 1.0, total)


def _visible(qpos, kpos, window, sinks):
    """[..., T] and [..., n] positions -> [..., T, n]"""
    qpos, kpos = qpos[..., :, None], kpos[..., None, :]
    seen = (kpos <= qpos) & (kpos >= 0)
    if window:
        seen &= (kpos > qpos - window) | (kpos < sinks)
    return seen


def _plain_cache(state):
    """Quantises the new rows; all rows held then, and their positions."""
    case = state["case"]
    held, fmt, pos = state["held"], case["fmt"], state["pos"]
    codes = {n: (state[n + "_codes"], state[n + "_exps"]) for n in ("k", "v")}
    rows = case["rows"]
    t = torch.arange(rows, device="cuda")
    counts = _i32(_rows(case)) if state["counts"] is None else state["counts"]
    real = t < counts[:, None]
    if case["op"] == "attend":
        at = held[:, None] - counts[:, None] + t
    else:
        at = held[:, None] + t
        for n in ("k", "v"):
            new = _quantise(state[n], fmt)
            codes[n] = tuple(torch.cat(pair, 1) for pair in zip(codes[n], new))
        pos = torch.cat([pos, torch.where(real, at, -1)], 1)
    k, v = (_values(*codes[n], fmt) for n in ("k", "v"))
    return k, v, pos, torch.where(real, at, -1)


def _plain_store(state):
    case = state["case"]
    k, v, pos, _ = _plain_cache(state)
    n = case["held"] + case["rows"]
    out = []
    for x in (k, v):
        full = x.new_zeros(x.shape[0], n + 1, x.shape[2])
        where = torch.where(pos < 0, n, pos).long()[:, :, None].expand_as(x)
        out.append(full.scatter_(1, where, x)[:, :n].to(BF16))
    return out


def _plain_attend(state):
    case = state["case"]
    heads, kv, rows = case["heads"], case["kv_heads"], case["rows"]
    k, v, kpos, qpos = _plain_cache(state)
    seen = _visible(qpos, kpos, case["window"], case["sinks"])
    q = _heads(state["q"].float(), heads).view(case["batch"], kv, -1, D)
    group = heads // kv
    o = _softmax_product(q, _heads(k, kv), _heads(v, kv), seen.repeat(1, group, 1)[:, None])
    o = o.view(case["batch"], heads, rows, D).transpose(1, 2)
    o = o.reshape(case["batch"], rows, heads * D).to(BF16)
    if case["op"] == "attend":
        return o
    real = (qpos >= 0)[:, :, None]
    return [o] + [torch.where(real, x[:, -rows:], 0.0).to(BF16) for x in (k, v)]


PIECE = 1024       # query rows at a time, over the keys that they can see


def _plain_window(state):
    case = state["case"]
    b, heads, kv, n = case["batch"], case["heads"], case["kv_heads"], case["length"]
    window, sinks = case["window"], case["sinks"]
    q, k, v = (_heads(state[x].float(), h) for x, h in (("q", heads), ("k", kv), ("v", kv)))
    where = torch.arange(n, device="cuda")
    kpos = where.expand(b, -1)
    if state["lens"] is not None:
        kpos = torch.where(kpos < state["lens"][:, None], kpos, -1)
    out = torch.empty_like(q)
    for at in range(0, n, PIECE):
        end = min(n, at + PIECE)
        lo = max(0, at - window + 1)
        near = where[lo:end]
        keys = torch.cat([where[:min(sinks, lo)], near])
        seen = _visible(where[at:end].expand(b, -1), kpos[:, keys], window, sinks)
        g = heads // kv
        rows = q[:, :, at:end].reshape(b, kv, -1, D)
        o = _softmax_product(rows, k[:, :, keys], v[:, :, keys], seen.repeat(1, g, 1)[:, None])
        out[:, :, at:end] = o.view(b, heads, end - at, D)
    return out.transpose(1, 2).reshape(b, n, heads * D).to(BF16)


# --------------------------------------------------------------------- run ---
def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"window": _plain_window, "store": _plain_store, "attend": _plain_attend,
                "step": _plain_attend}[op](state)
    if op == "window":
        from smolvla import ops
        return ops.attention(state["q"], state["k"], state["v"], state["out"], case["heads"],
                             case["kv_heads"], mask="window", window=case["window"],
                             sinks=case["sinks"], lens=state["lens"])
    cache = state["cache"]
    if op == "store":
        cache.append(state["k"], state["v"], counts=state["counts"], at=state["held"])
        return cache.read(0, case["held"] + case["rows"])
    if op == "attend":
        return cache.attend(state["q"], case["heads"], counts=state["counts"])
    out = cache.step(state["q"], state["k"], state["v"], case["heads"], counts=state["counts"],
                     at=state["held"])
    return [out, *cache.read(state["held"], case["rows"])]


# -------------------------------------------------------------------- work ---
def _pairs(first, rows, total, window, sinks):
    """(query, key) pairs of the rows at positions first .. first + rows - 1
    among ``total`` keys, and the number of keys that any of them sees."""
    pairs = 0
    for p in range(first, first + rows):
        lo = max(0, p - window + 1) if window else 0
        pairs += max(0, min(p + 1, total) - lo) + min(sinks, lo, total)
    lo = max(0, first - window + 1) if window else 0
    return pairs, max(0, min(first + rows, total) - lo) + min(sinks, lo, total)


def work(case):
    b, kv = case["batch"], case["kv_heads"]
    if case["op"] == "window":
        n = case["length"]
        pairs = keys = 0
        for total in _uneven(n, case):
            p, s = _pairs(0, n, total, case["window"], case["sinks"])
            pairs, keys = pairs + p, keys + s
        h = case["heads"]
        return {"bytes": 2 * D * (2 * b * n * h + 2 * keys * kv), "flops": 4 * D * h * pairs}
    per_row = 2 * kv * (D // 2 if case["fmt"] == "mxfp4" else D) + 2 * kv * D // BLOCK
    new = sum(_rows(case))
    if case["op"] == "store":
        total, n = sum(_totals(case)), case["held"] + case["rows"]
        return {"bytes": 2 * new * kv * D * 2 + (new + total) * per_row + 2 * b * n * kv * D * 2,
                "flops": 8 * kv * D * (new + total)}
    pairs = keys = 0
    for total, r in zip(_totals(case), _rows(case)):
        p, s = _pairs(total - r, r, total, case["window"], case["sinks"])
        pairs, keys = pairs + p, keys + s
    moved = keys * per_row + 2 * 2 * b * case["rows"] * case["heads"] * D
    if case["op"] == "step":
        moved += 2 * 2 * (new + b * case["rows"]) * kv * D
    return {"bytes": moved, "flops": 4 * D * case["heads"] * pairs}


# ------------------------------------------------------------------- exact ---
def _stored64(x, fmt):
    """The value that each element of a bf16 row is stored as: the nearest of the
    format's values times the smallest power of two that loses no element to
    saturation; of two equally near values the one with the even code."""
    table = torch.tensor(FORMATS[fmt][0], dtype=F64, device=x.device)
    x = x.double().clamp(-LIMIT, LIMIT).reshape(*x.shape[:-1], -1, BLOCK)
    top = x.abs().max(-1, keepdim=True).values
    unit = torch.full_like(top, 2.0 ** E_MIN)
    power = torch.exp2(torch.ceil(torch.log2(top / table[-1])))       # within one step of it
    for trial in (power * 2, power, power / 2):
        unit = torch.where((top <= table[-1] * trial) & (trial >= 2.0 ** E_MIN), trial, unit)
    y = x.abs() / unit
    between = (table[1:] + table[:-1]) / 2
    low = torch.bucketize(y, between)                                 # a tie goes down ...
    high = torch.bucketize(y, between, right=True)                    # ... or up
    code = torch.where(low % 2 == 0, low, high)
    return (torch.copysign(table[code], x) * unit).reshape(*x.shape[:-2], -1)


def _exact_rows(q, k, v, qpos, kpos, window, sinks):
    """float64 attention of one sequence's query head: q [T, D], k and v [n, D]."""
    s = q @ k.T / math.sqrt(D)
    hide = (kpos[None, :] > qpos[:, None])
    if window:
        hide |= (kpos[None, :] + window <= qpos[:, None]) & (kpos[None, :] >= sinks)
    s.masked_fill_(hide, -math.inf)
    s -= s.max(-1, keepdim=True).values.nan_to_num(neginf=0.0)
    s.exp_()
    total = s.sum(-1, keepdim=True)
    return (s @ v) / total.masked_fill(total == 0, 1.0)


def exact(case, seed):
    inp = _inputs(case, seed)
    b, kv = case["batch"], case["kv_heads"]
    if case["op"] == "store":
        n = case["held"] + case["rows"]
        out = []
        for name in ("k", "v"):
            full = torch.zeros(b, n, kv * D, dtype=F64, device="cuda")
            for i, (h, r) in enumerate(zip(_held(case), _rows(case))):
                rows = torch.cat([inp[name + "_held"][i, :h], inp[name][i, :r]])
                full[i, :h + r] = _stored64(rows, case["fmt"])
            out.append(full)
        return out
    heads = case["heads"]
    out = torch.zeros(*inp["q"].shape, dtype=F64, device="cuda")
    for i in range(b):
        if case["op"] == "window":
            n = _uneven(case["length"], case)[i]
            rows, first = case["length"], 0
            k, v = inp["k"][i, :n].double(), inp["v"][i, :n].double()
        else:
            rows, n = _rows(case)[i], _totals(case)[i]
            first = n - rows
            parts = [(inp["k_held"][i, :_held(case)[i]], inp["v_held"][i, :_held(case)[i]])]
            if case["op"] == "step":
                parts.append((inp["k"][i, :rows], inp["v"][i, :rows]))
            k, v = (_stored64(torch.cat(p), case["fmt"]) for p in zip(*parts))
        kpos = torch.arange(n, device="cuda")
        for at in range(0, rows, 4096):
            end = min(rows, at + 4096)
            qpos = torch.arange(first + at, first + end, device="cuda")
            for h in range(heads):
                c = (h * kv // heads) * D
                out[i, at:end, h * D:(h + 1) * D] = _exact_rows(
                    inp["q"][i, at:end, h * D:(h + 1) * D].double(), k[:, c:c + D], v[:, c:c + D],
                    qpos, kpos, case["window"], case["sinks"])
    if case["op"] != "step":
        return out
    stored = []
    for name in ("k", "v"):
        real = torch.arange(case["rows"], device="cuda") < _i32(_rows(case))[:, None]
        stored.append(_stored64(inp[name], case["fmt"]) * real[:, :, None])
    return [out] + stored
