"""The bounded context in float64 on the CPU: microscaled storage, windowed
attention with sinks, and a K/V cache that is a plain list of rows."""

import math

import torch

D = 64
FP4 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
FP8 = [(m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
       for e in range(16) for m in range(8)][:127]
TABLES = {"mxfp4": FP4, "mxfp8": FP8}
LIMIT = 1.5 * 2.0 ** 127


def stored(x, fmt):
    """The values a bf16 tensor ``[..., 32 n]`` is stored as, element by element
    from the definition: the nearest table entry (ties to the even index) times
    the smallest power of two, 2^-110 to 2^126, that lets the largest of 32 fit."""
    table = torch.tensor(TABLES[fmt], dtype=torch.float64)
    blocks = x.double().reshape(-1, 32)
    finite = torch.isfinite(blocks).all(1)
    y = torch.where(finite[:, None], blocks, 0.0).clamp(-LIMIT, LIMIT)
    top = y.abs().max(1).values
    unit = torch.full_like(top, 2.0 ** -110)
    for e in range(-109, 127):
        unit = torch.where(top > table[-1] * unit, 2.0 ** e, unit)
    a = (y / unit[:, None]).abs()
    i = torch.searchsorted(table, a).clamp(1, len(table) - 1)      # table[i-1] < a <= table[i]
    up, down = table[i] - a, a - table[i - 1]
    i = torch.where((down < up) | ((down == up) & (i % 2 == 1)), i - 1, i)
    out = torch.copysign(table[i], y) * unit[:, None]
    return torch.where(finite[:, None], out, math.nan).reshape(x.shape)


def attention(q, k, v, qpos, kpos, hq, hkv, window=None, sinks=0, scale=None):
    """One sequence: ``q [T, hq * D]`` at positions ``qpos``, ``k`` / ``v [n, hkv * D]``
    at ``kpos``; returns the output and a bound on what a kernel may be off by that
    rounds its probabilities and its output to bf16 and keeps everything else in
    fp32: with weights w and |dw| <= e w,

        |do| <= e sum w |v - o| + 2^-8 |o|,   sum w |v - o| <= sum w |v| + |o|

    e = 2^-8 for the rounding (the sum of the weights takes the rounded ones),
    plus the scores' error: a product of 64 terms in fp32 is off by 64 2^-24
    sum |q k|, its scaling and exponent by 2^-23 of its value and 2^-22 more."""
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(q.shape[0], hq * D, dtype=torch.float64)
    bound = torch.zeros_like(out)
    seen = kpos[None, :] <= qpos[:, None]
    if window is not None:
        seen &= (kpos[None, :] > qpos[:, None] - window) | (kpos[None, :] < sinks)
    for h in range(hq):
        a = h * hkv // hq * D
        qh = q[:, h * D:(h + 1) * D].double()
        kh, vh = k[:, a:a + D].double(), v[:, a:a + D].double()
        for t in range(q.shape[0]):
            s = seen[t]
            if not s.any():
                continue
            x = (kh[s] @ qh[t]) * scale
            w = torch.exp(x - x.max())
            w = w / w.sum()
            size = (kh[s].abs() @ qh[t].abs()) * scale
            e = 2 ** -8 + float((64 * 2.0 ** -24 * size + 2.0 ** -23 * x.abs()).max()) * 2 + 2 ** -21
            o = w @ vh[s]
            out[t, h * D:(h + 1) * D] = o
            bound[t, h * D:(h + 1) * D] = (1.02 * e * (w @ vh[s].abs() + o.abs())
                                           + 2 ** -8 * 1.02 * o.abs() + 1e-30)
    return out, bound


class CacheRef:
    """Every row ever written, as stored."""

    def __init__(self, batch, hkv, fmt, window=None, sinks=0):
        self.k = [torch.zeros(0, hkv * D, dtype=torch.float64) for _ in range(batch)]
        self.v = [torch.zeros(0, hkv * D, dtype=torch.float64) for _ in range(batch)]
        self.hkv, self.fmt, self.window, self.sinks = hkv, fmt, window, sinks

    def append(self, k, v, counts=None, at=None):
        for b in range(len(self.k)):
            c = k.shape[1] if counts is None else int(counts[b])
            p = len(self.k[b]) if at is None else int(at[b])
            self.k[b] = torch.cat([self.k[b][:p], stored(k[b, :c].cpu(), self.fmt)])
            self.v[b] = torch.cat([self.v[b][:p], stored(v[b, :c].cpu(), self.fmt)])

    def attend(self, q, hq, counts=None, scale=None):
        out = torch.zeros(*q.shape, dtype=torch.float64)
        bound = torch.zeros_like(out)
        for b in range(len(self.k)):
            c = q.shape[1] if counts is None else int(counts[b])
            n = len(self.k[b])
            out[b, :c], bound[b, :c] = attention(
                q[b, :c].cpu(), self.k[b], self.v[b], torch.arange(n - c, n), torch.arange(n), hq,
                self.hkv, self.window, self.sinks, scale)
        return out, bound
