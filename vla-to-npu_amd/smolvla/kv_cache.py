"""A K/V cache in microscaled 8 or 4 bits and the attention over it.

The reference recomputes its whole prefix for every chunk (vla/vla.py:194-212);
a program that feeds a decoder layer token by token, or for longer than its
memory lasts, keeps the layer's keys and values here instead::

    cache = KVCache(batch, n_kv_heads, fmt="mxfp4", window=4096, sinks=4)
    cache.append(k, v)                    # a prompt, [B, T, n_kv_heads * 64]
    cache.attend(q, n_heads)              # its attention, [B, T, n_heads * 64]
    cache.step(q1, k1, v1, n_heads)       # one more token: both at once

Keys are stored as they come, so they carry their RoPE already.  Calls run on
the current stream, allocate with torch's allocator only and can be captured
in a HIP graph: the number of tokens lives on the device and moves on with
every replay.  Calls that write one cache must not overlap with other calls on
it.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

BF16 = torch.bfloat16
HEAD_DIM = 64
SCALE = 1.0 / math.sqrt(HEAD_DIM)
TOKENS = 32                     # tokens of a record
MAX_POS = 1 << 30               # positions stay below it
FORMATS = {"mxfp4": 4, "mxfp8": 8}


def _bad(name, t, batch, rows, width, device):
    """Why ``t`` is no bf16 ``[batch, rows, >= width]`` view on the device."""
    if not torch.is_tensor(t):
        return f"{name}: a tensor expected"
    if not t.is_cuda:
        return "smolvla ops take GPU tensors (no CPU fallback)"
    if t.device != device:
        return f"{name} on {t.device}, cache on {device}"
    if t.dim() == 3 and t.stride(2) != 1:
        return f"{name}: rows must be contiguous"
    return (f"{name}: bf16 [{batch}, {'rows' if rows is None else rows}, {width}] expected, got "
            f"{t.dtype} {tuple(t.shape)}")


class KVCache:
    """K and V of ``n_kv_heads`` heads of 64 for ``batch`` sequences, quantised
    as they are written (``fmt``: ``"mxfp4"``, e2m1 elements, or ``"mxfp8"``,
    e4m3; 32 values of a row share a power of two).

    ``max_len`` bounds the tokens of a sequence.  With ``window`` a query sees
    the last ``window`` tokens up to itself and the first ``sinks`` of the
    sequence; without ``max_len`` the cache is then the smallest one for calls
    of up to ``rows`` queries and the sequence may go on without end.
    """

    def __init__(self, batch, n_kv_heads, max_len=None, fmt="mxfp4", window=None, sinks=0,
                 rows=1, device=None):
        if fmt not in FORMATS:
            raise ValueError(f"fmt {fmt!r}: one of {sorted(FORMATS)} expected")
        for name, v in (("batch", batch), ("n_kv_heads", n_kv_heads), ("rows", rows)):
            if v < 1:
                raise ValueError(f"{name} must be positive, got {v}")
        if (window is None and sinks) or sinks < 0:
            raise ValueError("sinks: a number of first tokens beside a window")
        if window is not None and window < 1:
            raise ValueError(f"window must be positive, got {window}")
        if max_len is None and window is None:
            raise ValueError("a cache without a window needs max_len")
        if max_len is not None and max_len < 1:
            raise ValueError(f"max_len must be positive, got {max_len}")
        # a call of `rows` queries reaches window + rows - 1 tokens back, which
        # may begin and end inside a record
        ring = window + rows + TOKENS - 2 if max_len is None else max(1, max_len - sinks)
        self.batch, self.n_kv_heads, self.fmt = batch, n_kv_heads, fmt
        self.window, self.sinks = window, sinks
        self.max_rows = rows if max_len is None else None
        self.max_len = max_len
        self.ring = (ring + TOKENS - 1) // TOKENS * TOKENS
        if self.ring > MAX_POS or sinks > MAX_POS // 2 or batch * n_kv_heads > 65535:
            raise ValueError("KVCache: size not supported")
        self._lib = _lib.load()
        nbytes = self._lib.svla_kv_cache_bytes(batch, n_kv_heads, HEAD_DIM, FORMATS[fmt], sinks,
                                               self.ring)
        if nbytes <= 0:
            raise ValueError("KVCache: size not supported")
        self.device = torch.device(device if device is not None else "cuda")
        if self.device.type != "cuda":
            raise ValueError("smolvla ops take GPU tensors (no CPU fallback)")
        # (zeros: a record may be decoded before every token of it was written)
        self.data = torch.zeros(nbytes, dtype=torch.uint8, device=self.device)
        self.device = self.data.device
        self.state = torch.zeros(batch, 4, dtype=torch.int32, device=self.device)
        self._desc = _lib.KVCacheDesc(self.data.data_ptr(), self.state.data_ptr(), batch,
                                      n_kv_heads, HEAD_DIM, FORMATS[fmt], sinks, self.ring)
        self._ref = ctypes.byref(self._desc)
        self._scratch = {}

    @property
    def lengths(self):
        """Tokens per sequence, ``[B]`` int32 on the device (a view)."""
        return self.state[:, 0]

    def check(self):
        """Raise if a sequence is lost or has outgrown ``max_len`` (waits for the
        device)."""
        state = self.state.cpu()
        lost = (state[:, 1] == 0x7fffffff).nonzero().flatten().tolist()
        if lost:
            raise RuntimeError(f"KVCache: sequences {lost} were written at a position that they "
                               "had not reached; write them from position 0 again")
        if self.window is None:
            over = (state[:, 0] > self.max_len).nonzero().flatten().tolist()
            if over:
                raise RuntimeError(f"KVCache: sequences {over} hold more than {self.max_len} tokens")

    # ---------------------------------------------------------------- calls --
    def _view(self, name, t, rows, width, written=False):
        """(address, row stride, batch stride) of a bf16 ``[B, rows, >= width]``
        view; a stride that no index uses is any valid one."""
        try:
            b, r, w = t.shape
            sb, sr, sw = t.stride()
            ok = (b == self.batch and (rows is None or r == rows) and w >= width and sw == 1
                  and t.dtype is BF16 and t.device == self.device)
        except (ValueError, AttributeError):
            ok = False
        if not ok:
            raise ValueError(_bad(name, t, self.batch, rows, width, self.device))
        if written and b > 1 and not (sb >= (r - 1) * sr + width
                                      or sb >= width and sr >= (b - 1) * sb + width):
            raise ValueError(f"{name}: rows must not overlap")
        return t.data_ptr(), (sr if r > 1 else (w + 7) // 8 * 8), (sb if b > 1 else 0)

    def _new(self, rows, width):
        return torch.empty((self.batch, rows, width), dtype=BF16, device=self.device)

    def _ints(self, name, t):
        if t is None:
            return None
        if not (torch.is_tensor(t) and t.dtype is torch.int32 and t.dim() == 1
                and t.shape[0] == self.batch and (t.stride(0) == 1 or self.batch == 1)
                and t.device == self.device):
            raise ValueError(f"{name}: contiguous int32 [{self.batch}] tensor on {self.device} "
                             "expected")
        return t.data_ptr()

    def _call(self, name, *args):
        index = self.device.index
        if torch.cuda.current_device() == index:
            return _lib.call(name, self._ref, *args, torch._C._cuda_getCurrentRawStream(index))
        with torch.cuda.device(index):
            return _lib.call(name, self._ref, *args, torch._C._cuda_getCurrentRawStream(index))

    def reset(self):
        """Every sequence empty."""
        self._call("svla_kv_reset")

    def append(self, k, v, counts=None, at=None):
        """Quantise ``k``, ``v`` ``[B, T, n_kv_heads * 64]`` into the next
        positions of every sequence, or from position ``at[b]`` (int32
        ``[B]``; tokens behind it are taken back).  ``counts`` (int32 ``[B]``):
        how many of the rows are real."""
        width = self.n_kv_heads * HEAD_DIM
        kv = self._view("k", k, None, width)
        self._call("svla_kv_append_bf16", *kv, *self._view("v", v, k.shape[1], width), k.shape[1],
                   self._ints("counts", counts), self._ints("at", at))

    def read(self, start=0, rows=None, k_out=None, v_out=None):
        """``(k, v)`` of positions ``start`` (an int, or int32 ``[B]``) to
        ``start + rows - 1`` as bf16 ``[B, rows, n_kv_heads * 64]``, exactly as
        they are stored; zeros where the cache holds none."""
        rows = self.max_len if rows is None else rows
        if rows is None or rows < 0:
            raise ValueError("read: rows (a cache without max_len has no default)")
        width = self.n_kv_heads * HEAD_DIM
        if k_out is None:
            k_out = self._new(rows, width)
            kv = (k_out.data_ptr(), width, rows * width)
        else:
            kv = self._view("k_out", k_out, rows, width, True)
        if v_out is None:
            v_out = self._new(rows, width)
            kv += (v_out.data_ptr(), width, rows * width)
        else:
            kv += self._view("v_out", v_out, rows, width, True)
        starts = None
        if torch.is_tensor(start):
            starts, start = self._ints("start", start), 0
        elif not 0 <= start <= MAX_POS:
            raise ValueError(f"start must be a position, got {start}")
        self._call("svla_kv_read_bf16", *kv, start, starts, rows)
        return k_out, v_out

    def attend(self, q, n_heads, out=None, counts=None, scale=None):
        """Attention of the last T tokens of every sequence (``q`` ``[B, T,
        n_heads * 64]``; with ``counts`` the last ``counts[b]``, rows behind
        them give zeros) over the cache: causal, within the cache's window and
        sinks.  A sequence of which needed tokens are gone gives NaN."""
        return self._attend("svla_kv_attention_bf16", q, n_heads, (), out, counts, (), scale)

    def step(self, q, k, v, n_heads, out=None, counts=None, at=None, scale=None):
        """:meth:`append` of new rows and :meth:`attend` of their queries, in one
        call (one launch less for a single row)."""
        width = self.n_kv_heads * HEAD_DIM
        if q.shape[1:2] != k.shape[1:2]:
            raise ValueError("step: a query for every new row")
        kv = (*self._view("k", k, None, width), *self._view("v", v, k.shape[1], width))
        return self._attend("svla_kv_step_bf16", q, n_heads, kv, out, counts,
                            (self._ints("at", at),), scale)

    def _attend(self, name, q, n_heads, kv, out, counts, at, scale):
        width = n_heads * HEAD_DIM
        qv = self._view("q", q, None, width)
        rows = q.shape[1]
        if self.max_rows is not None and rows > self.max_rows:
            raise ValueError(f"{rows} rows, the cache was made for {self.max_rows}")
        if out is None:
            out = torch.empty_like(q) if qv[1:] == (width, rows * width) else self._new(rows, width)
            ov = (out.data_ptr(), width, rows * width)
        else:
            ov = self._view("out", out, rows, width, True)
        key = (rows, n_heads)
        nbytes = self._scratch.get(key)
        if nbytes is None:
            nbytes = self._scratch[key] = self._lib.svla_kv_attention_scratch(
                self._ref, rows, n_heads, self.window or 0)
        # (of this call alone: the allocator keeps it until the stream has passed)
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=self.device) if nbytes else None
        self._call(name, *qv, *kv, *ov, rows, self._ints("counts", counts), *at, n_heads,
                   SCALE if scale is None else scale, self.window or 0,
                   scratch.data_ptr() if nbytes else None, nbytes)
        return out
