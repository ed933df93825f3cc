"""The decoder layer on a bounded context, as a stream runs it: a prompt, then a
few tokens at a time through a microscaled cache, and the windowed mask.

With Wo the identity (960 = 15 heads of 64) and an MLP of zeros the layer is
x + attention, so its output is held against the float64 attention of the rows
that the cache really stores (read back), Q and K from the layer's own
projection.  Off by the attention's bound, a rounding to bf16 of the sum, and
none more: |attention| <= max |v|."""

import pytest
import torch

from oracle import context_ref as ref
from smolvla import layers, ops
from smolvla.config import DecoderConfig
from smolvla.kv_cache import KVCache
from smolvla.params import _Gen, decoder_layer_params
from smolvla.vla.text_encoder_bf16 import text_encoder_forward

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
CFG = DecoderConfig()


def params(seed=0):
    p = dict(decoder_layer_params(_Gen(seed), CFG))
    p["Wo"] = torch.eye(960).to(BF16)
    for k in ("W_gate", "W_up", "W_down"):
        p[k] = torch.zeros_like(p[k])
    return p


def projected(x, p, position):
    """q, k, v [B, L, .] of the layer's own kernels."""
    B, L, H = x.shape
    P = layers.prep_decoder(p, "cuda")
    rope = layers.Rope.make(L, 64, CFG.rope_theta, "cuda", position)
    h = ops.rmsnorm(x.reshape(-1, H), P["n1"], CFG.rms_eps)
    qkv = ops.linear_rope(h, P["wqkv"], 960 + 320, L, rope.cos, rope.sin).view(B, L, -1)
    return qkv[:, :, :960], qkv[:, :, 960:1280], qkv[:, :, 1280:]


def check(out, x, q, keys, values, first, window, sinks):
    L = q.shape[1]
    for b in range(q.shape[0]):
        n = first + L
        want, bound = ref.attention(q[b].cpu(), keys[b, :n].cpu(), values[b, :n].cpu(),
                                    torch.arange(first, n), torch.arange(n), 15, 5, window, sinks)
        want = want + x[b].double().cpu()
        off = (out[b].double().cpu() - want).abs()
        assert (off <= bound + 2 ** -8 * 1.02 * (want.abs() + bound)).all()


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("window,sinks", [(None, 0), (48, 4)])
def test_a_stream_of_tokens(fmt, window, sinks):
    p = params()
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(2, 130, 960, generator=g, device="cuda").to(BF16)
    cache = KVCache(2, 5, fmt=fmt, max_len=None if window else 130, window=window, sinks=sinks,
                    rows=100)
    # what the cache stores of a row does not depend on the pieces: all of them
    # in a second cache that keeps everything
    everything = KVCache(2, 5, fmt=fmt, max_len=130)
    at = 0
    for n in (100, 1, 1, 5, 1, 20, 1, 1):
        piece = x[:, at:at + n]
        out, key, value = text_encoder_forward(piece, p, cache=cache, position=at)
        q, k, v = projected(piece, p, at)
        assert torch.equal(key, k) and torch.equal(value, v)
        everything.append(k, v)
        keys, values = everything.read()
        check(out, piece, q, keys, values, at, window, sinks)
        at += n
    assert at == 130 and cache.lengths.tolist() == [130, 130]
    cache.check()


@pytest.mark.parametrize("length", [5, 130])
def test_windowed_mask(length):
    p = params(1)
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(2, length, 960, generator=g, device="cuda").to(BF16)
    out, key, value = text_encoder_forward(x, p, mask="window", window=40, sinks=2)
    q, k, v = projected(x, p, 0)
    assert torch.equal(key, k) and torch.equal(value, v)
    check(out, x, q, k, v, 0, 40, 2)
    # a single sequence, as the reference's callers pass it
    one, _, _ = text_encoder_forward(x[0], p, mask="window", window=40, sinks=2)
    assert one.shape == (length, 960)


def test_rope_rows_of_later_positions():
    c, s = ops.rope_table(300, 64, 1e5)
    c2, s2 = ops.rope_table(50, 64, 1e5, first=250)
    assert torch.equal(c[250:], c2) and torch.equal(s[250:], s2)


def test_refusals():
    p = params()
    x = torch.zeros(1, 4, 960, dtype=BF16, device="cuda")
    cache = KVCache(1, 5, max_len=32)
    for kw in (dict(position=3), dict(cache=cache, mask="window", window=4),
               dict(cache=cache, window=4), dict(window=4), dict(mask="window")):
        with pytest.raises(ValueError):
            text_encoder_forward(x, p, **kw)
    with pytest.raises(ValueError):
        text_encoder_forward(torch.cat([x, x]), p, cache=cache)      # two sequences
    assert cache.lengths.tolist() == [0]
