"""Host-side checks of the bounded-context entry points (no GPU: every call here
returns before a launch, its pointers are never dereferenced)."""

import ctypes as C

import pytest
import torch

from oracle import context_ref as ref

FAKE = C.c_void_p(1 << 20)
ODD = C.c_void_p((1 << 20) + 4)


def cache(**kw):
    from smolvla import _lib
    f = dict(data=1 << 20, state=1 << 20, batch=2, n_kv_heads=2, head_dim=64, format=4, sinks=4,
             ring=64)
    f.update(kw)
    return _lib.KVCacheDesc(**f)


BAD_CACHES = [dict(data=None), dict(state=None), dict(data=(1 << 20) + 8), dict(batch=0),
              dict(n_kv_heads=-1), dict(head_dim=128), dict(format=5), dict(sinks=-1),
              dict(ring=0), dict(ring=33), dict(ring=2 ** 30 + 32), dict(batch=65536),
              dict(sinks=2 ** 30)]


def test_cache_bytes():
    from smolvla import _lib
    f = _lib.load().svla_kv_cache_bytes
    assert f(1, 1, 64, 4, 0, 32) == 32 * 68
    assert f(1, 1, 64, 8, 0, 32) == 32 * 132
    assert f(3, 5, 64, 4, 33, 96) == 15 * 5 * 32 * 68           # 2 records of sinks, 3 of the ring
    assert f(64, 8, 64, 8, 0, 1 << 24) == 512 * (1 << 24) * 132      # past 32 bits
    for kw in BAD_CACHES[3:]:
        c = cache(**kw)
        assert f(c.batch, c.n_kv_heads, c.head_dim, c.format, c.sinks, c.ring) == 0


def calls(lib, c):
    r = C.byref(c) if c is not None else None
    return [lib.svla_kv_reset(r, None),
            lib.svla_kv_append_bf16(r, FAKE, 128, 0, FAKE, 128, 0, 1, None, None, None),
            lib.svla_kv_read_bf16(r, FAKE, 128, 0, FAKE, 128, 0, 0, None, 1, None),
            lib.svla_kv_attention_bf16(r, FAKE, 128, 0, FAKE, 128, 0, 1, None, 2, 0.125, 0, FAKE,
                                       1 << 40, None)]


def test_bad_caches():
    from smolvla import _lib
    lib = _lib.load()
    assert calls(lib, None) == [-22] * 4
    for kw in BAD_CACHES:
        assert calls(lib, cache(**kw)) == [-22] * 4, kw
        assert lib.svla_kv_attention_scratch(C.byref(cache(**kw)), 1, 2, 0) == 0


def test_bad_arguments():
    from smolvla import _lib
    lib = _lib.load()
    r = C.byref(cache())
    app = lambda k=FAKE, ldk=128, kbs=0, v=FAKE, ldv=128, vbs=0, rows=1: lib.svla_kv_append_bf16(  # noqa: E731
        r, k, ldk, kbs, v, ldv, vbs, rows, None, None, None)
    read = lambda k=FAKE, ldk=128, kbs=0, v=FAKE, ldv=128, vbs=0, rows=1, start=0: lib.svla_kv_read_bf16(  # noqa: E731
        r, k, ldk, kbs, v, ldv, vbs, start, None, rows, None)
    for f in (app, read):
        for kw in (dict(k=None), dict(v=ODD), dict(ldk=120), dict(ldv=132), dict(kbs=4),
                   dict(rows=-1), dict(rows=2 ** 30 + 1)):
            assert f(**kw) == -22, kw
        assert f(rows=0) == 0
    assert read(start=-1) == -22
    att = lambda q=FAKE, ldq=256, qbs=0, o=FAKE, ldo=256, obs=0, rows=1, hq=4, scale=0.125, window=0, scratch=FAKE, nbytes=1 << 40: lib.svla_kv_attention_bf16(  # noqa: E501,E731
        r, q, ldq, qbs, o, ldo, obs, rows, None, hq, scale, window, scratch, nbytes, None)
    for kw in (dict(q=None), dict(q=ODD), dict(ldq=192), dict(o=None), dict(ldo=192), dict(ldo=258),
               dict(obs=2), dict(qbs=4), dict(rows=-1), dict(hq=0), dict(hq=3), dict(scale=0.0),
               dict(scale=float("nan")), dict(window=-1), dict(rows=1 << 23)):
        assert att(**kw) == -22, kw
    assert att(rows=0) == 0


def test_scratch_has_to_fit():
    from smolvla import _lib
    lib = _lib.load()
    c = cache(ring=1 << 20, batch=1)
    need = lib.svla_kv_attention_scratch(C.byref(c), 1, 4, 0)
    assert need > 0
    for scratch, n in ((FAKE, need - 1), (None, need), (None, 0)):
        assert lib.svla_kv_attention_bf16(C.byref(c), FAKE, 256, 0, FAKE, 256, 0, 1, None, 4, 0.125,
                                          0, scratch, n, None) == -22


def test_bad_window_arguments():
    from smolvla import _lib
    lib = _lib.load()
    call = lambda q=FAKE, ldq=128, qbs=0, k=FAKE, ldk=64, v=FAKE, o=FAKE, ldo=128, batch=1, sq=4, sk=4, hq=2, hkv=1, d=64, scale=0.125, q_pos=0, window=4, sinks=0: lib.svla_attention_window_bf16(  # noqa: E501,E731
        q, ldq, qbs, k, ldk, 0, v, 64, 0, o, ldo, 0, batch, sq, sk, hq, hkv, d, scale, q_pos, None,
        window, sinks, None)
    for kw in (dict(q=None), dict(k=ODD), dict(o=None), dict(ldq=64), dict(ldk=60), dict(ldo=130),
               dict(qbs=4), dict(ldk=2 ** 24 + 64), dict(batch=-1), dict(batch=65536), dict(sq=-1), dict(sk=0), dict(hq=0),
               dict(hq=3, hkv=2), dict(d=32), dict(scale=0.0), dict(scale=float("inf")),
               dict(q_pos=-1), dict(q_pos=2 ** 30), dict(window=0), dict(sinks=-1)):
        assert call(**kw) == -22, kw
    assert call(sq=0, q=None, o=None) == 0 and call(batch=0) == 0


@pytest.mark.parametrize("kw", [dict(fmt="fp4"), dict(batch=0), dict(n_kv_heads=0), dict(rows=0),
                                dict(window=0), dict(max_len=None), dict(max_len=0), dict(sinks=2),
                                dict(window=4, sinks=-1), dict(device="cpu"), dict(max_len=2 ** 32 + 5),
                                dict(batch=2 ** 32 + 1), dict(window=2 ** 32 + 1, max_len=None),
                                dict(window=4, sinks=2 ** 32)])
def test_constructor(kw):
    from smolvla.kv_cache import KVCache
    args = dict(batch=1, n_kv_heads=1, max_len=32)
    args.update(kw)
    with pytest.raises(ValueError):
        KVCache(**args)


def test_the_oracle_stores_what_the_formats_say():
    x = torch.zeros(1, 32)
    x[0, :8] = torch.tensor([6.0, 5.0, 2.5, 0.25, 0.75, -1.75, 3.5, 0.1])
    want = torch.zeros(1, 32)
    want[0, :8] = torch.tensor([6.0, 4.0, 2.0, 0.0, 1.0, -2.0, 4.0, 0.0])
    assert torch.equal(ref.stored(x, "mxfp4"), want.double())
    assert torch.equal(ref.stored(x * 2.0 ** 20, "mxfp4"), want.double() * 2.0 ** 20)
    x[0, 0] = 6.25                              # past 6: the next power of two
    assert ref.stored(x, "mxfp4")[0, :3].tolist() == [6.0, 4.0, 2.0]
    x = torch.zeros(1, 32)
    x[0, :4] = torch.tensor([448.0, 17.0, 19.0, 2.0 ** -10])
    assert ref.stored(x, "mxfp8")[0, :4].tolist() == [448.0, 16.0, 20.0, 0.0]


def test_the_oracle_attends_as_torch_does():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(9, 64 * h, generator=g, dtype=torch.float64) for h in (4, 2, 2))
    pos = torch.arange(9)
    got, _ = ref.attention(q, k, v, pos, pos, 4, 2, window=3, sinks=1)
    heads = lambda x: x.view(9, -1, 64).transpose(0, 1)  # noqa: E731
    k4, v4 = (heads(x).repeat_interleave(2, 0) for x in (k, v))
    s = heads(q) @ k4.transpose(1, 2) / 8
    d = pos[:, None] - pos[None, :]
    s = s.masked_fill((d < 0) | ((d >= 3) & (pos >= 1)), float("-inf"))
    want = (s.softmax(-1) @ v4).transpose(0, 1).reshape(9, 256)
    assert torch.allclose(got, want, atol=1e-12)
