"""The microscaled K/V cache against a plain float64 one: what it stores, which
positions it keeps, and attention over it (bounds: ``oracle.context_ref``)."""

import pytest
import torch

from oracle import context_ref as ref
from smolvla.kv_cache import KVCache

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
FMTS = ["mxfp4", "mxfp8"]


def rand(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(BF16)


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def same(got, want):
    got, want = got.double().cpu(), want.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))


def close(got, want):
    want, bound = want
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = ((got - want).abs() <= bound) | torch.isnan(want)
    assert ok.all(), f"{(~ok).sum()} off, worst {((got - want).abs() / bound).nan_to_num().max()} bounds"


# ------------------------------------------------------------------ storage ---
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows", [1, 5, 32, 77])
def test_stored_values(fmt, rows):
    g = gen(rows)
    cache = KVCache(2, 3, max_len=100, fmt=fmt)
    k = rand(g, 2, rows, 192) * torch.exp2(torch.randint(-30, 30, (2, rows, 192), generator=g,
                                                         device="cuda")).to(BF16)
    v = rand(g, 2, rows, 192)
    cache.append(k, v)
    ko, vo = cache.read(0, rows)
    same(ko, ref.stored(k.cpu(), fmt))
    same(vo, ref.stored(v.cpu(), fmt))
    assert cache.lengths.tolist() == [rows, rows]


@pytest.mark.parametrize("fmt", FMTS)
def test_every_bf16_value(fmt):
    """All finite bf16 numbers, each in a block with the power of two that scales
    it into every binade of the format, and the extremes of the range."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.uint16).view(BF16)
    x = x[torch.isfinite(x)]
    x = torch.cat([x, x.new_zeros(-len(x) % 2048)]).view(1, -1, 64)
    lead = x.clone()
    lead[..., ::32] = torch.exp2(torch.arange(x.shape[1]).remainder(250) - 125.0)[:, None].to(BF16)
    for k, v in ((x, lead), (lead, x.flip(1))):
        cache = KVCache(1, 1, max_len=x.shape[1], fmt=fmt)
        cache.append(k.cuda(), v.cuda())
        ko, vo = cache.read()
        same(ko, ref.stored(k, fmt))
        same(vo, ref.stored(v, fmt))


@pytest.mark.parametrize("fmt", FMTS)
def test_block_with_infinity_or_nan_reads_as_nan(fmt):
    k = torch.ones(1, 40, 64, dtype=BF16, device="cuda")
    v = k.clone()
    k[0, 3, 5], k[0, 33, 40], v[0, 7, 63], v[0, 39, 0] = (float(x) for x in ("nan", "inf", "-inf", "nan"))
    cache = KVCache(1, 1, max_len=40, fmt=fmt)
    cache.append(k, v)
    ko, vo = cache.read()
    same(ko, ref.stored(k.cpu(), fmt))
    same(vo, ref.stored(v.cpu(), fmt))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("sinks,window", [(0, None), (4, 40), (33, 64)])
def test_pieces_equal_the_whole(fmt, sinks, window):
    """Appends of any sizes leave the same rows as one; views with other strides."""
    g = gen(1)
    n = 150
    wide = rand(g, 2, n, 2 * 128 + 16)
    k, v = wide[:, :, :128], wide[:, :, 136:264]
    make = lambda: KVCache(2, 2, fmt=fmt, max_len=None if window else n, window=window,  # noqa: E731
                           sinks=sinks, rows=70)
    a, b = make(), make()
    a.append(k, v)
    at = 0
    for c in (1, 1, 30, 2, 64, 31, 21):
        b.append(k[:, at:at + c], v[:, at:at + c])
        at += c
    assert at == n
    for x, y in zip(a.read(0, n), b.read(0, n)):
        same(x, y)
    assert torch.equal(a.state, b.state)


@pytest.mark.parametrize("fmt", FMTS)
def test_uneven_rows_and_positions(fmt):
    """counts (clamped to the rows there are) and at; rows behind a count are not
    read, rows of the cache that are not written stay."""
    g = gen(2)
    cache, want = KVCache(5, 1, max_len=80, fmt=fmt), ref.CacheRef(5, 1, fmt)
    k, v = rand(g, 5, 37, 64), rand(g, 5, 37, 64)
    counts = ints(37, 0, 1, 33, 99)
    pad = k.clone()
    pad[2, 1:] = float("nan")
    cache.append(pad, v, counts=counts)
    want.append(k, v, counts.clamp(0, 37))
    k, v = rand(g, 5, 3, 64), rand(g, 5, 3, 64)
    at = ints(30, 0, 1, 32, 37)
    counts = ints(3, 2, -4, 3, 1)
    cache.append(k, v, counts=counts, at=at)
    want.append(k, v, counts.clamp(0, 3), at)
    ko, vo = cache.read(0, 40)
    for b in range(5):
        n = len(want.k[b])
        assert int(cache.lengths[b]) == n
        same(ko[b, :n], want.k[b])
        same(vo[b, :n], want.v[b])
        assert (ko[b, n:] == 0).all() and (vo[b, n:] == 0).all()
    # from a position of its own each; below 0 and behind the end: zeros
    starts = ints(31, -2, 0, 500, 36)
    ko, vo = cache.read(starts, 4)
    for b, s in enumerate(starts.tolist()):
        for r in range(4):
            inside = 0 <= s + r < len(want.k[b])
            same(ko[b, r], want.k[b][s + r] if inside else torch.zeros(64))
            same(vo[b, r], want.v[b][s + r] if inside else torch.zeros(64))


def test_rows_that_left_the_ring_read_as_zeros():
    g = gen(3)
    cache = KVCache(1, 1, fmt="mxfp8", window=40, sinks=5, rows=1)
    want = ref.CacheRef(1, 1, "mxfp8")
    for c in (3, 30, 100, 1, 40, 64, 1):
        k, v = rand(g, 1, c, 64), rand(g, 1, c, 64)
        cache.append(k, v)
        want.append(k, v)
    n = len(want.k[0])
    ko, vo = cache.read(0, n + 3)
    held = (ko[0].abs().amax(1) > 0).cpu()
    assert held[:5].all() and held[n - 40:n].all() and not held[n:].any()
    assert not held[5:n - cache.ring].any()
    for p in held.nonzero().flatten().tolist():
        same(ko[0, p], want.k[0][p])
        same(vo[0, p], want.v[0][p])


# ---------------------------------------------------------------- attention ---
CASES = [  # batch, hq, hkv, held, rows, window, sinks
    (1, 3, 1, 1, 1, None, 0), (2, 15, 5, 31, 1, None, 0), (1, 15, 5, 32, 1, None, 0),
    (3, 4, 4, 33, 1, None, 0), (1, 8, 1, 700, 1, None, 0), (1, 32, 2, 65, 1, None, 0),
    (1, 15, 5, 241, 50, None, 0), (2, 2, 2, 130, 129, None, 0), (1, 17, 1, 40, 5, None, 0),
    (1, 6, 2, 300, 1, 64, 4), (2, 15, 5, 200, 1, 1, 0), (1, 4, 2, 90, 7, 33, 1),
    (1, 3, 1, 500, 70, 100, 40), (1, 2, 1, 20, 20, 64, 64), (1, 5, 5, 64, 3, 7, 3),
    (1, 9, 3, 5000, 1, None, 0),
]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("batch,hq,hkv,held,rows,window,sinks", CASES)
def test_attend(fmt, batch, hq, hkv, held, rows, window, sinks):
    g = gen(held)
    cache = KVCache(batch, hkv, fmt=fmt, max_len=None if window else held, window=window,
                    sinks=sinks, rows=rows)
    want = ref.CacheRef(batch, hkv, fmt, window, sinks)
    k, v = rand(g, batch, held, hkv * 64, scale=2.0), rand(g, batch, held, hkv * 64)
    cache.append(k, v)
    want.append(k, v)
    q = rand(g, batch, rows, hq * 64)
    close(cache.attend(q, hq), want.attend(q, hq))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 3)])
def test_uneven_sequences(fmt, window, sinks):
    """Sequences of other lengths and query counts, one empty, one of one token;
    views of a fused projection; rows behind a count give zeros."""
    g = gen(5)
    cache = KVCache(5, 2, fmt=fmt, max_len=None if window else 400, window=window, sinks=sinks,
                    rows=40)
    want = ref.CacheRef(5, 2, fmt, window, sinks)
    held = ints(300, 0, 97, 32, 1)
    k, v = rand(g, 5, 300, 128), rand(g, 5, 300, 128)
    cache.append(k, v, counts=held)
    want.append(k, v, held)
    qkv = rand(g, 5, 40, 6 * 64 + 256)
    counts = ints(40, 1, 0, 33, 7)
    out = torch.full((5, 40, 6 * 64 + 8), 7.0, dtype=BF16, device="cuda")
    cache.step(qkv[:, :, :384], qkv[:, :, 384:512], qkv[:, :, 512:], 6, out=out[:, :, :384],
               counts=counts)
    want.append(qkv[:, :, 384:512], qkv[:, :, 512:], counts)
    close(out[:, :, :384], want.attend(qkv[:, :, :384], 6, counts))
    assert (out[:, :, 384:] == 7).all()
    for b, c in enumerate(counts.tolist()):
        assert (out[b, c:, :384] == 0).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows", [1, 6, 40])
def test_scores_of_any_size(fmt, rows):
    """Scores of several hundred, where the running maximum moves, and a scale."""
    g = gen(6)
    cache, want = KVCache(1, 2, max_len=600, fmt=fmt), ref.CacheRef(1, 2, fmt)
    k, v = rand(g, 1, 600, 128, scale=8.0), rand(g, 1, 600, 128)
    k *= torch.linspace(0.1, 4, 600, device="cuda")[:, None].to(BF16)
    cache.append(k, v)
    want.append(k, v)
    q = rand(g, 1, rows, 256, scale=3.0)
    close(cache.attend(q, 4, scale=0.25), want.attend(q, 4, scale=0.25))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 2)])
def test_unseen_tokens_do_not_reach_a_row(fmt, window, sinks):
    """A NaN token spoils the rows that see it and no others: not those before it,
    not those whose window has passed it."""
    g = gen(7)
    n, rows = 90, 60
    k, v = rand(g, 1, n, 64), rand(g, 1, n, 64)
    q = rand(g, 1, rows, 128)
    for where, (tk, tv) in {70: (False, True), 45: (True, False), 0: (True, True)}.items():
        cache = KVCache(1, 1, fmt=fmt, max_len=None if window else n, window=window, sinks=sinks,
                        rows=rows)
        k2, v2 = k.clone(), v.clone()
        if tk:
            k2[0, where, 3] = float("nan")
        if tv:
            v2[0, where, 40:] = float("inf")
        want = ref.CacheRef(1, 1, fmt, window, sinks)
        cache.append(k2, v2)
        want.append(k2, v2)
        got = cache.attend(q, 2)
        close(got, want.attend(q, 2))
        # (every row sees token 0 where there is no window or it is a sink)
        sees = [p for p in range(n - rows, n) if where <= p and
                (window is None or where > p - window or where < sinks)]
        assert torch.isnan(got).any(2)[0].nonzero().flatten().tolist() == [p - n + rows for p in sees]


def test_a_query_that_is_not_finite_spoils_its_row_only():
    g = gen(8)
    cache, want = KVCache(1, 1, max_len=50), ref.CacheRef(1, 1, "mxfp4")
    k, v, q = rand(g, 1, 50, 64), rand(g, 1, 50, 64), rand(g, 1, 5, 128)
    cache.append(k, v)
    want.append(k, v)
    q[0, 2, 10] = float("nan")
    close(cache.attend(q, 2), want.attend(q, 2))


@pytest.mark.parametrize("fmt", FMTS)
def test_a_long_stream_through_the_ring(fmt):
    """A prompt longer than the ring, then steps of one and of several tokens."""
    g = gen(9)
    cache = KVCache(2, 1, fmt=fmt, window=45, sinks=3, rows=4)
    want = ref.CacheRef(2, 1, fmt, 45, 3)
    for c in [200] + [1, 1, 4, 1, 3] * 12:
        k, v, q = rand(g, 2, c, 64), rand(g, 2, c, 64), rand(g, 2, min(c, 4), 192)
        if c > 4:
            cache.append(k, v)
            want.append(k, v)
            close(cache.attend(q, 3), want.attend(q, 3))
        else:
            got = cache.step(q, k, v, 3)
            want.append(k, v)
            close(got, want.attend(q, 3))
    cache.check()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hq,hkv", [(3, 3), (16, 1), (40, 2), (64, 1), (96, 1)])
@pytest.mark.parametrize("held", [0, 31, 32, 1100])
def test_a_step_of_one_token(fmt, hq, hkv, held):
    """One new row per sequence (of some): written by the attention itself where
    one workgroup has all of a record's columns; the cache is then the one that
    append leaves."""
    g = gen(held + hq)
    cache = KVCache(3, hkv, fmt=fmt, max_len=held + 3)
    other = KVCache(3, hkv, fmt=fmt, max_len=held + 3)
    want = ref.CacheRef(3, hkv, fmt)
    k, v = rand(g, 3, held, hkv * 64), rand(g, 3, held, hkv * 64)
    for c in (cache, other, want):
        c.append(k, v)
    for counts in (None, ints(1, 0, 1), None):
        q, k, v = rand(g, 3, 1, hq * 64), rand(g, 3, 1, hkv * 64), rand(g, 3, 1, hkv * 64)
        got = cache.step(q, k, v, hq, counts=counts)
        other.append(k, v, counts=counts)
        want.append(k, v, counts)
        close(got, want.attend(q, hq, counts))
    assert torch.equal(cache.state, other.state)
    for x, y in zip(cache.read(), other.read()):
        assert torch.equal(x, y)


@pytest.mark.parametrize("fmt", FMTS)
def test_a_step_at_a_position(fmt):
    """Steps that go back, one that skips ahead (lost), and one whose row is NaN."""
    g = gen(20)
    cache, want = KVCache(3, 2, max_len=100, fmt=fmt), ref.CacheRef(3, 2, fmt)
    k, v = rand(g, 3, 70, 128), rand(g, 3, 70, 128)
    cache.append(k, v)
    want.append(k, v)
    q, k, v = rand(g, 3, 1, 384), rand(g, 3, 1, 128), rand(g, 3, 1, 128)
    v[2, 0, 40] = float("nan")
    at = ints(70, 33, 64)
    got = cache.step(q, k, v, 6, at=at)
    want.append(k, v, at=at)
    close(got, want.attend(q, 6))
    same(cache.read(at, 1)[1], torch.stack([x[-1:] for x in want.v]))
    got = cache.step(q, k, v, 6, at=ints(72, 0, 1))
    want.append(k, v, at=[0, 0, 1])
    assert torch.isnan(got[0]).all() and not torch.isnan(got[1]).any()
    close(got[1:], tuple(x[1:] for x in want.attend(q, 6)))
    with pytest.raises(RuntimeError, match=r"\[0\] were written"):
        cache.check()


def test_a_first_score_far_below_the_others():
    """Scores that outgrow the first record's by hundreds of powers of two."""
    g = gen(21)
    for rows in (1, 20):
        cache, want = KVCache(1, 1, max_len=900, fmt="mxfp8"), ref.CacheRef(1, 1, "mxfp8")
        k, v = rand(g, 1, 900, 64), rand(g, 1, 900, 64)
        k *= torch.linspace(0.01, 60, 900, device="cuda")[:, None].to(BF16)
        v[0, 100:200] *= 2.0 ** 104
        cache.append(k, v)
        want.append(k, v)
        q = rand(g, 1, rows, 128, scale=2.0)
        close(cache.attend(q, 2, scale=2.0), want.attend(q, 2, scale=2.0))


@pytest.mark.parametrize("level", [-12.0, -25.0, -60.0, -2000.0])
def test_scores_far_below_zero_and_tiny_values(level):
    """Every score around ``level``: sums of exp(s) that are small or zero, with
    values that a product with them would lose."""
    g = gen(23)
    for rows in (1, 24, 90):
        cache, want = KVCache(1, 1, max_len=200, fmt="mxfp8"), ref.CacheRef(1, 1, "mxfp8")
        k, v = rand(g, 1, 200, 64, scale=0.05), rand(g, 1, 200, 64, scale=2.0 ** -80)
        k[..., 0], k[..., 32] = 1.0, 1.0
        q = rand(g, 1, rows, 128)
        q.view(1, rows, 2, 64)[..., 0] = level * 8
        cache.append(k, v)
        want.append(k, v)
        close(cache.attend(q, 2), want.attend(q, 2))


def test_time_before_batch_and_in_place():
    """[T, B, .] tensors as [B, T, .] views, and the output over the queries."""
    g = gen(22)
    cache, want = KVCache(3, 1, max_len=60), ref.CacheRef(3, 1, "mxfp4")
    q, k, v = (rand(g, 50, 3, w).transpose(0, 1) for w in (128, 64, 64))
    expect = q.clone()
    out = torch.empty(50, 3, 128, dtype=BF16, device="cuda").transpose(0, 1)
    cache.step(q, k, v, 2, out=out)
    want.append(k, v)
    close(out, want.attend(expect, 2))
    cache.attend(q, 2, out=q)
    assert torch.equal(q, out)
    ko, vo = (torch.empty(60, 3, 64, dtype=BF16, device="cuda").transpose(0, 1) for _ in range(2))
    cache.read(0, 60, k_out=ko, v_out=vo)
    same(ko[:, :50], ref.stored(k.cpu(), "mxfp4"))
    same(vo[:, :50], ref.stored(v.cpu(), "mxfp4"))
    assert (ko[:, 50:] == 0).all()


# ------------------------------------------------------------------- errors ---
@pytest.mark.parametrize("fmt", FMTS)
def test_lost_sequences(fmt):
    """Too many tokens, or a position not reached: NaN and check(), the other
    sequences untouched; writing from 0 starts anew."""
    g = gen(10)
    cache, want = KVCache(2, 1, max_len=64, fmt=fmt), ref.CacheRef(2, 1, fmt)
    k, v, q = rand(g, 2, 70, 64), rand(g, 2, 70, 64), rand(g, 2, 1, 64)
    cache.append(k, v, counts=ints(70, 50))
    want.append(k, v, ints(70, 50))
    out = cache.attend(q, 1)
    assert torch.isnan(out[0]).all()
    close(out[1:], tuple(x[1:] for x in want.attend(q, 1)))
    with pytest.raises(RuntimeError, match=r"\[0\] hold more"):
        cache.check()
    cache.append(k[:, :5], v[:, :5], at=ints(0, 60))
    out = cache.attend(q, 1)
    assert torch.isnan(out[1]).all() and (cache.read(0, 60)[0][1] == 0).all()
    with pytest.raises(RuntimeError, match=r"\[1\] were written"):
        cache.check()
    cache.append(k[:, :7], v[:, :7], at=ints(5, 0))
    want = ref.CacheRef(2, 1, fmt)
    want.append(torch.cat([k[:, :5], k[:, :7]], 1), torch.cat([v[:, :5], v[:, :7]], 1), ints(12, 0))
    want.append(k[:, :7], v[:, :7], ints(0, 7))
    close(cache.attend(q, 1), want.attend(q, 1))
    cache.check()
    cache.append(k[:, :1], v[:, :1], at=ints(-1, 7))
    assert torch.isnan(cache.attend(q, 1)[0]).all()
    cache.reset()
    cache.check()
    assert cache.lengths.tolist() == [0, 0]


def test_more_queries_than_tokens():
    g = gen(11)
    cache = KVCache(1, 1, max_len=64)
    cache.append(rand(g, 1, 3, 64), rand(g, 1, 3, 64))
    assert torch.isnan(cache.attend(rand(g, 1, 4, 64), 1)).all()


def test_tokens_taken_back_within_a_ring():
    """What a rewound write has pushed out of the ring stays lost: a call that
    needs it gives NaN, never the later tokens' values."""
    g = gen(12)
    cache, want = KVCache(1, 1, window=32, rows=1), ref.CacheRef(1, 1, "mxfp4", 32)
    k, v, q = rand(g, 1, 400, 64), rand(g, 1, 400, 64), rand(g, 1, 1, 64)
    cache.append(k[:, :300], v[:, :300])
    want.append(k[:, :300], v[:, :300])
    cache.append(k[:, 300:303], v[:, 300:303], at=ints(299))
    want.append(k[:, 300:303], v[:, 300:303], at=[299])
    close(cache.attend(q, 1), want.attend(q, 1))
    cache.append(k[:, :1], v[:, :1], at=ints(200))
    assert torch.isnan(cache.attend(q, 1)).all()


# ----------------------------------------------------------- graphs, streams ---
def test_captured_steps_move_on_with_every_replay():
    g = gen(13)
    make = lambda: KVCache(2, 2, fmt="mxfp4", window=40, sinks=2, rows=1)  # noqa: E731
    eager, replay = make(), make()
    k, v = rand(g, 2, 90, 128), rand(g, 2, 90, 128)
    for c in (eager, replay):
        c.append(k[:, :60], v[:, :60])
    q1, k1, v1 = (torch.zeros(2, 1, w, dtype=BF16, device="cuda") for w in (384, 128, 128))
    start = replay.state.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        replay.step(q1, k1, v1, 6)
    torch.cuda.current_stream().wait_stream(side)
    replay.state.copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = replay.step(q1, k1, v1, 6)
    for t in range(60, 90):
        q = rand(g, 2, 1, 384)
        q1.copy_(q); k1.copy_(k[:, t:t + 1]); v1.copy_(v[:, t:t + 1])
        graph.replay()
        want = eager.step(q, k[:, t:t + 1], v[:, t:t + 1], 6)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert torch.equal(eager.state, replay.state)


def test_two_graphs_read_one_cache_at_once():
    """Every call has its own workspace: two captured calls on two streams."""
    g = gen(14)
    cache = KVCache(1, 1, max_len=6000, fmt="mxfp8")
    cache.append(rand(g, 1, 6000, 64), rand(g, 1, 6000, 64))
    qs = [rand(g, 1, 1, 128), rand(g, 1, 1, 128)]
    want = [cache.attend(q, 2) for q in qs]
    graphs, outs = [], []
    for q in qs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(cache.attend(q, 2))
        graphs.append(gr)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        torch.cuda.synchronize()
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


def test_rows_on_another_stream():
    g = gen(15)
    side = torch.cuda.Stream()
    cache, want = KVCache(1, 1, max_len=64), ref.CacheRef(1, 1, "mxfp4")
    k, v, q = rand(g, 1, 9, 64), rand(g, 1, 9, 64), rand(g, 1, 9, 64)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = cache.step(q, k, v, 1)
    torch.cuda.current_stream().wait_stream(side)
    want.append(k, v)
    close(out, want.attend(q, 1))


# ----------------------------------------------------------------- refusals ---
def test_refusals():
    from smolvla._lib import SvlaError
    g = gen(16)
    cache = KVCache(2, 2, fmt="mxfp4", window=8, rows=2)
    k = rand(g, 2, 1, 128)
    with pytest.raises(ValueError, match="GPU tensors"):
        cache.append(k.cpu(), k.cpu())
    for bad in (k[:1], k[:, :, :64], k.float(), k[0]):
        with pytest.raises(ValueError):
            cache.append(bad, k)
        with pytest.raises(ValueError):
            cache.append(k, bad)
    with pytest.raises(ValueError, match="contiguous"):
        cache.append(rand(g, 2, 1, 256)[:, :, ::2], k)
    with pytest.raises(SvlaError):
        cache.append(rand(g, 2, 1, 129)[:, :, 1:], k)           # not 16-byte aligned
    for bad in (ints(1), torch.ones(2, device="cuda"), ints(1, 1).cpu(), [1, 1]):
        with pytest.raises(ValueError):
            cache.append(k, k, counts=bad)
        with pytest.raises(ValueError):
            cache.append(k, k, at=bad)
    with pytest.raises(ValueError, match="made for 2"):
        cache.attend(rand(g, 2, 3, 128), 2)
    with pytest.raises(SvlaError):
        cache.attend(rand(g, 2, 1, 192), 3)                     # 3 heads over 2
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(SvlaError):
            cache.attend(k, 2, scale=scale)
    with pytest.raises(ValueError):
        cache.attend(k, 2, out=rand(g, 2, 1, 64))
    with pytest.raises(ValueError):
        cache.step(k, rand(g, 2, 2, 128), rand(g, 2, 2, 128), 2)
    with pytest.raises(ValueError):
        cache.read()                                            # no max_len
    for start in (-1, 2 ** 32):
        with pytest.raises(ValueError):
            cache.read(start, 4)
    with pytest.raises(ValueError, match="overlap"):
        cache.read(0, 4, k_out=rand(g, 1, 4, 128).expand(2, -1, -1))
    with pytest.raises(ValueError, match="overlap"):
        cache.attend(k, 2, out=k[:1].expand(2, -1, -1))
    assert cache.lengths.tolist() == [0, 0]
    # nothing to do
    cache.append(k[:, :0], k[:, :0])
    assert cache.attend(k[:, :0], 2).shape == (2, 0, 128)
    assert cache.read(0, 0)[0].shape == (2, 0, 128)
