"""Attention with a sliding window and sinks against float64 (bounds:
``oracle.context_ref``)."""

import pytest
import torch

from oracle import context_ref as ref
from smolvla import ops

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def rand(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(BF16)


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def check(q, k, v, hq, hkv, window, sinks=0, lens=None, q_pos=0, out=None, scale=None):
    out = torch.empty(q.shape[0], q.shape[1], hq * 64, dtype=BF16, device="cuda") if out is None else out
    got = ops.attention(q, k, v, out, hq, hkv, mask="window", window=window, sinks=sinks,
                        lens=lens, q_pos=q_pos, scale=scale)
    assert got is out
    got = got.double().cpu()
    for b in range(q.shape[0]):
        n = k.shape[1] if lens is None else min(max(int(lens[b]), 0), k.shape[1])
        want, bound = ref.attention(q[b].cpu(), k[b, :n].cpu(), v[b, :n].cpu(),
                                    q_pos + torch.arange(q.shape[1]), torch.arange(n), hq, hkv,
                                    window, sinks, scale)
        assert torch.equal(torch.isnan(got[b]), torch.isnan(want))
        same_inf = torch.isinf(want) & (got[b] == want)
        ok = same_inf | torch.isnan(want) | ((got[b] - want).abs() <= bound)
        assert ok.all(), f"sequence {b}: {(~ok).sum()} off"
    return out


@pytest.mark.parametrize("batch,hq,hkv,n,window,sinks", [
    (1, 1, 1, 1, 1, 0), (2, 3, 1, 5, 2, 1), (1, 15, 5, 241, 64, 1), (1, 2, 2, 64, 64, 0),
    (1, 2, 1, 65, 63, 4), (1, 4, 2, 300, 1, 0), (1, 2, 1, 300, 7, 70), (1, 3, 3, 257, 1000, 0),
    (2, 2, 1, 130, 32, 130), (1, 1, 1, 700, 200, 3),
])
def test_sizes(batch, hq, hkv, n, window, sinks):
    g = gen(n)
    check(rand(g, batch, n, hq * 64), rand(g, batch, n, hkv * 64, scale=2.0),
          rand(g, batch, n, hkv * 64), hq, hkv, window, sinks)


def test_many_rows_take_the_larger_tile():
    """Enough workgroups of 128 rows for the chip: the other tile, against the
    oracle on two sequences and against the small tile's rows on all: either is
    within (2^-8 (|v| + |o|) + 2^-8 |o|) of the value, |o| <= max |v|."""
    g = gen(1)
    b, n, hq = 14, 1600, 3
    q, k, v = rand(g, b, n, hq * 64), rand(g, b, n, 64), rand(g, b, n, 64)
    out = ops.attention(q, k, v, torch.empty_like(q), hq, 1, mask="window", window=1100, sinks=2)
    for i in range(b):
        part = ops.attention(q[i:i + 1], k[i:i + 1], v[i:i + 1], torch.empty_like(q[:1]), hq, 1,
                             mask="window", window=1100, sinks=2)
        assert (part[0].float() - out[i].float()).abs().max() <= 2 * 3 * 2 ** -8 * v.abs().max()
    for i in (7, 13):
        n_ok = ref.attention(q[i].cpu(), k[i].cpu(), v[i].cpu(), torch.arange(n), torch.arange(n),
                             hq, 1, 1100, 2)
        assert ((out[i].double().cpu() - n_ok[0]).abs() <= n_ok[1]).all()


@pytest.mark.parametrize("n", [40, 500])
def test_scores_that_outgrow_the_first_ones(n):
    """Scores that pass those of the first keys by hundreds of powers of two,
    late in the row, and values near the end of the range: the workgroup takes
    its keys a second time."""
    g = gen(10)
    q, k, v = rand(g, 1, n, 128), rand(g, 1, n, 64), rand(g, 1, n, 64)
    k *= torch.linspace(0.01, 40, n, device="cuda")[:, None].to(BF16)
    check(q, k, v, 2, 1, 300, 1, scale=2.0)
    k = k.flip(1).contiguous()
    check(q, k, v, 2, 1, 300, 1, scale=2.0)
    v[0, 10:20] *= 2.0 ** 105
    check(q, k, v, 2, 1, 300, 1)


@pytest.mark.parametrize("level", [-12.0, -25.0, -60.0, -2000.0])
def test_scores_far_below_zero_and_tiny_values(level):
    """Every score around ``level``: sums of exp(s) that are small or zero, with
    values that a product with them would lose."""
    g = gen(13)
    n = 150
    q, k, v = rand(g, 1, n, 128), rand(g, 1, n, 64, scale=0.05), rand(g, 1, n, 64, scale=2.0 ** -80)
    k[..., 0] = 1.0
    q.view(1, n, 2, 64)[..., 0] = level * 8
    check(q, k, v, 2, 1, 60, 2)


def test_uneven_lengths_and_views():
    """Padded sequences (one empty), fused projection views, a strided output
    whose other columns stay; rows past their window of a short sequence see
    nothing and give zeros."""
    g = gen(2)
    qkv = rand(g, 4, 150, 4 * 64 + 2 * 128)
    lens = torch.tensor([150, 0, 20, 1000], dtype=torch.int32, device="cuda")
    wide = torch.full((4, 150, 4 * 64 + 4), 3.0, dtype=BF16, device="cuda")
    out = check(qkv[:, :, :256], qkv[:, :, 256:384], qkv[:, :, 384:], 4, 2, 30, 0, lens,
                out=wide[:, :, :256])
    assert (wide[:, :, 256:] == 3).all()
    assert (out[1] == 0).all() and (out[2, 49:] == 0).all() and (out[2, :49] != 0).any()


@pytest.mark.parametrize("window,sinks", [(40, 3), (200, 0)])
def test_pieces_of_a_prompt(window, sinks):
    """Rows at a position of their own (one at a time and several) are the
    whole call's rows."""
    g = gen(3)
    n = 170
    q, k, v = rand(g, 1, n, 192), rand(g, 1, n, 64), rand(g, 1, n, 64)
    whole = check(q, k, v, 3, 1, window, sinks)
    for a, b in ((0, 1), (1, 64), (64, 100), (100, 169), (169, 170)):
        part = check(q[:, a:b], k, v, 3, 1, window, sinks, q_pos=a)
        assert (part.float() - whole[:, a:b].float()).abs().max() < 2 ** -6 * whole.abs().max()


@pytest.mark.parametrize("bad", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("where", [0, 90, 64])
def test_unseen_keys_do_not_reach_a_row(bad, where):
    g = gen(4)
    n = 200
    q, k, v = rand(g, 1, n, 128), rand(g, 1, n, 64), rand(g, 1, n, 64)
    v[0, where, 10:30] = float(bad)
    check(q, k, v, 2, 1, 33, 1)
    k[0, where, 5] = float("nan")
    check(q, k, v, 2, 1, 33, 1)
    # behind the end of a sequence nothing counts
    lens = torch.tensor([where], dtype=torch.int32, device="cuda")
    out = check(q, k, v, 2, 1, 33, 1, lens)
    assert torch.isfinite(out).all()


def test_both_infinities_make_nan():
    g = gen(5)
    q, k, v = rand(g, 1, 70, 64), rand(g, 1, 70, 64), rand(g, 1, 70, 64)
    v[0, 10, 3], v[0, 12, 3] = float("inf"), float("-inf")
    check(q, k, v, 1, 1, 16)


def test_large_scores_and_scale():
    g = gen(6)
    n = 300
    q, k, v = rand(g, 1, n, 128, scale=5.0), rand(g, 1, n, 64, scale=5.0), rand(g, 1, n, 64)
    check(q, k, v, 2, 1, 100, 2, scale=0.5)


def test_a_window_over_everything_equals_the_causal_kernel():
    """The library's causal attention is the case of a window that holds all."""
    g = gen(7)
    for b, n, hq in ((1, 241, 3), (40, 300, 6)):
        q, k, v = rand(g, b, n, hq * 64), rand(g, b, n, 64), rand(g, b, n, 64)
        a = ops.attention(q, k, v, torch.empty_like(q), hq, 1, mask="causal")
        w = ops.attention(q, k, v, torch.empty_like(q), hq, 1, mask="window", window=n)
        # both round the probabilities and the output: twice the bound of one
        scale = 2 * (2 ** -8 * 2 + 2 ** -8) * v.float().abs().max()
        assert (a.float() - w.float()).abs().max() <= scale


def test_sizes_past_32_bits_mean_everything():
    g = gen(11)
    q, k, v = rand(g, 1, 90, 128), rand(g, 1, 90, 64), rand(g, 1, 90, 64)
    a = ops.attention(q, k, v, torch.empty_like(q), 2, 1, mask="window", window=90)
    for kw in (dict(window=2 ** 32 + 1), dict(window=1, sinks=2 ** 32 + 1)):
        b = ops.attention(q, k, v, torch.empty_like(q), 2, 1, mask="window", **kw)
        assert torch.equal(a, b)


def test_time_before_batch_and_in_place():
    """[T, B, .] tensors as [B, T, .] views, and the output over the queries."""
    g = gen(12)
    q, k, v = (rand(g, 70, 3, w).transpose(0, 1) for w in (128, 64, 64))
    out = torch.empty(70, 3, 128, dtype=BF16, device="cuda").transpose(0, 1)
    check(q, k, v, 2, 1, 20, 2, out=out)
    want = out.clone()
    ops.attention(q, k, v, q, 2, 1, mask="window", window=20, sinks=2)
    assert torch.equal(q, want)


def test_captured_call():
    g = gen(8)
    q, k, v = rand(g, 2, 100, 128), rand(g, 2, 100, 64), rand(g, 2, 100, 64)
    lens = torch.tensor([100, 60], dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    run = lambda o: ops.attention(q, k, v, o, 2, 1, mask="window", window=9, sinks=1, lens=lens)  # noqa: E731
    run(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(out)
    for i in range(4):
        q.copy_(rand(g, 2, 100, 128))
        lens.fill_(100 - 20 * i)
        graph.replay()
        assert torch.equal(out, run(torch.empty_like(q)))
        torch.cuda.synchronize()


def test_refusals():
    from smolvla._lib import SvlaError
    g = gen(9)
    q, k = rand(g, 2, 8, 128), rand(g, 2, 8, 64)
    o = torch.empty_like(q)
    call = lambda q=q, k=k, v=k, o=o, hq=2, hkv=1, **kw: ops.attention(  # noqa: E731
        q, k, v, o, hq, hkv, **{"mask": "window", "window": 4, **kw})
    for kw in (dict(window=None), dict(q=q.float()), dict(k=k[:1]), dict(v=k[:, :4]),
               dict(o=o[:, :, :64]), dict(lens=torch.ones(1, dtype=torch.int32, device="cuda")),
               dict(lens=torch.ones(2, device="cuda")), dict(prefix_len=3), dict(q_lo=q),
               dict(window=0), dict(window=-1), dict(sinks=-1), dict(q_pos=-1), dict(q_pos=2 ** 32),
               dict(o=o[:1].expand(2, -1, -1)), dict(mask="causal"), dict(q=q.cpu()), dict(mask="none", window=None, sinks=1)):
        with pytest.raises(ValueError):
            call(**kw)
    for kw in (dict(scale=0.0), dict(scale=float("nan")), dict(hq=2, hkv=3, k=rand(g, 2, 8, 192), v=rand(g, 2, 8, 192)),
               dict(q=rand(g, 2, 8, 129)[:, :, 1:])):
        with pytest.raises(SvlaError):
            call(**kw)
    assert call(q=q[:, :0], o=o[:, :0]).shape == (2, 0, 128)
