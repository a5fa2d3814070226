"""ops.attention_weights against a 64-bit softmax summed over queries and grouped heads."""

import pytest
import torch

from chunkkv_amd import ops
from tests import decode_cache_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def _randn(shape, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(BF).to(DEV)


def _check(q, K, pos, prior=None, scale=None, out=None):
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    base = None if prior is None else prior.clone()
    got = ops.attention_weights(q, K, pos.to(DEV), scale, prior=prior, out=out, err=err)
    assert int(err) == 0 and got.shape == K.shape[:3] and got.dtype == torch.float32
    want, most = R.weights(q, K, pos, q.shape[3] ** -0.5 if scale is None else scale, base)
    off = (got.double().cpu() - want).abs()
    assert (off <= most).all(), f"{float((off / most).max())} times the bound"
    last = int(pos.max())
    assert torch.equal(got[:, :, last + 1 :].cpu(), (torch.zeros_like(got) if base is None else base)[:, :, last + 1 :].cpu())
    return got


@pytest.mark.parametrize(
    "Hq,Hkv,D,N,n",
    [
        (28, 4, 128, 1, 1),
        (28, 4, 128, 100, 1),
        (28, 4, 128, 8257, 1),  # split over the cache
        (14, 2, 64, 333, 1),
        (28, 4, 128, 4100, 64),  # a window of the last tokens
        (14, 2, 64, 1103, 251),
        (8, 8, 64, 200, 200),  # no shared heads, causal
        (28, 4, 128, 700, 700),
        (6, 3, 64, 129, 65),  # heads that do not divide 8
        (64, 1, 128, 130, 9),  # a group of 64
        (4, 4, 128, 64, 17),
        (28, 4, 128, 1024, 2),  # up to 16 rows of a KV head: whole, and split from 1025 cached rows on
        (28, 4, 128, 1025, 2),
        (16, 1, 64, 1024, 1),
        (17, 1, 64, 1024, 1),  # 17 rows
        (4, 4, 64, 1023, 16),
        (28, 4, 128, 64, 64),  # a short cache: one launch
        (28, 4, 128, 256, 27),
        (28, 4, 128, 256, 28),  # and three
        (14, 2, 64, 257, 3),
        (14, 2, 64, 33, 33),
        (16, 16, 64, 193, 190),
        (40, 2, 128, 2, 2),
        (14, 2, 64, 13000, 520),  # more splits over a long cache
        (28, 4, 128, 2050, 18),  # 64 rows a workgroup, a split joined by the second pass
        (28, 4, 128, 1103, 128),  # in parts too
        (28, 4, 128, 2050, 64),  # 448 rows and 11 splits: joined by a launch
        (28, 4, 128, 5185, 3),
        (14, 2, 64, 16500, 300),  # 128 rows a workgroup in both passes
        (14, 2, 64, 40000, 90),  # in the second only
        (16, 16, 64, 650, 250),
        (1, 1, 128, 300, 257),
    ],
)
def test_weights_match_the_plain_form(Hq, Hkv, D, N, n):
    q = _randn((1, n, Hq, D), N).transpose(1, 2)
    K = _randn((1, Hkv, N, D), n, 1.5)
    pos = torch.randperm(N, generator=torch.Generator().manual_seed(n))[:n].sort().values
    pos[-1] = N - 1
    prior = torch.rand((1, Hkv, N), device=DEV) if n % 2 else None
    _check(q, K, pos, prior)


def test_every_weight_of_a_query_sums_to_one():
    q, K = _randn((1, 28, 40, 128), 1), _randn((1, 4, 500, 128), 2, 3.0)
    got = ops.attention_weights(q, K, torch.arange(460, 500, device=DEV))
    assert torch.allclose(got.double().sum(2), torch.full((1, 4), 7 * 40.0, dtype=torch.float64, device=DEV), rtol=1e-5)


def test_rows_behind_the_positions_and_views_of_longer_caches():
    """Rows past the last position hold NaN; K and its positions are views of a longer slab; positions unsorted."""
    slab = _randn((1, 2, 640, 64), 3)
    slab[:, :, 301:] = float("nan")
    pos = torch.tensor([300, 0, 77, 5, 77, 300, 64, 63])
    _check(_randn((1, 14, 8, 64), 4), slab[:, :, :400], pos)


@pytest.mark.parametrize("Hq,Hkv,D,N,last,n", [(28, 4, 128, 200, 130, 12), (14, 2, 64, 60, 0, 40), (28, 4, 128, 1103, 700, 128),
                                               (14, 2, 64, 9000, 8200, 100), (28, 4, 128, 4100, 65, 40), (28, 4, 128, 900, 777, 1)])
def test_rows_behind_the_positions_in_every_form(Hq, Hkv, D, N, last, n):
    K = _randn((1, Hkv, N, D), 3)
    K[:, :, last + 1 :] = float("nan")
    pos = torch.randint(0, last + 1, (n,), generator=torch.Generator().manual_seed(N))
    pos[n // 2] = last
    _check(_randn((1, Hq, n, D), 4), K, pos, torch.rand((1, Hkv, N), device=DEV))


@pytest.mark.parametrize("Hq,Hkv,D,N,n", [(28, 4, 128, 100, 20), (14, 2, 64, 600, 300), (28, 4, 128, 5000, 40)])
def test_positions_outside_in_every_form(Hq, Hkv, D, N, n):
    q, K, err = _randn((1, Hq, n, D), 1), _randn((1, Hkv, N, D), 2), torch.zeros(1, dtype=torch.int32, device=DEV)
    pos = torch.randint(0, N, (n,), generator=torch.Generator().manual_seed(n)).to(DEV)
    wild = pos.clone()
    pos[0], pos[n - 1], wild[0], wild[n - 1] = 0, N - 1, -(2**40), N
    got = ops.attention_weights(q, K, wild, err=err)
    assert int(err) == 1
    assert torch.equal(got, ops.attention_weights(q, K, pos))


def test_rows_of_very_different_scores():
    """Scores from -600 to 600: sums that start far below a later maximum, weights that vanish."""
    K = _randn((1, 2, 777, 64), 5, 30.0)
    _check(_randn((1, 4, 50, 64), 6, 4.0), K, torch.arange(727, 777))
    _check(_randn((1, 4, 50, 64), 6, 4.0), K[:, :, :200], torch.arange(150, 200))
    _check(_randn((1, 4, 1, 64), 6, 0.0), K, torch.tensor([776]))  # all scores 0: 1 / 777 each


def test_weights_that_grow_in_place_over_a_captured_step():
    """prior and out one tensor, one token a step, captured: 6 replays against the eager sum."""
    N, steps = 900, 6
    K, q = _randn((1, 4, N + steps, 128), 7), _randn((1, 28, steps, 128), 8)
    at, qb = torch.tensor([N], device=DEV), torch.empty_like(q[:, :, :1])
    w, eager = torch.zeros((1, 4, N + steps), device=DEV), torch.zeros((1, 4, N + steps), device=DEV)
    qb.copy_(q[:, :, :1])
    ops.attention_weights(qb, K, at)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_weights(qb, K, at, prior=w, out=w)
        at.add_(1)
    for i in range(steps):
        qb.copy_(q[:, :, i : i + 1])
        graph.replay()
        eager = ops.attention_weights(q[:, :, i : i + 1], K, torch.tensor([N + i], device=DEV), prior=eager)
        assert torch.equal(w, eager)


@pytest.mark.parametrize("Hq,Hkv,D,N,n", [(28, 4, 128, 64, 20), (28, 4, 128, 2050, 64), (28, 4, 128, 1103, 128), (14, 2, 64, 9000, 1)])
def test_graph_replays_match_eager(Hq, Hkv, D, N, n):
    K, q, pos = _randn((1, Hkv, N, D), 1), _randn((1, Hq, n, D), 2), torch.arange(N - n, N, device=DEV)
    prior = torch.rand((1, Hkv, N), device=DEV)
    ops.attention_weights(q, K, pos, prior=prior)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.attention_weights(q, K, pos, prior=prior)
    for step in range(5):
        q.copy_(_randn((1, Hq, n, D), 20 + step))
        pos.copy_(torch.randint(0, N, (n,), generator=torch.Generator().manual_seed(step)))
        graph.replay()
        assert torch.equal(out, ops.attention_weights(q, K, pos, prior=prior))


def test_two_calls_give_the_same_bits_and_streams_do_not_mix():
    q, K, pos = _randn((1, 28, 100, 128), 9), _randn((1, 4, 3000, 128), 10), torch.arange(2900, 3000, device=DEV)
    want = ops.attention_weights(q, K, pos)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.attention_weights(q, K, pos))
    torch.cuda.synchronize()
    assert all(torch.equal(want, g) for g in got)


def test_positions_outside_are_clamped_and_flagged():
    q, K, err = _randn((1, 4, 3, 64), 1), _randn((1, 2, 100, 64), 2), torch.zeros(1, dtype=torch.int32, device=DEV)
    got = ops.attention_weights(q, K, torch.tensor([-3, 50, 10**12], device=DEV), err=err)
    assert int(err) == 1
    assert torch.equal(got, ops.attention_weights(q, K, torch.tensor([0, 50, 99], device=DEV)))


def test_no_queries():
    K, none = _randn((1, 2, 100, 64), 2), torch.zeros(0, dtype=torch.int64, device=DEV)
    q, prior = _randn((1, 4, 0, 64), 1), torch.rand((1, 2, 100), device=DEV)
    assert not ops.attention_weights(q, K, none).any()
    assert torch.equal(ops.attention_weights(q, K, none, prior=prior), prior)
    assert ops.attention_weights(q, K, none, prior=prior, out=prior) is prior


def test_offsets_past_32_bits():
    N, D = 17_000_001, 128  # 4.35 GB of keys
    K = torch.zeros((1, 1, N, D), dtype=BF, device=DEV)
    K[0, 0, N - 1] = 8.0
    q = torch.full((1, 2, 1, D), 2.0, dtype=BF, device=DEV)
    got = ops.attention_weights(q, K, torch.tensor([N - 1], device=DEV))
    assert float(got[0, 0, N - 1]) == pytest.approx(2.0, rel=1e-6) and float(got[0, 0, : N - 1].max()) < 1e-30


def test_refusals():
    q, K, pos = _randn((1, 4, 2, 64), 1), _randn((1, 2, 100, 64), 2), torch.tensor([0, 1], device=DEV)
    f = lambda *s: torch.zeros(s, device=DEV)  # noqa: E731
    for args, kw in (((q, K[:, :, ::2], pos), {}), ((q[:, :3], K, pos), {}), ((q[..., :32], K, pos), {}), ((q, K, pos[:1]), {}),
                     ((q, K, pos.int()), {}), ((q, K, pos.cpu()), {}), ((q, K.cpu(), pos), {}), ((q, K, pos, 0.0), {}),
                     ((q, K, pos), {"prior": f(1, 2, 99)}), ((q, K, pos), {"out": f(1, 2, 100).double()}),
                     ((q, K, pos), {"prior": f(1, 2, 200)[:, :, ::2]}), ((q, K, pos), {"err": f(1)}),
                     ((torch.cat([q, q]), K, pos), {}), ((q, torch.cat([K, K]), pos), {}),
                     ((_randn((1, 4, 2, 96), 1), _randn((1, 2, 100, 96), 2), pos), {})):
        with pytest.raises(ValueError):
            ops.attention_weights(*args, **kw)
    buf = f(201)  # out moved by one row against prior
    with pytest.raises(ValueError):
        ops.attention_weights(q, K, pos, prior=buf[:200].view(1, 2, 100), out=buf[1:].view(1, 2, 100))
    with pytest.raises(TypeError):
        ops.attention_weights(q.float(), K, pos)
    with pytest.raises(TypeError):
        ops.attention_weights(q, K.float(), pos)
