"""ops.attention_paged against a 64-bit form, over every kernel form, ragged batches, lengths and pages."""

import random

import pytest
import torch

from chunkkv_amd import ops
from tests import paged_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, I32 = torch.bfloat16, torch.int32
HEADS = [(28, 4, 128), (14, 2, 64), (8, 8, 64), (6, 3, 128), (32, 1, 64), (3, 1, 128)]


def _batch(heads, T, seqs, seed, extra=2, fill=None):
    """seqs: (rows, new tokens) of each sequence, pages anywhere in the pool; rows that no sequence has hold `fill`."""
    hq, h, d = heads
    rng = random.Random(seed)
    g = torch.Generator().manual_seed(seed)
    need = [-(-r // T) for r, _ in seqs]
    P, M = sum(need) + extra, max(need + [1]) + 1
    order = list(range(P))
    rng.shuffle(order)
    table = torch.full((len(seqs), M), rng.choice([-1, 7 * 10**8]), dtype=I32)
    used = torch.zeros(P * T, dtype=torch.bool)
    for s, (r, _) in enumerate(seqs):
        for j in range(need[s]):
            table[s, j] = order.pop()
        at = torch.arange(r)
        used[table[s, at // T].long() * T + at % T] = True
    K = torch.randn((1, 1, h, P * T, d), generator=g) * torch.where(torch.rand((1, 1, h, 1, d), generator=g) < 0.06, 4.0, 0.8)
    V = torch.randn((1, 1, h, P * T, d), generator=g) * torch.exp(0.5 * torch.randn((1, 1, h, P * T, 1), generator=g))
    if fill is not None:
        K[:, :, :, ~used], V[:, :, :, ~used] = fill, fill
    n = sum(c for _, c in seqs)
    q = (0.7 * torch.randn((1, n, hq, d), generator=g)).to(BF).to(DEV).transpose(1, 2)
    starts = torch.tensor([sum(c for _, c in seqs[:i]) for i in range(len(seqs) + 1)], dtype=I32)
    cache = ops.PagedCache(K.to(BF).to(DEV), V.to(BF).to(DEV), table.to(DEV), torch.tensor([r for r, _ in seqs], dtype=I32, device=DEV),
                           torch.ones(P, dtype=I32, device=DEV), T)
    return q, cache, starts.to(DEV)


def _want(q, cache, seqs, scale=None):
    """(n, Hq, D) results and bounds, sequence by sequence."""
    out, bound, t = [], [], 0
    for s, (r, c) in enumerate(seqs):
        at = torch.arange(r)
        rows = cache.table[s].cpu()[at // cache.page_tokens].long() * cache.page_tokens + at % cache.page_tokens
        K, V = (x[0, 0][:, rows.to(DEV)] for x in (cache.k, cache.v))
        o, b = R.attention(q[0, :, t:t + c], K, V, c, scale)
        out.append(o)
        bound.append(b)
        t += c
    return torch.cat(out), torch.cat(bound)


def _check(got, want):
    got = got[0].double().cpu()
    bad = ~((got - want[0]).abs() <= want[1])
    assert not bad.any(), (bad.sum().item(), (got - want[0]).abs().max().item(), ((got - want[0]).abs() / want[1]).max().item())


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("T", [32, 64, 128])
@pytest.mark.parametrize("seqs", [
    [(1, 1)], [(33, 1)], [(1000, 1)], [(2500, 1)],
    [(5, 1), (0, 0), (700, 1), (64, 1), (31, 0), (1300, 1)],  # a decode step, slots without a sequence and without a token
    [(3, 3)], [(40, 7), (129, 2)], [(900, 5), (64, 64), (0, 0), (257, 33)],
    [(300, 300)], [(1500, 130), (77, 1), (200, 200), (513, 40)],
])
def test_matches_the_64_bit_form(heads, T, seqs):
    q, cache, starts = _batch(heads, T, seqs, seed=len(seqs) * 1000 + T)
    want = _want(q, cache, seqs)
    most = max(c for _, c in seqs)
    err = torch.zeros(1, dtype=I32, device=DEV)
    for kw in (dict(most=most), dict(), dict(most=1), dict(most=most, split=False)):  # most chooses the form only
        _check(ops.attention_paged(q, cache, 0, starts, err=err, **kw), want)
    assert int(err.item()) == 0


@pytest.mark.parametrize("form", range(len(R.FORMS)))
def test_every_kernel_form(form):
    heads, seqs, most, known = R.FORMS[form]
    q, cache, starts = _batch(heads, 64, seqs, seed=form)
    total = sum(r for r, _ in seqs) if known else None
    _check(ops.attention_paged(q, cache, 0, starts, most=most, total=total), _want(q, cache, seqs))


@pytest.mark.parametrize("seqs", [[(1, 1)], [(700, 1), (0, 0), (64, 30), (3000, 2)], [(900, 300), (40, 1)], [(60, 1)] * 70 + [(4000, 9)]])
@pytest.mark.parametrize("heads", [(28, 4, 128), (14, 2, 64)])
def test_estimates_choose_the_form_only(heads, seqs):
    """Whatever most, longest and total say, far too little or too much."""
    q, cache, starts = _batch(heads, 32, seqs, seed=11)
    want = _want(q, cache, seqs)
    for most in (1, 5, 10**6):
        for longest in (1, 600, 2**31 - 1):
            for total in (None, 1, 10**12):
                _check(ops.attention_paged(q, cache, 0, starts, most=most, longest=longest, total=total), want)


@pytest.mark.parametrize("heads", [(28, 4, 128), (14, 2, 64)])
@pytest.mark.parametrize("seqs", [[(9000, 1)], [(9000, 3), (100, 1)], [(6000, 20)], [(5000, 1)] * 3 + [(17, 1)] * 40, [(20000, 4)]])
def test_long_caches(heads, seqs):
    q, cache, starts = _batch(heads, 64, seqs, seed=len(seqs))
    want = _want(q, cache, seqs)
    for kw in (dict(most=max(c for _, c in seqs)), dict(most=1000)):
        _check(ops.attention_paged(q, cache, 0, starts, **kw), want)


@pytest.mark.parametrize("S", [64, 65, 200, 1000, 4096])
def test_many_sequences(S):
    rng = random.Random(S)
    seqs = [(rng.choice([1, 5, 33, 64, 200]), 1) if rng.random() < 0.8 else (rng.choice([0, 9]), 0) for _ in range(S)]
    q, cache, starts = _batch((4, 2, 64), 32, seqs, seed=S)
    _check(ops.attention_paged(q, cache, 0, starts, most=1), _want(q, cache, seqs))
    _check(ops.attention_paged(q, cache, 0, starts), _want(q, cache, seqs))


@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
@pytest.mark.parametrize("most", [1, 2, 40])
def test_rows_that_no_sequence_has_may_hold_anything(fill, most):
    seqs = [(r, min(r, most)) for r in (1, 31, 33, 64, 65, 127, 300, 1025)]
    q, cache, starts = _batch((28, 4, 128), 64, seqs, seed=3, fill=fill)
    for kw in (dict(most=most), dict(most=500)):
        _check(ops.attention_paged(q, cache, 0, starts, **kw), _want(q, cache, seqs))


@pytest.mark.parametrize("most", [1, 20, 200])
def test_tokens_that_see_no_row_give_zeros(most):
    """More new tokens than rows: the first of them are in front of the sequence."""
    seqs, given = [(0, 0), (7, 7), (700, 1)], [(0, 3), (7, 10), (700, 1)]
    q, cache, _ = _batch((28, 4, 128), 32, given, seed=4)
    starts = torch.tensor([0, 3, 13, 14], dtype=I32, device=DEV)
    got = ops.attention_paged(q, cache, 0, starts, most=most)
    assert not got[0, :6].any()
    want = _want(torch.cat([q[:, :, 6:]], 2), cache, seqs)
    _check(got[:, 6:], want)


def test_tokens_outside_the_starts_stay():
    seqs = [(50, 2), (100, 1)]
    q, cache, starts = _batch((14, 2, 64), 32, seqs, seed=5)
    q = torch.cat([q[:, :, :1], q, q[:, :, :2]], 2)
    for most in (1, 2, 300):
        out = torch.full((1, 6, 14, 64), 5.0, dtype=BF, device=DEV)
        got = ops.attention_paged(q, cache, 0, starts + 1, most=most, out=out)
        assert got.data_ptr() == out.data_ptr() and (out[0, 0] == 5).all() and (out[0, 4:] == 5).all()
        _check(out[:, 1:4], _want(q[:, :, 1:4], cache, seqs))


@pytest.mark.parametrize("starts", [[0, 5, 3, 8], [8, 0, 0, 8], [-4, 2, 900, 8], [0, 0, 0, 0]])
def test_starts_that_are_none_touch_nothing_else(starts):
    """Whatever starts, lengths and table hold: tokens outside every range stay, and the call ends."""
    q, cache, _ = _batch((28, 4, 128), 32, [(60, 2), (300, 3), (9, 3)], seed=6)
    guard = torch.full((3, 8, 28, 128), 7.0, dtype=BF, device=DEV)
    cache.lengths.copy_(torch.tensor([10**9, -5, 40], dtype=I32))
    err = torch.zeros(1, dtype=I32, device=DEV)
    for most in (1, 3, 400):
        ops.attention_paged(q, cache, 0, torch.tensor(starts, dtype=I32, device=DEV), most=most, out=guard[1:2], err=err)
        assert (guard[0] == 7).all() and (guard[2] == 7).all()
    if starts == [0, 0, 0, 0]:
        assert (guard == 7).all()


def test_layers_strides_and_scale():
    """Another layer of a pool of three, queries as a view with room between the heads, a scale of its own."""
    seqs = [(333, 5), (40, 40)]
    q, cache, starts = _batch((6, 3, 128), 64, seqs, seed=7)
    pools = [torch.randn((3, *p.shape[1:]), device=DEV).to(BF) for p in (cache.k, cache.v)]
    for pool, one in zip(pools, (cache.k, cache.v)):
        pool[1] = one[0]
    three = ops.PagedCache(*pools, cache.table, cache.lengths, cache.refs, 64)
    wide = torch.randn((1, 45, 9, 136), device=DEV).to(BF)
    wide[:, :, 2:8, :128] = q.transpose(1, 2)
    view = wide[:, :, 2:8, :128].transpose(1, 2)
    _check(ops.attention_paged(view, three, 1, starts, 0.05), _want(q, cache, seqs, 0.05))


def test_graph_replays_follow_the_lengths():
    """A captured decode step: lengths grow between replays, partial rows of other lengths stand in the workspace."""
    rows = [700, 3, 5000, 64]
    q, cache, starts = _batch((28, 4, 128), 64, [(r + 40, 1) for r in rows], seed=8)
    q2 = q.clone(memory_format=torch.preserve_format)
    ops.attention_paged(q2, cache, 0, starts, most=1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.attention_paged(q2, cache, 0, starts, most=1)
    for add in (0, 1, 40, 7):
        seqs = [(r + add, 1) for r in rows]
        cache.lengths.copy_(torch.tensor([r for r, _ in seqs], dtype=I32))
        graph.replay()
        _check(got, _want(q2, cache, seqs))
        eager = ops.attention_paged(q2, cache, 0, starts, most=1)
        assert torch.equal(eager, got)


def test_other_streams_and_two_calls_at_once():
    seqs = [(3000, 1), (40, 1)]
    q, cache, starts = _batch((28, 4, 128), 32, seqs, seed=9)
    want = _want(q, cache, seqs)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for st in streams:
        with torch.cuda.stream(st):
            got.append(ops.attention_paged(q, cache, 0, starts, most=1))
    torch.cuda.synchronize()
    for o in got:
        _check(o, want)
