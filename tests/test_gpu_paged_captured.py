"""The page calls captured together, a session over blended prefills, and attention of no token."""

import pytest
import torch

from chunkkv_amd import ops
from chunkkv_amd.types import BlendConfig, Placement
from tests import paged_ref as R
from tests.test_gpu_attention_paged import _batch
from tests.test_gpu_paged_session import _engine, _greedy, _tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = torch.int32


def _ints(v):
    return torch.tensor(v, dtype=I32, device=DEV)


def test_every_page_call_in_one_graph():
    """Extension, forks, going back, ends and compaction, replayed from one book again and again, eager calls between the replays."""
    c = ops.paged_cache(2, 40, 2, 64, 6, 400, DEV, 32)
    err = torch.zeros(1, dtype=I32, device=DEV)
    rows = [100, 40, 70, 0, 0, 33]
    ops.extend_pages(c, _ints(rows), sum(rows), err)
    for t in (c.k, c.v):
        t.normal_()
    parts = (c.table, c.lengths, c.refs, c.k, c.v)
    saved = [t.clone() for t in parts]
    counts, sources, targets, back, keep, ended = _ints([1, 30, 0, 0, 0, 1]), _ints([0, 2]), _ints([3, 4]), _ints([0, 4]), _ints([96, 5]), _ints([1, 5])

    def restore():
        for t, s in zip(parts, saved):
            t.copy_(s)

    def calls():
        new = ops.extend_pages(c, counts, 32, err)
        ops.fork_pages(c, sources, targets, err)
        ops.free_pages(c, back, keep, err)
        ops.free_pages(c, ended, err=err)
        return new, ops.compact_pages(c, err)

    def state(got):
        return [t.clone() for t in (*parts, got[0].positions, got[0].rows, got[0].starts, got[1])]

    want = state(calls())
    b = R.Book(6, c.table.shape[1], 40, 32)
    b.extend(rows, sum(rows))
    assert want[6].tolist() == b.extend([1, 30, 0, 0, 0, 1], 32)[1]
    b.fork([0, 2], [3, 4])
    b.free([0, 4], [96, 5])
    b.free([1, 5])
    assert want[8].tolist() == [b.compact()]
    b.check(c, err)
    restore()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls()
    for _ in range(4):
        restore()
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(state(got), want))
        restore()
        assert all(torch.equal(x, y) for x, y in zip(state(calls()), want))
    assert int(err.item()) == b.err == R.RANGE  # sequence 4 shares the page of its row 5 with sequence 2


def test_blended_prefills_fill_the_cache():
    """Sequences of prefills whose chunks were cached elsewhere; greedy tokens of the blended caches' own decode."""
    eng = _engine()
    a, b = _tokens(40, 1), _tokens(75, 2)
    source = eng.prefill([7] + a + b)
    ca, cb = source.chunks([(1, 41), (41, 116)])
    prompts = [_tokens(9, 3) + b + a + _tokens(11, 4), b + _tokens(21, 5)]
    placed = [[Placement(cb, 9), Placement(ca, 84)], [Placement(cb, 0)]]
    s = eng.paged(n_pages=30, n_sequences=3, max_tokens=300, page_tokens=32)
    results = [eng.prefill(p, pl, BlendConfig()) for p, pl in zip(prompts, placed)]
    ids = [s.add(r, p) for r, p in zip(results, prompts)]
    for i, r in zip(ids, results):
        n = len(prompts[i])
        at = torch.arange(n, device=DEV)
        rows = s.cache.table[i, at // 32].long() * 32 + at % 32
        for layer in range(3):
            assert torch.equal(s.cache.k[layer][:, :, rows], r.keys[layer]) and torch.equal(s.cache.v[layer][:, :, rows], r.values[layer])
    for i, tokens in zip(ids, s.generate(ids, 10)):
        _greedy(results[i].logits[-1], tokens[0])
        assert len(tokens) == 10 and s.tokens[i] == prompts[i] + tokens


def test_attention_of_no_token():
    q, cache, starts = _batch((14, 2, 64), 64, [(70, 2), (5, 1)], seed=1)
    none = torch.zeros_like(starts)
    got = ops.attention_paged(q[:, :, :0], cache, 0, none)
    assert got.shape == (1, 0, 14, 64)
    assert ops.attention_paged(q[:, :, :0], cache, 0, none, out=got).data_ptr() == got.data_ptr()
