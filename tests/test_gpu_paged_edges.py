"""The paged cache's and the logits' operators at requests past what they count in, broken tables, infinities, and buffers that overlap."""

import pytest
import torch

from chunkkv_amd import _native, ops
from tests import paged_ref as R
from tests.test_gpu_attention_paged import _batch, _check, _want

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, I32, F32 = torch.bfloat16, torch.int32, torch.float32


def _ints(v):
    return torch.tensor(v, dtype=I32, device=DEV)


def test_more_pages_asked_for_than_32_bits_count():
    """65 sequences ask for 2^26 - 2 pages each, 2^32 and some together, of a pool of four; the one behind them for one: none grows."""
    M, T, S = 2**26 - 1, 32, 66
    k = torch.zeros((1, 1, 1, 4 * T, 64), dtype=BF, device=DEV)
    c = ops.PagedCache(k, k.clone(), torch.empty((S, M), dtype=I32, device=DEV), torch.zeros(S, dtype=I32, device=DEV), torch.zeros(4, dtype=I32, device=DEV), T)
    c.table[:, 0] = 3  # an entry from before
    err = torch.zeros(1, dtype=I32, device=DEV)
    got = ops.extend_pages(c, _ints([2**31 - 64] * 65 + [1]), 1, err)
    assert int(err.item()) == _native.DEVICE_ERR_PAGES
    assert got.rows.tolist() == [-1] and got.positions.tolist() == [0] and not got.starts.any() and not c.lengths.any() and not c.refs.any()


@pytest.mark.parametrize("page", [400, 999, -5, 2**31 - 1, -2**31])
@pytest.mark.parametrize("more", [1, 5000])  # rows by the one launch, and by one of their own
def test_rows_of_a_page_that_the_pool_does_not_have(page, more):
    """A partial last page outside the pool: its new rows are -1 and flagged, the other sequences' are theirs."""
    T, P = 32, 400
    c = ops.paged_cache(1, P, 1, 64, 3, 6000, DEV, T)
    err = torch.zeros(1, dtype=I32, device=DEV)
    ops.extend_pages(c, _ints([70, 40, 0]), 110, err)
    c.table[0, 2] = page
    got = ops.extend_pages(c, _ints([30, more, 0]), 30 + more, err)
    assert int(err.item()) == _native.DEVICE_ERR_RANGE
    assert got.positions.tolist() == [*range(70, 100), *range(40, 40 + more)]
    rows = got.rows.tolist()
    assert rows[:26] == [-1] * 26
    at = got.positions[26:]
    of = torch.tensor([0] * 4 + [1] * more, device=DEV)
    assert rows[26:] == (c.table[of, at // T].long() * T + at % T).tolist() and min(rows[26:]) >= 0


@pytest.mark.parametrize("form", range(len(R.FORMS)))
def test_rows_whose_scores_are_all_minus_infinity(form):
    """They are NaN, as the softmax of -infinities is and as over a contiguous cache; a token that sees no row is zeros; others as ever."""
    heads, seqs, most, known = R.FORMS[form]
    q, cache, starts = _batch(heads, 64, seqs, seed=form)
    q = q.clone(memory_format=torch.preserve_format)
    q[..., 0] = 1.0
    c, last = seqs[0][1], len(seqs) - 1
    at = torch.arange(seqs[0][0], device=DEV)
    rows = cache.table[0, at // 64].long() * 64 + at % 64
    cache.k[0, 0, :, rows, 0] = float("-inf")
    if last > 0:
        cache.lengths[last] = 0  # its new tokens see no row
    total = sum(r for r, _ in seqs) if known else None
    got = ops.attention_paged(q, cache, 0, starts, most=most, total=total)
    assert got[0, :c].isnan().all()
    if last > 0:
        assert not got[0, -seqs[-1][1]:].any()
        middle = slice(c, got.shape[1] - seqs[-1][1])
        if middle.stop > middle.start:
            part = ops.PagedCache(cache.k, cache.v, cache.table[1:-1], cache.lengths[1:-1], cache.refs, 64)
            _check(got[:, middle], _want(q[:, :, middle], part, seqs[1:-1]))
    K, V = (x[0][:, :, rows].contiguous() for x in (cache.k, cache.v))
    assert ops.attention_active(q[:, :, :c], K, V, at[-c:].contiguous()).isnan().all()
