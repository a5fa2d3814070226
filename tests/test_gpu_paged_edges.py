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


@pytest.mark.parametrize("most", [1, 40])
@pytest.mark.parametrize("seqs", [[(700, 1), (40, 1)], [(900, 40), (2000, 3)], [(3000, 300)]])
def test_attention_into_a_buffer_that_it_reads_is_refused(seqs, most):
    """Its queries alone may be written over, where each is."""
    hq, _, d = heads = (14, 2, 64)
    q, cache, starts = _batch(heads, 64, seqs, seed=2)
    n = q.shape[2]
    want = ops.attention_paged(q, cache, 0, starts, most=most)
    size = n * hq * d
    for t in (cache.k, cache.v):
        for at in (0, t.numel() - size):
            if 0 <= at:
                with pytest.raises(ValueError, match="overlap"):
                    ops.attention_paged(q, cache, 0, starts, most=most, out=t.view(-1)[at:at + size].view(1, n, hq, d))
    room = torch.zeros(3 * size, dtype=BF, device=DEV)
    held = room[size:2 * size].view(1, n, hq, d)
    held.copy_(q.transpose(1, 2))
    for at in (size - 8, size + 8, 2 * size - 8, 8):
        with pytest.raises(ValueError, match="overlap"):
            ops.attention_paged(held.transpose(1, 2), cache, 0, starts, most=most, out=room[at:at + size].view(1, n, hq, d))
    for at in (0, 2 * size):
        out = room[at:at + size].view(1, n, hq, d)
        assert torch.equal(ops.attention_paged(held.transpose(1, 2), cache, 0, starts, most=most, out=out), want)
    assert ops.attention_paged(held.transpose(1, 2), cache, 0, starts, most=most, out=held).data_ptr() == held.data_ptr() and torch.equal(held, want)
    held.copy_(q.transpose(1, 2))
    if n > 1:
        with pytest.raises(ValueError, match="overlap"):  # heads first: another query is where a result goes
            ops.attention_paged(held.view(1, hq, n, d), cache, 0, starts, most=most, out=held)


def test_attention_beside_its_queries_in_one_buffer_is_accepted():
    """Queries in a wider buffer's columns, the results in what lies between two of its rows: no byte is shared."""
    heads = (4, 2, 64)
    q, cache, starts = _batch(heads, 64, [(300, 2)], seed=2)
    want = ops.attention_paged(q, cache, 0, starts)
    room = torch.zeros((2, 6 * 64 * 4), dtype=BF, device=DEV)
    view = room[:, :256].view(1, 2, 4, 64).transpose(1, 2)
    view.copy_(q)
    out = room[0, 512:1024].view(1, 2, 4, 64)
    assert torch.equal(ops.attention_paged(view, cache, 0, starts, out=out), want)


@pytest.mark.parametrize("vocab", [1000, 5000])
def test_logits_into_a_buffer_that_they_are_made_from_are_refused(vocab):
    g = torch.Generator().manual_seed(1)
    logits = torch.randn((3, vocab), generator=g).to(BF).to(DEV)
    room = torch.zeros(8 * vocab, device=DEV)
    out = room[vocab:4 * vocab].view(3, vocab)
    ids = torch.randint(0, vocab, (3, 10), generator=g).to(DEV)

    def inside(at, x):
        """x's values in the room, `at` elements of fp32 from its front."""
        view = room[at:at + x.numel() * x.element_size() // 4].view(x.dtype).view(x.shape)
        view.copy_(x)
        return view

    bias = torch.randn((3, vocab), generator=g).to(DEV)
    words = -(-vocab // 32)
    bits = torch.randint(-2**31, 2**31, (3, words), generator=g).to(I32).to(DEV)
    rows = torch.rand(3, generator=g).to(DEV)
    for at in (vocab, 2 * vocab + 4, 4 * vocab - 2):
        for kw in (dict(prompt=ids), dict(generated=ids), dict(repetition=rows + 1, prompt=ids), dict(frequency=rows, generated=ids), dict(presence=rows, generated=ids),
                   dict(bias=bias[0]), dict(bias=bias), dict(allowed=bits[0]), dict(allowed=bits)):
            name = next(iter(kw))
            if name == "bias" and kw[name].dim() == 2 and at == vocab:
                continue  # where the result goes: below
            with pytest.raises(ValueError, match="overlap"):
                ops.adjust_logits(logits, out=out, **dict(kw, **{name: inside(at, kw[name])}))
    # a bias of each row where that row's result goes is read first, as float32 logits are; one row's for one row too
    want = ops.adjust_logits(logits, bias=bias)
    assert torch.equal(ops.adjust_logits(logits, bias=inside(vocab, bias), out=out), want)
    want = ops.adjust_logits(logits[:1], bias=bias[0])
    assert torch.equal(ops.adjust_logits(logits[:1], bias=inside(vocab, bias[0]), out=out[:1]), want)
    # beside it
    want = ops.adjust_logits(logits, bias=bias[0], prompt=ids, repetition=2.0)
    assert torch.equal(ops.adjust_logits(logits, bias=inside(0, bias[0]), prompt=inside(4 * vocab, ids), repetition=2.0, out=out), want)


@pytest.mark.parametrize("vocab", [1000, 5000])
def test_tokens_into_a_buffer_that_they_are_chosen_from(vocab):
    """A row's token may go behind its own history; rows of one slice of the vocabulary end in any order, so over others' histories only where a second
    launch writes the tokens."""
    g = torch.Generator().manual_seed(1)
    logits = torch.randn((3, vocab), generator=g).to(BF).to(DEV)
    logits[:, 7] = 9.0
    ids = torch.randint(0, vocab, (3, 10), generator=g).to(DEV)
    ids[:, 4] = 7
    want = ops.next_tokens(logits, generated=ids, presence=20.0)
    for i in range(3):
        one = ids[i:i + 1].clone()
        assert ops.next_tokens(logits[i:i + 1], generated=one, presence=20.0, out=one[0, 4:5]).item() == want[i] == one[0, 4]
    for at in (0, 9, 27):
        held = ids.clone()
        call = lambda: ops.next_tokens(logits, generated=held, presence=20.0, out=held.view(-1)[at:at + 3])  # noqa: E731
        if vocab > 4096:
            assert torch.equal(call(), want)
        else:
            with pytest.raises(ValueError, match="overlap"):
                call()
    wide = ids.t().contiguous()  # tokens first: a step's tokens lie together
    assert torch.equal(ops.next_tokens(logits, generated=wide.t(), presence=20.0, out=wide[4]), want) and torch.equal(wide[4], want)


def test_a_sequence_named_twice_going_back_counts_the_first_time():
    """What is asked for it the second time is no error, whatever it is."""
    c = ops.paged_cache(1, 12, 1, 64, 3, 200, DEV, 32)
    book, err = R.Book(3, c.table.shape[1], 12, 32), torch.zeros(1, dtype=I32, device=DEV)
    for call in (lambda x: x.extend([70, 0, 40], 110), lambda x: x.fork([0], [1])):
        call(book)
    ops.extend_pages(c, _ints([70, 0, 40]), 110, err)
    ops.fork_pages(c, _ints([0]), _ints([1]), err)
    for at, left in (([0, 0], [66, -1]), ([0, 2, 0, 2], [64, 39, 40, -7]), ([1, 1], [70, 33]), ([2, 2], [-1, 5]), ([0, 0], [40, 32])):
        book.err = 0
        err.zero_()
        book.free(at, left)
        ops.free_pages(c, _ints(at), _ints(left), err)
        book.check(c, err)
