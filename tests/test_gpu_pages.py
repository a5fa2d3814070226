"""The book and the copies of a paged cache against a Python form of it: every table entry, count and row."""

import random

import pytest
import torch

from chunkkv_amd import ops
from tests.paged_ref import Book

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = torch.int32


def _ints(v):
    return torch.tensor(v, dtype=I32, device=DEV)


def _cache(S, max_tokens, P, T, layers=2, H=2, D=64, dtype=torch.bfloat16):
    c = ops.paged_cache(layers, P, H, D, S, max_tokens, DEV, T, dtype)
    for t in (c.k, c.v):  # any finite values
        t.copy_(torch.randn(t.shape[2:], device=DEV).to(dtype).expand(t.shape))
    return c, Book(S, c.table.shape[1], P, T), torch.zeros(1, dtype=I32, device=DEV)


class Held:
    """What every row of every sequence holds, written at extension and read back through the table."""

    def __init__(self, cache, book):
        self.cache, self.book, self.rows = cache, book, [[] for _ in book.lengths]
        self.next = 1

    def write(self, rows, starts):
        c = self.cache
        for s in range(len(self.rows)):
            at = [r for r in rows[starts[s]:starts[s + 1]]]
            ids = list(range(self.next, self.next + len(at)))
            self.next += len(at)
            self.rows[s] += ids
            if at:
                i = torch.tensor(at, device=DEV)
                v = torch.tensor(ids, device=DEV)
                for t, k in ((c.k, 0), (c.v, 128)):  # ids up to 2^14 as two exact parts
                    t[:, :, :, i, 0] = (v % 128 + k).to(t.dtype)
                    t[:, :, :, i, -1] = (v // 128).to(t.dtype)

    def check(self):
        c = self.cache
        for s, ids in enumerate(self.rows):
            i = self.book.rows(s).to(DEV)
            assert len(i) == len(ids)
            if not ids:
                continue
            for t, k in ((c.k, 0), (c.v, 128)):
                got = t[:, 0, :, i, 0].float() - k + 128 * t[:, 0, :, i, -1].float()
                want = torch.tensor(ids, device=DEV).float().expand(got.shape)
                assert torch.equal(got, want), f"sequence {s}"


@pytest.mark.parametrize("T,S,max_tokens,P,dtype,D", [(32, 5, 300, 30, torch.bfloat16, 64), (64, 9, 700, 41, torch.float32, 128), (128, 3, 500, 9, torch.bfloat16, 256),
                                                      (32, 40, 90, 65, torch.bfloat16, 128)])
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_a_life_of_calls(T, S, max_tokens, P, dtype, D, seed):
    """Random calls, some of which do not fit: the book, the rows' contents and the flags after each."""
    rng = random.Random(seed * 100 + T)
    c, book, err = _cache(S, max_tokens, P, T, D=D, dtype=dtype)
    held = Held(c, book)
    for _ in range(25):
        what = rng.choice(["extend", "extend", "extend", "fork", "free", "keep", "compact"])
        if what == "extend":
            counts = [rng.choice([0, 0, 1, 1, rng.randint(0, max_tokens // 2), T, max_tokens + T, -1][:8 if rng.random() < 0.2 else 6]) for _ in range(S)]
            fits = [x for x in counts if x > 0]
            n = rng.choice([sum(fits), sum(fits) + 3, max(0, sum(fits) - 1)])
            want = book.extend(counts, n)
            got = ops.extend_pages(c, _ints(counts), n, err)
            assert got.positions.tolist() == want[0] and got.rows.tolist() == want[1] and got.starts.tolist() == want[2]
            held.write(want[1], want[2])
        elif what == "fork":
            pairs = [(rng.randrange(-1 if rng.random() < 0.1 else 0, S), rng.randrange(S)) for _ in range(rng.randint(1, 4))]
            before = [list(r) for r in held.rows]
            lengths = list(book.lengths)
            book.fork([a for a, _ in pairs], [b for _, b in pairs])
            ops.fork_pages(c, _ints([a for a, _ in pairs]), _ints([b for _, b in pairs]), err)
            for a, b in pairs:
                if lengths[b] == 0 and book.lengths[b] > 0:
                    held.rows[b] = list(before[next(x for x, y in pairs if y == b)])
        elif what == "free":
            ended = [rng.randrange(S) for _ in range(rng.randint(1, 3))] + ([S] if rng.random() < 0.1 else [])
            book.free(ended)
            ops.free_pages(c, _ints(ended), err=err)
            for s in ended:
                if s < S:
                    held.rows[s] = []
        elif what == "keep":
            at = rng.sample(range(S), min(S, 3))
            left = [rng.choice([0, rng.randint(-1, max_tokens), T * rng.randint(0, 4)]) for _ in at]
            book.free(at, left)
            ops.free_pages(c, _ints(at), _ints(left), err)
            for s in at:
                held.rows[s] = held.rows[s][:book.lengths[s]]
        else:
            assert ops.compact_pages(c, err).tolist() == [book.compact()]
        book.check(c, err)
        held.check()


@pytest.mark.parametrize("P", [1, 3, 1023, 1024, 1025, 4097, 40000])
def test_pools_of_all_sizes(P):
    """Pages are found wherever they are free, and moved together."""
    rng = random.Random(P)
    c, book, err = _cache(4, 32 * P, P, 32, layers=1, H=1)
    n = [32 * (P // 3), 1, 32 * (P // 4) + 5, 0]
    for _ in range(3):
        want = book.extend(n, sum(n))
        got = ops.extend_pages(c, _ints(n), sum(n), err)
        assert got.rows.tolist() == want[1]
        ended = rng.randrange(3)
        book.free([ended])
        ops.free_pages(c, _ints([ended]), err=err)
        book.check(c, err)
        assert ops.compact_pages(c, err).tolist() == [book.compact()]
        book.check(c, err)


@pytest.mark.parametrize("S", [1, 63, 1023, 1024, 1025, 4096])
def test_many_sequences(S):
    rng = random.Random(S)
    c, book, err = _cache(S, 64, 2 * S + 3, 32, layers=1, H=1)
    for _ in range(2):
        counts = [rng.choice([0, 1, 17, 32]) for _ in range(S)]
        want = book.extend(counts, sum(counts))
        got = ops.extend_pages(c, _ints(counts), sum(counts), err)
        assert got.positions.tolist() == want[0] and got.rows.tolist() == want[1] and got.starts.tolist() == want[2]
        book.check(c, err)
    ended = rng.sample(range(S), S // 2) + [0, 0]
    book.free(ended)
    ops.free_pages(c, _ints(ended), err=err)
    book.check(c, err)
    pairs = list(zip([rng.randrange(S) for _ in range(S)], rng.sample(range(S), S)))
    book.fork(*zip(*pairs))
    ops.fork_pages(c, _ints([a for a, _ in pairs]), _ints([b for _, b in pairs]), err)
    book.check(c, err)


def test_a_chain_of_forks_in_one_call_copies_what_was_there():
    """b continues a and c continues b, which was empty when the call began."""
    c, book, err = _cache(4, 200, 12, 32)
    ops.extend_pages(c, _ints([70, 0, 0, 0]), 70, err)
    book.extend([70, 0, 0, 0], 70)
    ops.fork_pages(c, _ints([0, 1, 0]), _ints([1, 2, 3]), err)
    book.fork([0, 1, 0], [1, 2, 3])
    book.check(c, err)
    assert book.lengths == [70, 70, 0, 70] and book.err == 0


def test_rows_of_other_pages_stay():
    """A fork and a compaction write the pages that they name and no byte beside them."""
    c, book, err = _cache(3, 300, 14, 32, layers=3)
    counts = [100, 70, 0]
    book.extend(counts, 170)
    ops.extend_pages(c, _ints(counts), 170, err)
    book.free([0])
    ops.free_pages(c, _ints([0]), err=err)
    for call in ("fork", "compact"):
        k, v = c.k.clone(), c.v.clone()
        if call == "fork":
            book.fork([1], [2])
            ops.fork_pages(c, _ints([1]), _ints([2]), err)
        else:
            book.compact()
            ops.compact_pages(c, err)
        assert book.moves
        for t, was in ((c.k, k), (c.v, v)):
            for a, b in book.moves:
                was[:, :, :, b * 32:(b + 1) * 32] = was[:, :, :, a * 32:(a + 1) * 32]
            assert torch.equal(t, was)
        book.check(c, err)


def test_a_broken_table_is_flagged():
    """Pages that the pool does not have: nothing outside it is read or written (bounds are the kernels' own), and err says so."""
    c, book, err = _cache(3, 200, 8, 32)
    ops.extend_pages(c, _ints([70, 40, 0]), 110)
    c.table[0, 0], c.table[0, 2], c.table[1, 1] = 99, -5, 2**30
    for call in (lambda: ops.fork_pages(c, _ints([0]), _ints([2]), err), lambda: ops.compact_pages(c, err), lambda: ops.free_pages(c, _ints([0, 1, 2]), err=err)):
        err.zero_()
        call()
        assert int(err.item()) == 1


def test_captured_steps_take_pages():
    """A captured extension takes the next pages on each replay, as eager calls do."""
    c, book, err = _cache(3, 400, 30, 32)
    counts = _ints([1, 0, 40])
    ops.extend_pages(c, _ints([31, 5, 1]), 37, err)
    book.extend([31, 5, 1], 37)
    ops.extend_pages(c, _ints([0, 0, 0]), 0, err)  # warm-up
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.extend_pages(c, counts, 41, err)
    for _ in range(6):
        graph.replay()
        want = book.extend([1, 0, 40], 41)
        assert got.positions.tolist() == want[0] and got.rows.tolist() == want[1]
        book.check(c, err)


def test_going_back_inside_a_shared_page_is_refused():
    """Two sequences share a page; one of them cannot go back into it, alone or together with the other, but to its end it can."""
    c, book, err = _cache(3, 200, 12, 32)
    book.extend([70, 0, 5], 75)
    ops.extend_pages(c, _ints([70, 0, 5]), 75, err)
    book.fork([0], [1])
    ops.fork_pages(c, _ints([0]), _ints([1]), err)
    for at, left in (([0], [40]), ([0, 1], [40, 50]), ([0, 1], [40, 0]), ([0], [64]), ([0, 0, 2], [32, 0, 3]), ([0, 2], [20, 9])):
        book.err = 0
        err.zero_()
        book.free(at, left)
        ops.free_pages(c, _ints(at), _ints(left), err)
        book.check(c, err)


def test_pages_past_4_gb():
    """Rows whose offsets in a head pass 32 bits: taken, copied, read by every form of the attention and moved, as in a small pool."""
    T, H, D, small = 64, 2, 128, 40
    big = 2 ** 32 // (T * D * 2) + small  # pages; the last `small` lie past 4 GB
    a, b = ops.paged_cache(1, small, H, D, 4, 1024, DEV, T), ops.paged_cache(1, big, H, D, 4, 1024, DEV, T)
    far = big - small
    b.refs[:far] = 1
    for t, u in ((a.k, b.k), (a.v, b.v)):
        t.normal_()
        u[:, :, :, far * T:] = t
    err = torch.zeros(1, dtype=I32, device=DEV)
    g = torch.Generator().manual_seed(3)
    for counts in ([700, 33, 0, 0], [3, 1, 0, 0], [1, 150, 0, 0]):
        n = sum(counts)
        news = [ops.extend_pages(c, _ints(counts), n, err) for c in (a, b)]
        assert torch.equal(news[0].rows + far * T, news[1].rows) and torch.equal(news[0].positions, news[1].positions)
        q = torch.randn((1, n, 14, D), generator=g).to(torch.bfloat16).to(DEV).transpose(1, 2)
        for most in (1, 16, n):
            x, y = (ops.attention_paged(q, c, 0, w.starts, most=most, err=err) for c, w in zip((a, b), news))
            assert torch.equal(x, y)
    for c in (a, b):
        ops.fork_pages(c, _ints([0, 1]), _ints([2, 3]), err)
        ops.free_pages(c, _ints([0]), err=err)
    for t, u in ((a.k, b.k), (a.v, b.v)):
        assert torch.equal(t, u[:, :, :, far * T:])
    b.refs[:far] = 0  # from there to the front
    assert int(ops.compact_pages(b, err).item()) == int((a.refs > 0).sum()) and int(err.item()) == 0
    for s in (1, 2, 3):
        at = torch.arange(int(a.lengths[s]), device=DEV)
        rows = [c.table[s].long()[at // T] * T + at % T for c in (a, b)]
        assert int(rows[1].max()) < small * T
        for t, u in ((a.k, b.k), (a.v, b.v)):
            assert torch.equal(t[:, :, :, rows[0]], u[:, :, :, rows[1]])


def test_as_many_pairs_as_there_may_be():
    """4095 continuations of one sequence in a call, all 4096 ended in another."""
    S, T = 4096, 32
    c, b, err = _cache(S, 128, 4200, T, layers=1, H=1)
    held = Held(c, b)
    counts = [70] + [0] * (S - 1)
    new = ops.extend_pages(c, _ints(counts), 70, err)
    held.write(b.extend(counts, 70)[1], new.starts.tolist())
    ops.fork_pages(c, _ints([0] * (S - 1)), _ints(list(range(1, S))), err)
    b.fork([0] * (S - 1), list(range(1, S)))
    b.check(c, err)
    assert int(c.refs.max()) == S
    for s in (0, 1, 2047, 4095):
        i = b.rows(s).to(DEV)
        assert torch.equal(c.k[0, 0, 0, i], c.k[0, 0, 0, b.rows(0).to(DEV)]) and torch.equal(c.v[0, 0, 0, i], c.v[0, 0, 0, b.rows(0).to(DEV)])
    ends = list(range(S - 1, -1, -1))
    ops.free_pages(c, _ints(ends), err=err)
    b.free(ends)
    b.check(c, err)
    assert not c.refs.any()
    with pytest.raises(ValueError):
        ops.free_pages(c, _ints(list(range(S)) + [0]), err=err)
