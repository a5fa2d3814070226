"""HipEngine.paged where a call fails: the sequences are what they were, and the next call is right."""

import pytest
import torch

from chunkkv_amd import ops
from tests.test_gpu_paged_session import DEV, VOCAB, _close, _engine, _greedy_run, _session, _tokens

pytestmark = pytest.mark.gpu


class Stop(BaseException):
    """As an interrupt: no Exception."""


def _state(s):
    return s.free_pages, s.cache.lengths.tolist(), s.cache.refs.tolist(), {k: list(v) for k, v in s.tokens.items()}, sorted(s._logits), int(s._err.item())


def _fails_at(monkeypatch, name, call, error):
    """ops.<name> raises at its call-th call from now on, once."""
    real, calls = getattr(ops, name), []

    def broken(*args, **kw):
        calls.append(0)
        if len(calls) == call:
            raise error("broken")
        return real(*args, **kw)

    monkeypatch.setattr(ops, name, broken)


@pytest.mark.parametrize("error", [RuntimeError, Stop])
@pytest.mark.parametrize("name,call", [("rope_qkv", 1), ("attention_paged", 1), ("attention_paged", 3)])
def test_a_feed_that_fails_takes_nothing(monkeypatch, name, call, error):
    eng = _engine()
    s, (a, b), prompts = _session(eng, (70, 33))
    (c,) = s.fork(a)
    before = _state(s)
    chunks = {c: _tokens(41, 1), a: _tokens(1, 2), b: _tokens(170, 3)}
    with monkeypatch.context() as m:
        _fails_at(m, name, call, error)
        with pytest.raises(error):
            s.feed(chunks)
    assert _state(s) == before
    got = s.feed(chunks)
    for i, prompt in ((a, prompts[0]), (b, prompts[1]), (c, prompts[0])):
        _close(got[i][0], eng.prefill(prompt + chunks[i]).logits[-1])
        assert int(s.cache.lengths[i]) == len(prompt) + len(chunks[i])


@pytest.mark.parametrize("error", [RuntimeError, Stop])
def test_an_addition_that_fails_takes_nothing(monkeypatch, error):
    eng = _engine()
    s, (a,), _ = _session(eng, (40,))
    before, p = _state(s), _tokens(90, 4)
    result = eng.prefill(p)
    with monkeypatch.context() as m:
        _fails_at(m, "scatter_rows", 2, error)
        with pytest.raises(error):
            s.add(result, p)
    assert _state(s) == before
    q = _tokens(50, 5)
    assert s.add(eng.prefill(q), q) == 1 and int(s.cache.lengths[1]) == 50
    _greedy_run(eng, q, s.generate([1], 12)[0], 12)


def test_prefills_of_another_shape_are_refused_before_anything_is_done():
    eng = _engine()
    s, _, _ = _session(eng, (40,))
    before, p = _state(s), _tokens(90, 4)
    result = eng.prefill(p)

    def changed(**kw):
        r = eng.prefill(p)
        for name, (layer, value) in kw.items():
            getattr(r, name)[layer] = value
        return r

    K = result.keys[0]
    for bad in (_engine(4, 4).prefill(p), changed(keys=(1, K[:, :, :80])), changed(values=(2, K[:, :1])), changed(keys=(2, K.float())),
                changed(values=(0, K[..., :32])), changed(values=(1, K.cpu()))):
        with pytest.raises((ValueError, TypeError)):
            s.add(bad, p)
        assert _state(s) == before
    short = eng.prefill(p)
    short.values.pop()
    with pytest.raises(ValueError):
        s.add(short, p)
    assert _state(s) == before and s.add(result, p) == 1


def test_a_fork_that_fails_takes_nothing(monkeypatch):
    eng = _engine()
    s, (a,), (prompt,) = _session(eng, (70,))
    before = _state(s)
    with monkeypatch.context() as m:
        def interrupted():
            raise Stop("broken")

        m.setattr(s, "_check_err", interrupted)  # behind the device's part
        with pytest.raises(Stop):
            s.fork(a, 3)
    assert _state(s) == before
    b = s.fork(a)[0]
    _greedy_run(eng, prompt, s.generate([b], 9)[0], 9)


@pytest.mark.parametrize("then", ["feed", "add", "fork", "generate"])
def test_what_a_failed_call_flagged_is_not_the_next_ones(monkeypatch, then):
    """A mask leaves nothing, and before that is read something else fails."""
    eng = _engine()
    s, (a, b), prompts = _session(eng, (40, 65))
    before = _state(s)
    with monkeypatch.context() as m:
        _fails_at(m, "attention_paged", 2, RuntimeError)
        with pytest.raises(RuntimeError, match="broken"):
            s.generate([a, b], 9, allowed=ops.token_bits([], VOCAB, DEV))
    assert _state(s) == before
    chunk = _tokens(9, 5)
    if then == "feed":
        _close(s.feed({b: chunk})[b][0], eng.prefill(prompts[1] + chunk).logits[-1])
    elif then == "add":
        assert s.add(eng.prefill(chunk), chunk) == 2
        _greedy_run(eng, chunk, s.generate([2], 5)[0], 5)
    elif then == "fork":
        (c,) = s.fork(b)
        _greedy_run(eng, prompts[1], s.generate([c], 5)[0], 5)
    else:
        _greedy_run(eng, prompts[0], s.generate([a], 5)[0], 5)


def test_ending_sequences_reads_its_own_flags():
    eng = _engine()
    s, (a, b), prompts = _session(eng, (40, 65))
    s.cache.table[a, 1] = 10**6  # a broken book
    with pytest.raises(RuntimeError, match="reported an error"):
        s.free([a])
    assert list(s.tokens) == [b] and s.cache.lengths.tolist()[:2] == [0, 65] and int(s._err.item()) == 0
    _greedy_run(eng, prompts[1], s.generate([b], 5)[0], 5)


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("order", [(0, 1), (1, 0)])
def test_a_mask_that_leaves_an_ended_sequence_nothing(graphs, order):
    """The one sequence ends at its third token and its mask is empty from then on; the other's tokens are those it has where it is not."""
    eng = _engine()
    eng.decode_graphs = graphs
    some, end, none = (ops.token_bits(t, VOCAB, DEV) for t in (range(7, 100), [0], []))
    got = []
    for behind in (none, some):
        s, ids, _ = _session(eng, (20, 50))
        calls = []

        def allowed(outs):
            calls.append(0)
            return torch.stack([some if len(calls) < 3 else end if len(calls) == 3 else behind, some])

        got.append(s.generate([ids[i] for i in order], 9, allowed=allowed))
        assert len(got[-1][0]) == 2 and len(got[-1][1]) == 9 and len(calls) == 9
    assert got[0] == got[1] and all(7 <= t < 100 for tokens in got[0] for t in tokens)


def test_one_mask_for_all_may_become_one_each():
    eng = _engine()
    s, ids, _ = _session(eng, (20, 50))
    some, end = ops.token_bits(range(7, 100), VOCAB, DEV), ops.token_bits([0], VOCAB, DEV)

    def allowed(outs):
        return some if len(outs[1]) < 2 else torch.stack([end, some]) if len(outs[1]) == 2 else some[None]

    assert [len(t) for t in s.generate(ids, 6, allowed=allowed)] == [2, 6]


@pytest.mark.parametrize("graphs", [True, False])
def test_a_mask_that_leaves_nothing_ends_the_call_at_its_step(graphs):
    eng = _engine()
    eng.decode_graphs = graphs
    s, ids, prompts = _session(eng, (33, 50))
    before, asked = _state(s), []

    def allowed(outs):
        asked.append([list(o) for o in outs])
        return torch.stack([ops.token_bits(range(7, 100), VOCAB, DEV), ops.token_bits(range(7, 100) if len(asked) != 4 else [], VOCAB, DEV)])

    with pytest.raises(ValueError, match="mask"):
        s.generate(ids, 40, allowed=allowed)
    assert _state(s) == before and len(asked) == 4
    for p, tokens in zip(prompts, s.generate(ids, 8)):
        _greedy_run(eng, p, tokens, 8)


@pytest.mark.parametrize("error", [RuntimeError, Stop])
def test_a_generate_that_fails_behind_its_last_step_takes_nothing(monkeypatch, error):
    eng = _engine()
    s, ids, prompts = _session(eng, (33, 50))
    before = _state(s)
    with monkeypatch.context() as m:
        _fails_at(m, "free_pages", 1, error)  # going back to what was generated
        with pytest.raises(error):
            s.generate(ids, 8)
    assert _state(s) == before
    for p, tokens in zip(prompts, s.generate(ids, 8)):
        _greedy_run(eng, p, tokens, 8)


@pytest.mark.parametrize("where", ["before", "behind"])
def test_sequences_whose_end_fails_have_ended(monkeypatch, where):
    """On the device and on the host alike, so that the next sequence begins with no rows."""
    eng = _engine()
    s, (a, b), prompts = _session(eng, (40, 65))
    with monkeypatch.context() as m:
        if where == "before":
            _fails_at(m, "free_pages", 1, Stop)
        else:
            def interrupted():
                raise Stop("broken")

            m.setattr(s, "_check_err", interrupted)
        with pytest.raises(Stop):
            s.free([a])
    assert list(s.tokens) == [b] and s.cache.lengths.tolist()[:2] == [0, 65] and s.free_pages == 60 - 3
    p = _tokens(50, 5)
    assert s.add(eng.prefill(p), p) == a
    _greedy_run(eng, p, s.generate([a], 9)[0], 9)
    _greedy_run(eng, prompts[1], s.generate([b], 9)[0], 9)
