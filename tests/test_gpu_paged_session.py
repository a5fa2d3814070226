"""The paged cache's operators together, as HipEngine.paged uses them: prefills added, forked, fed, decoded in one batch, ended,
their pages moved; against the engine's own prefill and generate of each sequence alone."""

import numpy as np
import pytest
import torch

from chunkkv_amd import ops
from chunkkv_amd.engine import HipEngine
from tests.helpers import StubTokenizer, tiny_qwen2
from tests.paged_ref import adjusted

pytestmark = pytest.mark.gpu
DEV = "cuda"
VOCAB = 512


def _engine(heads=8, kv=2, seed=6, **kw):
    gpu = tiny_qwen2(layers=3, hidden=512, heads=heads, kv=kv, inter=1024, vocab=VOCAB, seed=seed, dtype=torch.bfloat16).to(DEV)
    with torch.no_grad():
        gpu.model.norm.weight.mul_(20.0)  # greedy picks are not near-ties
    return HipEngine(gpu, StubTokenizer(), **kw)


def _tokens(n, seed=6):
    return np.random.default_rng(seed).integers(1, 511, n).tolist()


def _session(eng, lengths, **kw):
    kw = dict(dict(n_pages=60, n_sequences=8, max_tokens=700, page_tokens=32), **kw)
    s = eng.paged(**kw)
    prompts = [_tokens(n, 100 + i) for i, n in enumerate(lengths)]
    return s, [s.add(eng.prefill(p), p) for p in prompts], prompts


def _close(a, b):
    """Two forms of one attention in three bf16 layers: 3 2^-8 apart in each (its weights' and result's roundings), and 4 roundings behind it."""
    a, b = a.double().cpu(), b.double().cpu()
    assert (a - b).norm() <= 3 * 7 * 2.0 ** -8 * b.norm(), ((a - b).norm() / b.norm()).item()


def _greedy(logits, token):
    """Whether another form of the same attention may choose this token: logits are bf16 and tie (two of 55.5 among these models'), and two forms are
    3 7 2^-8 = 0.082 of the logits' norm apart (_close). The difference is spread over hundreds of dimensions, so one logit is off by 0.082 of
    their deviation, a difference of two by sqrt(2) of that: four times it, 0.46, and the logits' own roundings, 2 2^-8 of at most four deviations."""
    x = logits.float()
    assert x.amax() - x[token] <= 0.5 * x[x.isfinite()].std(), ((x.amax() - x[token]) / x[x.isfinite()].std()).item()


def _greedy_run(eng, prompt, tokens, most):
    """Whether tokens, and the end behind them if they are fewer than most, are greedy choices after prompt."""
    x = eng.prefill(prompt + tokens, logits_from=len(prompt) - 1).logits
    for i, t in enumerate(tokens):
        assert t not in eng.eos
        _greedy(x[i], t)
    if len(tokens) < most:
        _greedy(x[len(tokens)], max((t for t in eng.eos if t is not None), key=lambda t: x[len(tokens), t].item()))


@pytest.mark.parametrize("heads,kv", [(8, 2), (4, 4)])  # head_dim 64 and 128
@pytest.mark.parametrize("graphs", [True, False])
def test_sequences_decoded_together_are_those_decoded_alone(heads, kv, graphs):
    eng = _engine(heads, kv)
    eng.decode_graphs = graphs
    s, ids, prompts = _session(eng, (5, 200, 64, 31))
    assert ids == [0, 1, 2, 3]
    got = s.generate([2, 0, 3, 1], 40)
    for i, tokens in zip([2, 0, 3, 1], got):
        _greedy_run(eng, prompts[i], tokens, 40)
        assert s.tokens[i] == prompts[i] + tokens and int(s.cache.lengths[i]) == len(s.tokens[i])
    # and they go on from there
    on = [i for i in range(4) if i in s._logits]
    assert on
    for i, tokens in zip(on, s.generate(on, 9)):
        _greedy_run(eng, s.tokens[i][:len(s.tokens[i]) - len(tokens)], tokens, 9)


def test_forks_fed_with_questions_match_prefills():
    eng = _engine()
    s, (a,), (prompt,) = _session(eng, (150,))
    b, c = s.fork(a, 2)
    assert 60 - s.free_pages == 5 + 2  # four pages shared, the fifth copied for each
    chunks = {c: _tokens(41, 1), a: _tokens(1, 2), b: _tokens(170, 3)}
    got = s.feed(chunks)
    for i, chunk in chunks.items():
        _close(got[i][0], eng.prefill(prompt + chunk).logits[-1])
        assert s.tokens[i] == prompt + chunk
    assert int(s.cache.lengths[b]) == 320
    # a second chunk each, over pages of their own and shared ones
    again = {a: _tokens(33, 4), b: _tokens(2, 5), c: _tokens(90, 6)}
    got = s.feed(again)
    for i, chunk in again.items():
        _close(got[i][0], eng.prefill(prompt + chunks[i] + chunk).logits[-1])


def test_freed_and_compacted_pages_change_no_token():
    eng = _engine()
    got = []
    for moved in (False, True):
        s, ids, prompts = _session(eng, (100, 37, 250, 64, 90))
        s.generate([4, 2], 5)
        if moved:
            s.free([0, 3])
            used = s.compact()
            assert used == 60 - s.free_pages and int((s.cache.refs[:used] > 0).sum()) == used
        chunks = s.feed({1: _tokens(40, 1), 2: _tokens(3, 2), 4: _tokens(1, 3)})
        got.append((s.generate([1, 4, 2], 20), [chunks[i] for i in (1, 2, 4)]))
    assert got[0][0] == got[1][0] and all(torch.equal(a, b) for a, b in zip(got[0][1], got[1][1]))
    p = _tokens(77, 9)
    assert s.add(eng.prefill(p), p) == 0  # the lowest free number
    _greedy_run(eng, p, s.generate([0], 12)[0], 12)


@pytest.mark.parametrize("graphs", [True, False])
def test_penalties_and_masks_are_the_operators(graphs):
    """Each token is one of the largest of the adjusted logits, computed on the host, of the sequence fed token by token."""
    eng = _engine()
    eng.decode_graphs = graphs
    s, ids, prompts = _session(eng, (40, 65, 9))
    kw = dict(repetition=torch.tensor([1.3, 1.0, 2.0], device=DEV), frequency=0.5, presence=torch.tensor([0.0, 3.0, 8.0], device=DEV),
              bias=torch.randn(VOCAB, generator=torch.Generator().manual_seed(1)).to(DEV),
              allowed=torch.stack([ops.token_bits(range(k, VOCAB, 3), VOCAB, DEV) for k in (1, 2, 4)]))
    got = s.generate(ids, 12, **kw)
    for i, p in enumerate(prompts):
        other = eng.paged(n_pages=10, n_sequences=1, max_tokens=100, page_tokens=64)
        other.add(eng.prefill(p), p)
        one = {k: v[i:i + 1] if isinstance(v, torch.Tensor) and v.shape[0] == 3 else v for k, v in kw.items()}
        logits, tokens = other._logits[0], []
        for _ in range(12):
            x = adjusted(logits, torch.tensor([p]), torch.tensor([tokens], dtype=torch.int64).view(1, -1), **one)
            t = got[i][len(tokens)]
            _greedy(x[0], t)
            tokens.append(t)
            logits = other.feed({0: [t]})[0]
        assert all(t % 3 == (1, 2, 1)[i] for t in tokens) and len(got[i]) == 12  # the end is not allowed


def test_a_grammar_that_follows_the_tokens():
    """allowed as a function: the third token of the one sequence is the end, the other goes on; the ended one can be fed again."""
    eng = _engine()
    s, ids, prompts = _session(eng, (20, 50))
    calls = []

    def allowed(outs):
        calls.append([list(o) for o in outs])
        end = ops.token_bits([0], VOCAB, DEV)
        some = ops.token_bits(range(7, 100), VOCAB, DEV)
        return torch.stack([end if len(outs[0]) == 2 else some, some])

    got = s.generate([1, 0], 6, allowed=allowed)
    assert [len(t) for t in got] == [2, 6] and all(7 <= t < 100 for row in got for t in row)
    assert calls[0] == [[], []] and calls[2] == [got[0], got[1][:2]] and len(calls) == 6
    assert int(s.cache.lengths[1]) == 52 and int(s.cache.lengths[0]) == 26
    with pytest.raises(ValueError, match="feed it tokens"):
        s.generate([1], 3)
    chunk = _tokens(30, 8)
    _close(s.feed({1: chunk})[1][0], eng.prefill(prompts[1] + got[0] + chunk).logits[-1])
    assert len(s.generate([1], 4)[0]) <= 4


def test_a_mask_that_leaves_nothing_raises_and_takes_nothing():
    eng = _engine()
    s, ids, prompts = _session(eng, (33, 50))
    free = s.free_pages
    for bad in (ops.token_bits([], VOCAB, DEV), lambda outs: ops.token_bits(range(9) if len(outs[0]) < 4 else [], VOCAB, DEV)):
        with pytest.raises(ValueError, match="mask"):
            s.generate(ids, 40, allowed=bad, bias=-10.0 * torch.nn.functional.one_hot(torch.tensor(0), VOCAB).float().to(DEV))
        assert s.free_pages == free and s.cache.lengths.tolist()[:2] == [33, 50] and s.tokens[0] == prompts[0]

    def broken(outs):
        if len(outs[0]) == 3:
            raise KeyError("x")
        return ops.token_bits(range(1, VOCAB), VOCAB, DEV)

    with pytest.raises(KeyError):
        s.generate(ids, 40, allowed=broken)
    assert s.free_pages == free
    for p, tokens in zip(prompts, s.generate(ids, 15)):
        _greedy_run(eng, p, tokens, 15)


def test_what_does_not_fit_is_refused_before_anything_is_done():
    eng = _engine()
    s, ids, prompts = _session(eng, (100, 60), n_pages=8, n_sequences=3, max_tokens=224)
    free, lengths = s.free_pages, s.cache.lengths.tolist()
    p = _tokens(90)
    result = eng.prefill(p)
    for call, what in ((lambda: s.add(result, p), "pages"), (lambda: s.add(result, p[:-1]), "tokens"), (lambda: s.feed({0: _tokens(130)}), "rows"),
                       (lambda: s.feed({0: _tokens(70), 1: _tokens(30)}), "pages"), (lambda: s.feed({2: [1]}), "no sequence"), (lambda: s.feed({0: []}), "token"),
                       (lambda: s.feed({0: [VOCAB]}), "vocabulary"), (lambda: s.fork(0, 2), "sequences"), (lambda: s.generate([0, 0], 3), "twice"),
                       (lambda: s.generate([0, 1], 70), "pages"), (lambda: s.free([2]), "no sequence")):
        with pytest.raises(ValueError, match=what):
            call()
        assert s.free_pages == free and s.cache.lengths.tolist() == lengths
    for p, tokens in zip(prompts, s.generate([0, 1], 10)):
        _greedy_run(eng, p, tokens, 10)
    assert s.generate([], 5) == [] and s.generate([0], 0) == [[]] and s.feed({}) == {}


def test_a_number_of_forks_below_zero_is_refused():
    eng = _engine()
    s, _, _ = _session(eng, (40,))
    with pytest.raises(ValueError, match="0 or more"):
        s.fork(0, -1)
    assert s.fork(0, 0) == [] and list(s.tokens) == [0] and s.free_pages == 58


def test_a_prefill_of_many_logits_is_not_kept():
    eng = _engine()
    s = eng.paged(n_pages=8, n_sequences=2, max_tokens=64, page_tokens=32)
    p = _tokens(40)
    result = eng.prefill(p, logits_from=0)
    s.add(result, p)
    assert s._logits[0].untyped_storage().nbytes() == VOCAB * result.logits.element_size() < result.logits.untyped_storage().nbytes()


def test_the_library_attention_of_prefills_may_fill_the_cache():
    eng = _engine(attention="sdpa")
    s, ids, prompts = _session(eng, (40, 129))
    for p, tokens in zip(prompts, s.generate(ids, 12)):
        _greedy_run(eng, p, tokens, 12)


def test_models_without_the_kernel_are_refused():
    eng = _engine(attention="reference")
    with pytest.raises(ValueError, match="bf16"):
        eng.paged(4, 1, 64)
