"""ops.adjust_logits and ops.next_tokens against the definition's own steps in fp32 on the host: bit for bit."""

import pytest
import torch

from chunkkv_amd import _native, ops
from tests.paged_ref import adjusted

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def _tokens(g, b, n, vocab):
    t = (vocab * torch.rand((b, n), generator=g) ** 3).long().clamp_(max=vocab - 1)
    return torch.where(torch.rand((b, n), generator=g) < 0.1, torch.randint(-3, vocab + 3, (b, n), generator=g), t).to(DEV)


def _case(b, vocab, dtype, seed, prompt=0, generated=0, rows=True, bias=None, allowed=None):
    g = torch.Generator().manual_seed(seed)
    kw = {}
    if prompt:
        kw["prompt"] = _tokens(g, b, prompt, vocab)
    if generated:
        kw["generated"] = _tokens(g, b, generated, vocab)
    if rows:
        kw.update(repetition=(1 + torch.rand(b, generator=g)).to(DEV), frequency=torch.rand(b, generator=g).to(DEV), presence=torch.rand(b, generator=g).to(DEV))
    else:
        kw.update(repetition=1.25, frequency=0.375, presence=0.5)
    if bias is not None:
        kw["bias"] = torch.randn((vocab,) if bias == 1 else (b, vocab), generator=g).to(DEV)
    if allowed is not None:
        words = -(-vocab // 32)
        kw["allowed"] = torch.randint(-2**31, 2**31, (words,) if allowed == 1 else (b, words), generator=g).to(torch.int32).to(DEV)
    return (3 * torch.randn((b, vocab), generator=g)).to(dtype).to(DEV), kw


def _check(logits, kw):
    want = adjusted(logits, **kw)
    got = ops.adjust_logits(logits, **kw).cpu()
    assert torch.equal(torch.nan_to_num(got, nan=1.5), torch.nan_to_num(want, nan=1.5)) and torch.equal(got.isnan(), want.isnan())
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert ops.next_tokens(logits, err=err, **kw).tolist() == want.argmax(1).tolist()
    none = (want == -torch.inf).all(1).any()
    assert int(err.item()) == (_native.DEVICE_ERR_NO_TOKEN if none else 0)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("b,vocab", [(1, 1), (2, 7), (3, 31), (1, 32), (2, 33), (5, 512), (3, 4095), (1, 4096), (2, 4097), (1, 50001), (2, 152064)])
@pytest.mark.parametrize("prompt,generated,bias,allowed", [(0, 0, None, None), (5, 0, None, None), (0, 9, 1, None), (300, 77, 2, 2), (4100, 3000, None, 1)])
def test_matches_the_definition(dtype, b, vocab, prompt, generated, bias, allowed):
    _check(*_case(b, vocab, dtype, vocab + prompt, prompt, generated, b > 1, bias, allowed))


@pytest.mark.parametrize("n", [1, 2, 3, 1023, 1024, 1025, 4095, 4097, 8191, 8193, 20011])
def test_histories_of_all_lengths(n):
    """Every token counts once, also where a row starts at an odd one."""
    logits, kw = _case(3, 1000, BF, n, n, n)
    _check(logits, kw)
    long = _case(3, 1000, BF, n + 1, n + 3, n + 5)[1]
    _check(logits, dict(kw, prompt=long["prompt"][:, 1:n + 1], generated=long["generated"][:, 3:n + 3]))


def test_special_values():
    v = torch.tensor([float("nan"), float("inf"), -float("inf"), 0.0, -0.0, 1e-40, 3e38, -3e38, 1.0, -1.0])
    logits = v[torch.randint(0, 10, (6, 400), generator=torch.Generator().manual_seed(1))].to(DEV)
    for kw in (dict(), _case(6, 400, F32, 2, 300, 300)[1], _case(6, 400, F32, 3, 300, 300, allowed=2, bias=1)[1]):
        _check(logits, kw)
    for first, second in ((0.0, -0.0), (-0.0, 0.0), (float("nan"), float("inf")), (float("inf"), float("nan"))):
        row = torch.full((1, 5000), -1.0)
        row[0, 17], row[0, 4500] = first, second
        assert ops.next_tokens(row.to(DEV)).item() == row.argmax().item()


@pytest.mark.parametrize("vocab", [40, 9000])
def test_a_mask_that_leaves_nothing(vocab):
    logits = torch.randn((3, vocab), device=DEV).to(BF)
    logits[1] = float("nan")
    allowed = torch.stack([ops.token_bits([vocab - 1], vocab, DEV), ops.token_bits([], vocab, DEV), ops.token_bits(range(0, vocab, 7), vocab, DEV)])
    _check(logits, dict(allowed=allowed))
    assert ops.next_tokens(logits, allowed=allowed).tolist()[:2] == [vocab - 1, 0]


def test_ties_go_to_the_first():
    logits = torch.zeros((2, 20000), device=DEV)
    logits[0, [777, 5000, 19999]] = 2.0
    logits[1, [19999]] = 2.0
    assert ops.next_tokens(logits).tolist() == [777, 19999]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", [1001, 4104])
def test_strides_and_outputs(dtype, vocab):
    """Rows of a wider tensor, shared and strided biases, given outputs, float32 logits in place."""
    logits, kw = _case(4, vocab, dtype, 11, 40, 40, bias=2, allowed=2)
    wide = torch.zeros((4, vocab + 13), dtype=dtype, device=DEV)
    wide[:, 5:5 + vocab] = logits
    kw["bias"] = torch.cat([kw["bias"], kw["bias"]], 1)[:, 3:3 + vocab]
    _check(wide[:, 5:5 + vocab], kw)
    out = torch.full((4, vocab), 9.0, device=DEV)
    assert ops.adjust_logits(logits, out=out, **kw).data_ptr() == out.data_ptr() and torch.equal(out, ops.adjust_logits(logits, **kw))
    if dtype == F32:
        want = ops.adjust_logits(logits, **kw)
        assert torch.equal(ops.adjust_logits(logits, out=logits, **kw), want)
    token = torch.zeros(4, dtype=torch.int64, device=DEV)
    assert torch.equal(ops.next_tokens(wide[:, 5:5 + vocab], out=token, **kw), out.argmax(1)) and torch.equal(token, out.argmax(1))


def test_no_rows_and_empty_histories():
    empty = torch.zeros((0, 100), device=DEV)
    assert ops.adjust_logits(empty).shape == (0, 100) and ops.next_tokens(empty).shape == (0,)
    logits = torch.randn((2, 100), device=DEV)
    none = torch.zeros((2, 0), dtype=torch.int64, device=DEV)
    assert torch.equal(ops.adjust_logits(logits, prompt=none, generated=none, repetition=2.0), logits)


def test_graph_replays_follow_the_tokens():
    """A captured step: the token it chose is written behind the others, and the next replay counts it."""
    logits, kw = _case(3, 9001, BF, 5, 50, 0, allowed=1)
    seen = torch.full((3, 16), -1, dtype=torch.int64, device=DEV)
    at = torch.zeros((3, 1), dtype=torch.int64, device=DEV)
    kw = dict(kw, generated=seen, presence=4.0)

    def step():
        token = ops.next_tokens(logits, **kw)
        seen.scatter_(1, at, token[:, None])
        at.add_(1)

    def expect(held, n):
        for i in range(n):
            held[:, i] = adjusted(logits, **dict(kw, generated=held)).argmax(1)
        return held

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(5):
        graph.replay()
    want = expect(torch.full((3, 16), -1, dtype=torch.int64), 6)
    assert torch.equal(seen.cpu(), want)


def test_as_many_rows_as_there_may_be():
    """65535 rows, one more is refused; rows past 4 GB have the results that they have alone."""
    logits, kw = _case(3, 40, F32, 1, 5, 5)
    logits = logits[torch.arange(65535) % 3].contiguous()
    kw = {k: v[torch.arange(65535) % 3] if isinstance(v, torch.Tensor) and v.dim() and v.shape[0] == 3 else v for k, v in kw.items()}
    got, tokens = ops.adjust_logits(logits, **kw), ops.next_tokens(logits, **kw)
    assert torch.equal(got, got[:3][torch.arange(65535) % 3]) and torch.equal(tokens, got.argmax(1))
    more = torch.zeros((65536, 40), device=DEV)
    for call in (ops.adjust_logits, ops.next_tokens):
        with pytest.raises(ValueError):
            call(more)
    big = torch.zeros((16000, 152064), dtype=BF, device=DEV)
    big[-3:] = torch.randn((3, 152064), device=DEV).to(BF)
    history = torch.randint(0, 152064, (16000, 9), device=DEV)
    got = ops.adjust_logits(big, generated=history, repetition=1.5, frequency=0.25)
    want = ops.adjust_logits(big[-3:].clone(), generated=history[-3:], repetition=1.5, frequency=0.25)
    assert torch.equal(got[-3:], want)
    del got
    assert torch.equal(ops.next_tokens(big, generated=history, repetition=1.5, frequency=0.25)[-3:], want.argmax(1))
