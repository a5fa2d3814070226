"""The 8-bit cache on the GPU: rows written (ops.quantize_rows) against a plain 64-bit form, code for code, and attention
over it (ops.attention_quantized) against a 64-bit softmax over the rows that codes and scales stand for."""

import numpy as np
import pytest
import torch

from chunkkv_amd import ops
from tests import decode_cache_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def _new(H, N, D, block, seed=0):
    """A cache of arbitrary bytes that are numbers."""
    g = torch.Generator().manual_seed(seed)
    c = ops.quantized_cache(H, N, D, DEV, block)
    for t in (c.k, c.v):
        t.view(torch.uint8).copy_(torch.randint(0, 127, t.shape, generator=g, dtype=torch.uint8))
    for t in (c.k_scale, c.v_scale):
        t.view(torch.uint8).copy_(torch.randint(110, 130, t.shape, generator=g, dtype=torch.uint8))
    return c


def _copy(c):
    return ops.QuantizedCache(c.k.clone(), c.v.clone(), c.k_scale.clone(), c.v_scale.clone(), c.block_tokens)


def _bytes(c):
    return [t.view(torch.uint8).cpu() for t in (c.k, c.v, c.k_scale, c.v_scale)]


def _rows(H, n, D, dtype, seed, spread=3.0):
    """Rows whose sizes differ by orders of magnitude, so that blocks get different scales."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((1, H, n, D), generator=g) * torch.exp(spread * torch.randn((1, H, n, 1), generator=g))
    return x.to(dtype).to(DEV)


def _want(c, k, v, start):
    """What the plain form makes of a cache: (values, exponents) of K and of V."""
    out = []
    for codes, scales, x in ((c.k, c.k_scale, k), (c.v, c.v_scale, v)):
        val = codes[0].cpu().to(torch.float64).numpy()
        exp = scales[0].view(torch.uint8).cpu().numpy().astype(np.int64) - 127
        for h in range(val.shape[0]):
            R.write_rows(val[h], exp[h], x[0, h].double().cpu().numpy(), start, c.block_tokens)
        out.append((val, exp))
    return out


def _check(c, want):
    for codes, scales, (val, exp) in zip((c.k, c.v), (c.k_scale, c.v_scale), want):
        assert np.array_equal(scales[0].view(torch.uint8).cpu().numpy().astype(np.int64) - 127, exp)
        assert np.array_equal(codes[0].cpu().to(torch.float64).numpy(), val)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("N,start,n", [(1, 0, 1), (128, 0, 128), (300, 0, 300), (301, 77, 1), (301, 64, 1), (301, 127, 130),
                                       (301, 37, 264), (260, 31, 2)])
def test_rows_match_the_plain_form(dtype, D, block, N, start, n):
    c = _new(3, N, D, block)
    if start:
        ops.quantize_rows(c, _rows(3, start, D, dtype, 1), _rows(3, start, D, dtype, 2))
    k, v = _rows(3, n, D, dtype, 3), _rows(3, n, D, dtype, 4)
    want = _want(c, k, v, start)
    ops.quantize_rows(c, k, v, start)
    _check(c, want)


def test_strided_rows_and_a_second_write_over_the_same_rows():
    """k/v as views of a projection's token-major output; writing them again changes nothing."""
    H, D, n = 2, 64, 150
    lin = _rows(1, n, 4 * H * D, BF, 5)[0, 0]
    k = lin[:, : H * D].view(1, n, H, D).transpose(1, 2)
    v = lin[:, H * D : 2 * H * D].view(1, n, H, D).transpose(1, 2)
    c = _new(H, 200, D, 32)
    want = _want(c, k, v, 0)
    ops.quantize_rows(c, k, v)
    _check(c, want)
    before = _bytes(c)
    ops.quantize_rows(c, k[:, :, 40:], v[:, :, 40:], 40)
    assert all(torch.equal(a, b) for a, b in zip(before, _bytes(c)))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_appended_one_by_one(dtype):
    """The scales of a cache written at once; values off by one subnormal step of the final scale at most."""
    H, D, n, block = 2, 64, 100, 32
    k, v = _rows(H, n, D, dtype, 6), _rows(H, n, D, dtype, 7)
    one, all_ = _new(H, n, D, block), _new(H, n, D, block)
    ops.quantize_rows(all_, k, v)
    for i in range(n):
        ops.quantize_rows(one, k[:, :, i : i + 1], v[:, :, i : i + 1], i)
    for a, b in ((one.k_scale, all_.k_scale), (one.v_scale, all_.v_scale)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for a, b in ((one.k, all_.k), (one.v, all_.v)):
        assert float((a.float() - b.float()).abs().max()) <= 2.0 ** -9


def test_extreme_and_nonfinite_rows():
    H, D, block = 1, 64, 32
    k = torch.zeros(1, H, 6 * block, D)
    k[0, 0, 32, 5] = 3e38
    k[0, 0, 33, 6] = -1e30  # far below its block's scale: zero
    k[0, 0, 64:96] = 1e-40  # subnormal
    k[0, 0, 100, 3] = float("nan")
    k[0, 0, 130, 0] = float("inf")
    k[0, 0, 160:, 0], k[0, 0, 160:, 1] = 448.0, 449.0  # one step past 448 * 2^0
    v = torch.ones_like(k)
    c = _new(H, 6 * block, D, block)
    ops.quantize_rows(c, k.to(DEV), v.to(DEV))
    got, s = c.k[0, 0].float().cpu(), c.k_scale[0, 0].view(torch.uint8).cpu().tolist()
    assert s == [1, 127 + R.scale_exponent(float(np.float32(3e38))), 1, 255, 255, 128]
    assert not got[:32].any() and got[32, 5] == 224 and got[33, 6] == 0  # 3e38 = 225.7 * 2^120
    assert got[96:160].isnan().all()
    assert (got[160:, 0] == 224).all() and (got[160:, 1] == 224).all()
    assert R.rows_of(c.v, c.v_scale, block).eq(1).all()
    # a NaN appended to a good block takes the block; a good row appended to a NaN block leaves it one
    nan = torch.full((1, H, 1, D), float("nan"), device=DEV)
    ops.quantize_rows(c, nan, nan, 40)
    assert c.k[0, 0, 32:41].float().isnan().all() and c.k_scale[0, 0, 1].view(torch.uint8) == 255
    ops.quantize_rows(c, torch.ones_like(nan), torch.ones_like(nan), 41)
    assert c.k[0, 0, 32:42].float().isnan().all() and not c.k[0, 0, 64:96].float().isnan().any()


def test_start_on_the_device_in_a_graph():
    """A captured append, replayed as decoding does it: the eager cache after every step."""
    H, D, block, n0, steps = 2, 128, 64, 90, 45
    k, v = _rows(H, n0 + steps, D, BF, 8), _rows(H, n0 + steps, D, BF, 9)
    c = _new(H, n0 + steps, D, block)
    ops.quantize_rows(c, k[:, :, :n0], v[:, :, :n0])
    eager = _copy(c)
    kb, vb = torch.zeros_like(k[:, :, :1]), torch.zeros_like(v[:, :, :1])
    at, err = torch.tensor([n0], device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    kb.copy_(k[:, :, n0 : n0 + 1])
    vb.copy_(v[:, :, n0 : n0 + 1])
    ops.quantize_rows(_copy(c), kb, vb, at, err)  # warm-up, on another cache
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.quantize_rows(c, kb, vb, at, err)
        at.add_(1)
    for i in range(n0, n0 + steps):
        kb.copy_(k[:, :, i : i + 1])
        vb.copy_(v[:, :, i : i + 1])
        graph.replay()
        ops.quantize_rows(eager, k[:, :, i : i + 1], v[:, :, i : i + 1], i)
        if i % 11 == 0:
            assert all(torch.equal(a, b) for a, b in zip(_bytes(c), _bytes(eager)))
    assert all(torch.equal(a, b) for a, b in zip(_bytes(c), _bytes(eager))) and int(err) == 0
    before = _bytes(c)
    for bad in (n0 + steps, -1, 2**40):  # one row past the cache, and far outside it
        err.zero_()
        ops.quantize_rows(c, kb, vb, torch.tensor([bad], device=DEV), err)
        assert int(err) == 1
        assert all(torch.equal(a, b) for a, b in zip(before, _bytes(c)))


@pytest.mark.parametrize("start,n", [(0, 65), (63, 66), (1, 128)])
def test_start_on_the_device_over_several_blocks(start, n):
    c = _new(2, 200, 64, 64)
    ops.quantize_rows(c, _rows(2, 64, 64, BF, 1), _rows(2, 64, 64, BF, 2))
    k, v = _rows(2, n, 64, BF, 3), _rows(2, n, 64, BF, 4)
    want = _want(c, k, v, start)
    ops.quantize_rows(c, k, v, torch.tensor([start], device=DEV))
    _check(c, want)


def _filled(H, N, D, block, rows, seed, nan_behind=True):
    """A cache whose first `rows` rows are written; behind them NaN codes, and NaN scales of whole blocks."""
    c = ops.quantized_cache(H, N, D, DEV, block)
    for t in (c.k, c.v, c.k_scale, c.v_scale):
        t.view(torch.uint8).fill_((0x7F if t.dtype == torch.float8_e4m3fn else 255) if nan_behind else 0)
    g = torch.Generator().manual_seed(seed)
    k = torch.randn((1, H, rows, D), generator=g) * 1.5
    v = torch.randn((1, H, rows, D), generator=g) * torch.exp(torch.randn((1, H, rows, 1), generator=g))
    ops.quantize_rows(c, k.to(BF).to(DEV), v.to(BF).to(DEV))
    return c


def _q(Hq, n, D, seed, token_major=True):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn((1, n, Hq, D), generator=g).to(BF).to(DEV).transpose(1, 2)
    return q if token_major else q.contiguous()


def _attends(q, c, pos, rows, scale=None, **kw):
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = ops.attention_quantized(q, c, pos.to(DEV), scale, err=err, **kw)
    torch.cuda.synchronize()
    assert int(err) == 0
    K, V = (R.rows_of(t, s, c.block_tokens)[:, :, :rows] for t, s in ((c.k, c.k_scale), (c.v, c.v_scale)))
    want, most = R.attention(q, K, V, pos, q.shape[3] ** -0.5 if scale is None else scale)
    off = (out[0].double().cpu() - want).abs()
    assert (off <= most).all(), f"{float((off / most).max())} times the bound"
    return out


@pytest.mark.parametrize(
    "Hq,Hkv,D,N,rows,n,block",
    [
        (28, 4, 128, 40, 1, 1, 32),  # one cached row
        (28, 4, 128, 513, 450, 1, 64),  # a decoded token, the cache longer than its rows
        (28, 4, 128, 8256, 8200, 1, 64),  # split over the cache
        (14, 2, 64, 8192, 8192, 1, 128),
        (28, 4, 128, 2100, 2077, 5, 32),  # a few tokens at once
        (8, 8, 64, 333, 333, 333, 64),  # no shared heads, causal, ragged
        (14, 2, 64, 1103, 1103, 251, 32),
        (28, 4, 128, 1500, 1500, 1500, 64),  # 128-query workgroups: the cache read as bf16
        (28, 4, 128, 8256, 8250, 130, 128),  # a head's (token, query head) rows, in splits of the cache
        (28, 4, 128, 6001, 5985, 500, 32),
        (28, 4, 128, 6001, 5985, 501, 32),
        (14, 2, 64, 16390, 16385, 65, 64),
        (16, 16, 64, 5700, 5633, 130, 128),  # 128-query workgroups in splits, the codes converted by each
        (32, 32, 128, 1100, 1090, 1000, 32),  # no shared heads: the codes converted, unsplit
        (64, 64, 64, 1000, 993, 910, 64),
        (28, 4, 128, 8256, 8250, 33, 64),  # a head's (token, query head) rows in one block after another: two blocks
        (28, 4, 128, 8300, 8290, 251, 32),  # fourteen, and one of no rows
        (28, 4, 128, 4000, 3990, 160, 32),
        (16, 16, 64, 8300, 8258, 300, 32),  # no shared heads
        (8, 8, 128, 10500, 10433, 130, 64),
        (14, 2, 64, 4100, 4033, 251, 64),
        (32, 8, 128, 9000, 8999, 100, 128),
        (14, 2, 64, 16390, 16385, 40, 32),
        (14, 2, 64, 9000, 8901, 700, 64),
        (10, 2, 128, 12000, 11000, 66, 64),
        (6, 3, 64, 33000, 32990, 65, 128),
        (28, 4, 128, 1100, 1024, 1, 32),  # one token, whole and split
        (28, 4, 128, 1025, 1025, 1, 32),
        (14, 2, 64, 1536, 1536, 2, 64),
        (14, 2, 64, 1600, 1537, 1, 128),
        (6, 3, 64, 130, 129, 100, 32),  # heads that do not divide 8
        (64, 1, 128, 700, 700, 3, 64),  # a group of 64
    ],
)
@pytest.mark.parametrize("split", [True, False])
def test_attention_matches_the_plain_form(Hq, Hkv, D, N, rows, n, block, split):
    c = _filled(Hkv, N, D, block, rows, N + n)
    g = torch.Generator().manual_seed(n)
    pos = torch.randperm(rows, generator=g)[:n].sort().values
    pos[-1] = rows - 1
    _attends(_q(Hq, n, D, rows, token_major=n % 2 == 0), c, pos, rows, split=split)


@pytest.mark.parametrize("Hq,Hkv,D,N,n", [(28, 4, 128, 8256, 60), (14, 2, 64, 16390, 40), (28, 4, 128, 8256, 1), (28, 4, 128, 6000, 500)])
def test_a_workspace_may_hold_anything(Hq, Hkv, D, N, n):
    """The allocator hands out memory full of NaN; positions from the first row to the last, the first half near the front."""
    c = _filled(Hkv, N, D, 64, N, n)
    pos = torch.cat([torch.arange(n // 2), torch.arange(N - (n - n // 2), N)])
    q = _q(Hq, n, D, 7)
    for mb in (4, 32, 128):
        torch.full((mb << 18,), float("nan"), device=DEV)
    _attends(q, c, pos, N)


def test_attention_of_unsorted_and_repeated_positions_and_another_scale():
    c = _filled(2, 300, 64, 32, 300, 3)
    pos = torch.tensor([299, 0, 5, 5, 120, 64, 31, 32, 33, 0])
    _attends(_q(14, 10, 64, 4), c, pos, 300, scale=0.31)
    c = _filled(2, 16500, 64, 32, 16500, 3)  # over a long cache, blocks of rows in any order
    pos = torch.randint(0, 16500, (60,), generator=torch.Generator().manual_seed(1))
    _attends(_q(14, 60, 64, 4), c, pos, 16500, scale=0.31)


def test_positions_outside_over_a_long_cache():
    c = _filled(4, 8400, 128, 64, 8400, 3)
    q, err = _q(28, 60, 128, 5), torch.zeros(1, dtype=torch.int32, device=DEV)
    pos = torch.arange(8340, 8400, device=DEV)
    wild = pos.clone()
    wild[3], pos[3], wild[59] = -7, 0, 2**40
    got = ops.attention_quantized(q, c, wild, err=err)
    assert int(err) == 1
    assert torch.equal(got, ops.attention_quantized(q, c, pos))


def test_attention_clamps_and_flags_positions_outside():
    c = _filled(2, 100, 64, 32, 100, 3)
    q, err = _q(4, 3, 64, 5), torch.zeros(1, dtype=torch.int32, device=DEV)
    got = ops.attention_quantized(q, c, torch.tensor([-3, 50, 10**12], device=DEV), err=err)
    assert int(err) == 1
    assert torch.equal(got, ops.attention_quantized(q, c, torch.tensor([0, 50, 99], device=DEV)))


def test_attention_of_no_queries():
    c = _filled(2, 100, 64, 32, 100, 3)
    assert ops.attention_quantized(_q(4, 0, 64, 5), c, torch.zeros(0, dtype=torch.int64, device=DEV)).shape == (1, 0, 4, 64)


def test_a_nan_block_reaches_only_calls_that_see_it():
    """Rows up to a call's largest position are finite by contract; a NaN block past it is not met."""
    c = _filled(1, 128, 64, 32, 128, 3)
    bad = torch.full((1, 1, 1, 64), float("nan"), device=DEV)
    ops.quantize_rows(c, bad, bad, 127)  # block 3: rows 96..127
    q = _q(2, 2, 64, 5)
    at = lambda i, p: ops.attention_quantized(q[:, :, i : i + 1], c, torch.tensor([p], device=DEV)).float()  # noqa: E731
    assert torch.isfinite(at(0, 95)).all() and at(1, 96).isnan().all()


def test_decode_graph_replays_match_eager():
    """Append and attention as one captured step, 6 replays with eager work between them."""
    H, Hq, D, block, n0, steps = 2, 14, 64, 32, 1000, 6
    k, v = _rows(H, n0 + steps, D, BF, 8, 0.3), _rows(H, n0 + steps, D, BF, 9, 0.3)
    q = _q(Hq, n0 + steps, D, 10)
    c = ops.quantized_cache(H, n0 + 64, D, DEV, block)
    ops.quantize_rows(c, k[:, :, :n0], v[:, :, :n0])
    eager = _copy(c)
    kb, vb, qb = (torch.empty_like(t[:, :, :1]) for t in (k, v, q))
    at = torch.tensor([n0], device=DEV)

    def step():
        ops.quantize_rows(c, kb, vb, at)
        o = ops.attention_quantized(qb, c, at)
        at.add_(1)
        return o

    for t, s in ((kb, k), (vb, v), (qb, q)):
        t.copy_(s[:, :, n0 : n0 + 1])
    step()
    at.fill_(n0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(n0, n0 + steps):
        for t, s in ((kb, k), (vb, v), (qb, q)):
            t.copy_(s[:, :, i : i + 1])
        graph.replay()
        ops.quantize_rows(eager, k[:, :, i : i + 1], v[:, :, i : i + 1], i)
        want = ops.attention_quantized(q[:, :, i : i + 1], eager, torch.tensor([i], device=DEV))
        assert torch.equal(out, want)


@pytest.mark.parametrize("Hq,Hkv,D,N,n", [(28, 4, 128, 8256, 60), (14, 2, 64, 1103, 251), (28, 4, 128, 1500, 1500)])
def test_prompt_graph_replays_match_eager(Hq, Hkv, D, N, n):
    """Two graphs of one call each, replayed in turn with eager calls between, positions and queries changed every time."""
    c, bufs, graphs, outs = _filled(Hkv, N, D, 32, N, 5), [], [], []
    for i in range(2):
        bufs.append((_q(Hq, n, D, i), torch.arange(N - n, N, device=DEV)))
        ops.attention_quantized(bufs[i][0], c, bufs[i][1])
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(ops.attention_quantized(bufs[i][0], c, bufs[i][1]))
    for step in range(6):
        i = step % 2
        bufs[i][0].copy_(_q(Hq, n, D, 10 + step))
        bufs[i][1].copy_(torch.randint(0, N, (n,), generator=torch.Generator().manual_seed(step)).sort().values)
        graphs[i].replay()
        assert torch.equal(outs[i], ops.attention_quantized(bufs[i][0], c, bufs[i][1]))


def test_calls_on_two_streams_at_once():
    cs = [_filled(4, 3000, 128, 64, 3000, s) for s in (1, 2)]
    qs = [_q(28, n, 128, n) for n in (1, 200)]
    ps = [torch.tensor([2999], device=DEV), torch.arange(2800, 3000, device=DEV)]
    want = [ops.attention_quantized(q, c, p) for q, c, p in zip(qs, cs, ps)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.attention_quantized(qs[i], cs[i], ps[i]))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)


def test_offsets_past_32_bits():
    """40 million rows (5.1 GB of codes): all weight on the last row, whose values come back."""
    N, D = 40_000_001, 128
    c = ops.quantized_cache(1, N, D, DEV, 128)
    for t in (c.k, c.v):
        t.view(torch.uint8).zero_()
    for t in (c.k_scale, c.v_scale):
        t.view(torch.uint8).fill_(127)
    k, v = torch.full((1, 1, 1, D), 8.0, dtype=BF, device=DEV), _rows(1, 1, D, BF, 3, 0.0)
    ops.quantize_rows(c, k, v, N - 1)
    q = torch.full((1, 2, 1, D), 2.0, dtype=BF, device=DEV)  # score 16 * 128 / sqrt(128) = 181
    out = ops.attention_quantized(q, c, torch.tensor([N - 1], device=DEV))
    want = (c.v[0, 0, N - 1].float() * c.v_scale[0, 0, -1].float()).to(BF)
    assert torch.equal(out[0, 0, 0], want) and torch.equal(out[0, 0, 1], want)
    near = ops.attention_quantized(q, c, torch.tensor([1000], device=DEV))
    assert not near.any()


def test_refusals():
    c, q = _filled(2, 100, 64, 32, 100, 3), _q(4, 2, 64, 5)
    pos = torch.tensor([0, 1], device=DEV)
    k = torch.zeros((1, 2, 4, 64), dtype=BF, device=DEV)
    for bad in (dict(start=97), dict(start=-1), dict(start=torch.tensor([1, 2], device=DEV)), dict(start=torch.tensor([1])),
                dict(start=torch.tensor([1.0], device=DEV)), dict(k=k[:, :1]), dict(k=k[..., :32]), dict(k=k.cpu()),
                dict(err=torch.zeros(1, device=DEV)), dict(err=torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(ValueError):
            ops.quantize_rows(c, bad.get("k", k), k, bad.get("start", 0), bad.get("err"))
    with pytest.raises(TypeError):
        ops.quantize_rows(c, k.to(torch.float16), k.to(torch.float16))
    with pytest.raises(TypeError):
        ops.quantize_rows(c, k, k.float())
    with pytest.raises(ValueError):
        ops.quantize_rows(ops.quantized_cache(2, 2, 64, DEV, 32), k, k)
    with pytest.raises(ValueError):
        ops.quantized_cache(2, 100, 64, DEV, 48)
    wrong = [ops.QuantizedCache(c.k, c.v, c.k_scale, c.v_scale, 64), ops.QuantizedCache(c.k[:, :, ::2], c.v[:, :, ::2], c.k_scale, c.v_scale, 32),
             ops.QuantizedCache(c.k, c.v[:, :1], c.k_scale, c.v_scale, 32), ops.QuantizedCache(c.k, c.v, c.k_scale, c.v_scale, 16)]
    for w in wrong:
        with pytest.raises(ValueError):
            ops.attention_quantized(q, w, pos)
    with pytest.raises(TypeError):
        ops.attention_quantized(q, ops.QuantizedCache(c.k.view(torch.uint8), c.v, c.k_scale, c.v_scale, 32), pos)
    with pytest.raises(TypeError):
        ops.attention_quantized(q.float(), c, pos)
    for args in ((q[..., :32], c, pos), (q[:, :3], c, pos), (q, c, pos[:1]), (q, c, pos.int()), (q, c, pos.cpu()), (q, c, pos, -1.0),
                 (q, c, pos, float("nan")), (torch.cat([q, q]), c, pos)):
        with pytest.raises(ValueError):
            ops.attention_quantized(*args)
    with pytest.raises(ValueError):
        ops.attention_quantized(q, c, pos, out=torch.empty((1, 2, 4, 64), device=DEV))
