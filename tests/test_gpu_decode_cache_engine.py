"""The decode cache's operators together, as a program uses them: prefill with observed weights, caches cut, held in 8 bits, and
decoded over with appended rows; each against the same steps in plain 64-bit form."""

import numpy as np
import pytest
import torch

from chunkkv_amd import ops
from chunkkv_amd.engine import HipEngine
from chunkkv_amd.types import BlendConfig, Placement
from tests import decode_cache_ref as R
from tests.helpers import StubTokenizer, tiny_qwen2

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _engine(heads=8, kv=2, seed=6, **kw):
    gpu = tiny_qwen2(layers=3, hidden=512, heads=heads, kv=kv, inter=1024, vocab=512, seed=seed, dtype=torch.bfloat16).to(DEV)
    with torch.no_grad():
        gpu.model.norm.weight.mul_(20.0)  # greedy picks are not near-ties
    return HipEngine(gpu, StubTokenizer(), **kw)


def _tokens(n, seed=6):
    return np.random.default_rng(seed).integers(1, 511, n).tolist()


class _PlainCache:
    """One layer's decode cache in plain form: bf16 rows, or 8-bit ones."""

    def __init__(self, K, V, bits):
        self.bits, self.rows = bits, K.shape[2]
        self.kv = [t.cpu() for t in (K, V)]
        if bits == 8:
            self.val = [np.zeros((K.shape[1], self.rows + 64, K.shape[3])) for _ in range(2)]
            self.exp = [np.zeros((K.shape[1], -(-(self.rows + 64) // 64)), dtype=np.int64) for _ in range(2)]
            self._write(self.kv, 0)

    def _write(self, kv, start):
        for val, exp, t in zip(self.val, self.exp, kv):
            for h in range(val.shape[0]):
                R.write_rows(val[h], exp[h], t[0, h].double().numpy(), start, 64)

    def append(self, k, v):
        if self.bits == 8:
            self._write([k.cpu(), v.cpu()], self.rows)
        else:
            self.kv = [torch.cat([t, x.cpu()], 2) for t, x in zip(self.kv, (k, v))]
        self.rows += 1

    def tensors(self):
        if self.bits == 16:
            return self.kv
        at = np.arange(self.rows) // 64
        return [torch.from_numpy(val[:, : self.rows] * np.ldexp(1.0, exp[:, at])[..., None])[None] for val, exp in zip(self.val, self.exp)]


@torch.inference_mode()
def _plain_generate(eng, res, max_tokens, bits, keep, sink, recent):
    caches = []
    for K, V, w in zip(res.keys, res.values, res.weights or [None] * len(res.keys)):
        if keep is not None and keep < K.shape[2]:
            at = torch.tensor([R.kept_rows(w[0, h].cpu().numpy(), keep, sink, recent) for h in range(K.shape[1])], device=DEV)
            K, V = (torch.stack([t[0, h][at[h]] for h in range(t.shape[1])])[None] for t in (K, V))
        caches.append(_PlainCache(K, V, bits))
    pos, out, nxt = res.keys[0].shape[2], [], int(res.logits[-1].argmax())
    while len(out) < max_tokens and nxt not in eng.eos:
        out.append(nxt)
        h = eng.inner.embed_tokens(torch.tensor([[nxt]], device=DEV))
        for layer, c in zip(eng.layers, caches):
            q, k, v = eng._qkv(layer.self_attn, layer.input_layernorm(h), torch.tensor([pos], device=DEV))
            c.append(k, v)
            K, V = c.tensors()
            o, _ = R.attention(q, K, V, torch.tensor([c.rows - 1]), q.shape[3] ** -0.5)
            h = h + layer.self_attn.o_proj(o.to(torch.bfloat16).to(DEV).reshape(1, 1, -1))
            h = h + layer.mlp(layer.post_attention_layernorm(h))
        nxt = int(eng._logits(h)[0, -1].argmax())
        pos += 1
    return out


@pytest.mark.parametrize("heads,kv", [(8, 2), (4, 4)])  # head_dim 64 and 128
@pytest.mark.parametrize("bits,keep", [(8, None), (16, 90), (8, 90)])
def test_generate_matches_the_plain_steps(heads, kv, bits, keep):
    eng = _engine(heads, kv)
    res = eng.prefill(_tokens(300), observe=24)
    kw = dict(cache_bits=bits, keep=keep, keep_sink=3, keep_recent=16)
    ours = eng.generate(res, max_tokens=12, **kw)  # device loop, HIP graph replays
    assert len(ours) > 0 and ours == _plain_generate(eng, res, 12, bits, keep, 3, 16)
    eng.decode_graphs = False
    assert eng.generate(res, max_tokens=12, **kw) == ours  # the same steps issued eagerly


def test_nothing_to_cut_and_plain_calls_stay_as_they_were():
    eng = _engine()
    toks = _tokens(120)
    plain = eng.prefill(toks)
    res = eng.prefill(toks, observe=8)
    assert plain.weights is None and torch.equal(plain.logits, res.logits)
    assert all(torch.equal(a, b) for a, b in zip(plain.keys + plain.values, res.keys + res.values))
    want = eng.generate(plain, max_tokens=8)
    assert eng.generate(res, max_tokens=8) == want
    assert eng.generate(plain, max_tokens=8, keep=120) == want  # 120 rows or fewer: no weights needed
    assert eng.generate(res, max_tokens=8, keep=500) == want


@pytest.mark.parametrize("blend", [False, True])
def test_observed_weights_match_the_plain_form(blend):
    """Of the last rows computed in each layer, over the caches that the prefill returns: for a full prefill, and for a blend,
    whose later layers compute some rows only."""
    eng = _engine()
    toks, placements, cfg = _tokens(200), None, None
    if blend:
        base = eng.prefill(toks)
        placements, cfg = [Placement(base.chunk(20, 100), 60), Placement(base.chunk(100, 160), 0)], BlendConfig(recompute_ratio=0.3, n_sink=4)
    seen = []
    attend = eng._attend_active

    def record(li, layer, h, q, K, V, active, *rest):
        seen.append((q.clone(), active.clone()))
        return attend(li, layer, h, q, K, V, active, *rest)

    eng._attend_active = record
    res = eng.prefill(toks, placements, cfg, observe=24)
    assert len(res.weights) == len(seen) == 3
    for (q, active), K, w in zip(seen, res.keys, res.weights):
        last = q[:, -24:].transpose(1, 2)
        want, most = R.weights(last, K, active[-24:], q.shape[3] ** -0.5)
        assert ((w.double().cpu() - want).abs() <= most).all()
        assert float(w.double().sum()) == pytest.approx(24 * 8, rel=1e-5)


def test_observing_more_rows_than_there_are():
    eng = _engine()
    a, b = eng.prefill(_tokens(30), observe=30), eng.prefill(_tokens(30), observe=1000)
    assert all(torch.equal(x, y) for x, y in zip(a.weights, b.weights))


def test_refusals():
    eng = _engine()
    res = eng.prefill(_tokens(64))
    for kw in (dict(cache_bits=4), dict(keep=40), dict(keep=8, keep_sink=4, keep_recent=5), dict(keep=0, keep_sink=0, keep_recent=0),
               dict(keep=40, keep_sink=-1)):
        with pytest.raises(ValueError):
            eng.generate(res, max_tokens=4, **kw)
    with pytest.raises(ValueError):
        eng.prefill(_tokens(8), observe=-1)
    f32 = HipEngine(tiny_qwen2(layers=2, hidden=256, heads=4, kv=2, inter=512, vocab=512, seed=1).to(DEV), StubTokenizer())
    with pytest.raises(ValueError):
        f32.prefill(_tokens(8), observe=4)
    with pytest.raises(ValueError):
        f32.generate(f32.prefill(_tokens(8)), cache_bits=8)


def test_operators_in_a_run():
    """Weights of a window, the cut, 8-bit rows, attention with appended rows: each step's result against the plain form of that step
    on the same inputs."""
    H, Hq, D, N, keep, steps = 4, 28, 128, 1500, 257, 5
    g = torch.Generator().manual_seed(1)
    r = lambda *s, scale=1.0: (torch.randn(s, generator=g) * scale).to(torch.bfloat16).to(DEV)  # noqa: E731
    K, V, q = r(1, H, N, D, scale=1.5), r(1, H, N, D), r(1, 32, Hq, D).transpose(1, 2)
    pos = torch.arange(N - 32, N)
    w = ops.attention_weights(q, K, pos.to(DEV))
    want, most = R.weights(q, K, pos, D ** -0.5)
    assert ((w.double().cpu() - want).abs() <= most).all()
    e = ops.evict_rows(K, V, w, keep, 4, 32)
    assert e.rows[0].tolist() == [R.kept_rows(w[0, h].cpu().numpy(), keep, 4, 32) for h in range(H)]
    c = ops.quantized_cache(H, keep + steps, D, DEV, 64)
    ops.quantize_rows(c, e.K, e.V)
    for i in range(steps):
        k1, v1, q1 = r(1, H, 1, D, scale=3.0), r(1, H, 1, D, scale=4.0), r(1, 1, Hq, D).transpose(1, 2)
        ops.quantize_rows(c, k1, v1, keep + i)
        out = ops.attention_quantized(q1, c, torch.tensor([keep + i], device=DEV))
        rows = [R.rows_of(t, s, 64)[:, :, : keep + i + 1] for t, s in ((c.k, c.k_scale), (c.v, c.v_scale))]
        o, off = R.attention(q1, *rows, torch.tensor([keep + i]), D ** -0.5)
        assert ((out[0].double().cpu() - o).abs() <= off).all()
        # an appended row is within half a step of e4m3 (2^-4 of the value, or half a subnormal step of its block's scale)
        for got, x, s in ((rows[0], k1, c.k_scale), (rows[1], v1, c.v_scale)):
            sc = s.cpu().double()[0, :, (keep + i) // 64, None]
            assert ((got[0, :, -1] - x.cpu().double()[0, :, 0]).abs() <= torch.maximum(x.cpu().double()[0, :, 0].abs() * 2.0 ** -4, sc * 2.0 ** -10)).all()
