"""ops.evict_rows against a plain form: the kept rows exactly, the copies bit for bit."""

import pytest
import torch

from chunkkv_amd import ops
from tests import decode_cache_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def _caches(H, N, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn((1, H, N, D), generator=g).to(dtype).to(DEV) for _ in range(2)]


def _weights(H, N, kind, seed):
    g = torch.Generator().manual_seed(seed)
    w = torch.exp(2 * torch.randn((1, H, N), generator=g) - 6)
    if kind == "ties":  # a few values, many rows each
        w = torch.randint(0, 4, (1, H, N), generator=g).float() / 8
    elif kind == "equal":
        w = torch.zeros(1, H, N)
    elif kind == "signs":  # both zeros, negatives, infinities, NaN of both signs, subnormals
        v = torch.tensor([0.0, -0.0, 1.0, -1.0, torch.inf, -torch.inf, torch.nan, -torch.nan, 1e-40, -1e-40, 3e38])
        w = v[torch.randint(0, len(v), (1, H, N), generator=g)]
    elif kind == "close":  # the top 22 bits alike
        w = (0x3F800000 + torch.randint(0, 1024, (1, H, N), generator=g).int()).view(F32)
    return w.to(DEV)


def _check(K, V, w, keep, sink, recent, **kw):
    e = ops.evict_rows(K, V, w, keep, sink, recent, **kw)
    rows = e.rows.cpu()
    for h in range(K.shape[1]):
        want = R.kept_rows(w[0, h].cpu().numpy(), keep, sink, recent)
        assert rows[0, h].tolist() == want, f"head {h}"
        at = torch.tensor(want, dtype=torch.int64, device=DEV)
        for got, src in ((e.K, K), (e.V, V), (e.weights, w)):
            a, b = got[0, h], src[0, h][at]
            i = torch.int16 if a.dtype == BF else torch.int32
            assert torch.equal(a.contiguous().view(i), b.contiguous().view(i))
    return e


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "signs", "close"])
@pytest.mark.parametrize("N,keep,sink,recent", [(1, 1, 0, 0), (7, 3, 1, 1), (100, 100, 4, 32), (1103, 300, 4, 32), (1103, 36, 4, 32),
                                                (1024, 1, 0, 0), (5000, 4999, 0, 0), (8257, 2048, 0, 64), (20000, 77, 7, 0)])
def test_kept_rows_match_the_plain_form(kind, N, keep, sink, recent):
    K, V = _caches(2, N, 64, BF, N)
    _check(K, V, _weights(2, N, kind, keep), keep, sink, recent)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_types_and_head_sizes(dtype, D):
    K, V = _caches(3, 333, D, dtype, D)
    _check(K, V, _weights(3, 333, "spread", 1), 100, 2, 9)


@pytest.mark.parametrize("N", [16384, 16385, 36864, 36865, 70001, 131072])
@pytest.mark.parametrize("kind", ["spread", "equal", "close"])
def test_long_caches(N, kind):
    K, V = _caches(1, N, 64, BF, N)
    _check(K, V, _weights(1, N, kind, 3), N // 7, 4, 64)


def test_views_of_longer_caches_and_given_outputs():
    """K/V and weights as views of slabs with room behind the rows, the kept rows into the front of another slab, whose
    other rows stay."""
    H, N, D, keep = 2, 500, 128, 123
    ks, vs = _caches(H, 640, D, BF, 1)
    w = _weights(H, 640, "spread", 2)[:, :, :N]
    ko, vo = _caches(H, 200, D, BF, 3)
    kb, vb = ko.clone(), vo.clone()
    e = _check(ks[:, :, :N], vs[:, :, :N], w, keep, 4, 16, k_out=ko[:, :, :keep], v_out=vo[:, :, :keep])
    assert e.K.data_ptr() == ko.data_ptr()
    assert torch.equal(ko[:, :, keep:], kb[:, :, keep:]) and torch.equal(vo[:, :, keep:], vb[:, :, keep:])


def test_nothing_kept():
    K, V = _caches(2, 50, 64, BF, 1)
    e = ops.evict_rows(K, V, _weights(2, 50, "spread", 1), 0)
    assert e.K.shape == (1, 2, 0, 64) and e.rows.shape == (1, 2, 0) and e.weights.shape == (1, 2, 0)


def test_captured_and_replayed():
    K, V = _caches(4, 3001, 128, BF, 1)
    w = _weights(4, 3001, "spread", 0)
    ops.evict_rows(K, V, w, 700, 4, 32)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        e = ops.evict_rows(K, V, w, 700, 4, 32)
    for s in range(4):
        w.copy_(_weights(4, 3001, ["spread", "ties", "signs", "close"][s], s))
        graph.replay()
        want = ops.evict_rows(K, V, w, 700, 4, 32)
        assert torch.equal(e.rows, want.rows) and torch.equal(e.K, want.K) and torch.equal(e.V, want.V)


def test_offsets_past_32_bits():
    N = 17_000_001  # 4.35 GB of keys
    K = torch.zeros((1, 1, N, 128), dtype=BF, device=DEV)
    K[0, 0, N - 5], K[0, 0, 3] = 2.0, 1.0
    w = torch.zeros((1, 1, N), device=DEV)
    w[0, 0, N - 5] = 1.0
    e = ops.evict_rows(K, K, w, 5)
    assert e.rows[0, 0].tolist() == [0, 1, 2, 3, N - 5]
    assert torch.equal(e.K[0, 0, :, 0].float().cpu(), torch.tensor([0.0, 0.0, 0.0, 1.0, 2.0]))


def test_refusals():
    K, V = _caches(2, 50, 64, BF, 1)
    w = _weights(2, 50, "spread", 1)
    for args, kw in (((K, V, w, 51), {}), ((K, V, w, -1), {}), ((K, V, w, 10, 6, 5), {}), ((K, V, w, 10, -1, 0), {}),
                     ((K, V, w, 10, 0, -1), {}), ((K, V[:, :1], w, 10), {}), ((K[:, :, ::2], V[:, :, ::2], w[:, :, ::2], 10), {}),
                     ((K, V, w[:, :, :49], 10), {}), ((K, V, w.double(), 10), {}), ((K, V, w.cpu(), 10), {}),
                     ((K, V, w, 10), {"k_out": K[:, :, :10]}), ((K, V, w, 10), {"v_out": K[:, :, :11]}),
                     ((K, V, w, 10), {"k_out": V[:, :, 20:30]}), ((K, V, w, 10), {"k_out": K[:, :, :10].float()}),
                     ((torch.cat([K, K]), torch.cat([V, V]), w, 10), {})):
        with pytest.raises(ValueError):
            ops.evict_rows(*args, **kw)
    with pytest.raises(TypeError):
        ops.evict_rows(K, V.float(), w, 10)
    with pytest.raises(TypeError):
        ops.evict_rows(K.half(), V.half(), w, 10)
    both = torch.empty((1, 2, 10, 64), dtype=BF, device=DEV)
    with pytest.raises(ValueError):
        ops.evict_rows(K, V, w, 10, k_out=both, v_out=both)
