"""ops.evict_rows on both sides of each change between its kernel's forms: 1, 3 and 9 steps of 256 rows a wavefront, and from
34,817 rows on one workgroup a head and a copy behind it."""

import pytest
import torch

from chunkkv_amd import ops
from tests import test_gpu_evict as E

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32

# The last wavefront's run starts at row 34560 of the 9-step form: no rows of its own, one, and to the end of the integers' place.
EDGES = [4095, 4096, 4097, 8192, 8193, 12287, 12288, 12289, 16384, 32768, 32832, 34559, 34560, 34561, 34815, 34816, 34817, 34818]


@pytest.mark.parametrize("N", EDGES)
@pytest.mark.parametrize("kind", ["spread", "ties", "signs"])
def test_changes_between_the_forms(N, kind):
    K, V = E._caches(2, N, 64, BF, N)
    E._check(K, V, E._weights(2, N, kind, N), N // 5, 4, 64)


@pytest.mark.parametrize("N", [4097, 12289, 34816, 34817])
def test_nearly_every_row_and_hardly_any(N):
    K, V = E._caches(1, N, 64, F32, N)
    w = E._weights(1, N, "spread", N)
    for keep, sink, recent in ((N, 0, 0), (N - 1, 0, 0), (1, 0, 0), (1, 1, 0), (2, 0, 2), (N - 1, N // 2, N // 2 - 1)):
        E._check(K, V, w, keep, sink, recent)


@pytest.mark.parametrize("N", [32832, 34816, 50000])
def test_replays_match_eager(N):
    K, V = E._caches(2, N, 128, BF, 1)
    w = E._weights(2, N, "spread", 0)
    ops.evict_rows(K, V, w, 4000, 4, 32)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        e = ops.evict_rows(K, V, w, 4000, 4, 32)
    for s in range(4):
        w.copy_(E._weights(2, N, ["ties", "spread", "signs", "close"][s], s))
        graph.replay()
        want = ops.evict_rows(K, V, w, 4000, 4, 32)
        assert torch.equal(e.rows, want.rows) and torch.equal(e.K, want.K) and torch.equal(e.V, want.V)
        assert torch.equal(e.weights.view(torch.int32), want.weights.view(torch.int32))


def test_outputs_whose_heads_take_turns_with_others():
    """Disjoint caches that share a buffer: K's and V's kept rows head by head in one, and behind the rows of the caches
    that are cut."""
    H, N, D, keep = 4, 700, 64, 150
    K, V = E._caches(H, N, D, BF, 1)
    w = E._weights(H, N, "spread", 2)
    both = torch.zeros((1, H, 2, keep, D), dtype=BF, device=DEV)
    E._check(K, V, w, keep, 4, 16, k_out=both[:, :, 0], v_out=both[:, :, 1])
    assert both.any(-1).all()
    slabs = E._caches(H, N + 200, D, BF, 3)
    before = [t.clone() for t in slabs]
    k, v = (t[:, :, :N] for t in slabs)
    E._check(k, v, w, keep, 4, 16, k_out=slabs[0][:, :, N : N + keep], v_out=slabs[1][:, :, N : N + keep])
    for t, b in zip(slabs, before):
        assert torch.equal(t[:, :, :N], b[:, :, :N]) and torch.equal(t[:, :, N + keep :], b[:, :, N + keep :])
    for bad in (slabs[0][:, :, N - 1 : N - 1 + keep], slabs[1][:, :, 3 : 3 + keep]):  # the last row of each head, and inside V
        with pytest.raises(ValueError):
            ops.evict_rows(k, v, w, keep, k_out=bad)


def test_outputs_over_the_weights_are_refused():
    """fp32 caches: an output in the weights' buffer would be written while other workgroups still rank by it."""
    K, V = E._caches(2, 50, 64, F32, 1)
    flat = torch.rand(3000, device=DEV)
    w, keep = flat[: 2 * 50].view(1, 2, 50), 10
    out = lambda at: flat[at : at + 2 * keep * 64].view(1, 2, keep, 64)  # noqa: E731
    for kw in (dict(k_out=out(0)), dict(v_out=out(96)), dict(k_out=out(200), v_out=out(0))):
        with pytest.raises(ValueError, match="overlap"):
            ops.evict_rows(K, V, w, keep, **kw)
    E._check(K, V, w, keep, 0, 0, k_out=out(100), v_out=out(100 + 2 * keep * 64))
