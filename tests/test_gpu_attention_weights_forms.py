"""ops.attention_weights in every kernel form that a launch can take, against a 64-bit softmax summed over queries and grouped
heads. tests/test_decode_cache_forms.py checks on the host that the shapes below, with those of test_gpu_attention_weights.py, leave no
form out."""

import pytest
import torch

from chunkkv_amd import ops
from tests import decode_cache_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16

# Hq, Hkv, D, N, n. QG, KG: 16-row groups of a wavefront in the first pass (query rows) and in the second (cache rows).
SHAPES = [
    (28, 4, 128, 16500, 300),  # QG 2 split, KG 2 in parts, joined by a launch: a follow-up question over a long cache
    (28, 4, 128, 2100, 2100),  # QG 2 split, KG 2 in parts that join: a prompt's own rows
    (64, 8, 128, 1500, 1300),  # QG 2 unsplit, KG 2 in parts
    (64, 8, 64, 1500, 1300),
    (14, 2, 128, 41000, 10),  # QG 2 split, KG 2 in one part, joined by a launch
    (24, 24, 64, 12001, 129),
    (32, 32, 128, 8302, 129),  # the same, joined by the second pass
    (32, 32, 64, 8302, 129),
    (32, 32, 64, 3300, 513),  # and in parts
    (4, 4, 128, 16500, 19),  # QG 1 split, KG 2
    (4, 4, 64, 16500, 19),
    (16, 16, 128, 4100, 19),
    (16, 16, 64, 4100, 19),
    (8, 2, 128, 11000, 129),
    (32, 32, 128, 650, 513),
    (32, 32, 64, 650, 513),
    (64, 8, 128, 513, 513),  # QG 1 unsplit
    (64, 8, 64, 513, 513),
    (1, 1, 128, 41000, 65),  # QG 2 split, KG 1
    (1, 1, 128, 5121, 500),  # QG 1 split, KG 1 in parts, joined by a launch
    (1, 1, 64, 5121, 500),
    (1, 1, 64, 5121, 19),  # and in one part
    (6, 2, 64, 1500, 4),  # one token's kernels, split, at head_dim 64
]


def _randn(shape, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(BF).to(DEV)


def _want(q, K, pos, prior=None):
    """The plain form, and its bound with a row's sum as one chain: unsplit, a lane adds a quarter of the cache's exponentials."""
    want, most = R.weights(q, K, pos, q.shape[3] ** -0.5, prior)
    added = want if prior is None else want - prior.double().cpu()
    return want, most + K.shape[2] / 4 * R.F32_STEP * added


def _check(q, K, pos, prior):
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = ops.attention_weights(q, K, pos.to(DEV), prior=prior, err=err)
    assert int(err) == 0
    want, most = _want(q, K, pos, prior)
    off = (got.double().cpu() - want).abs()
    assert (off <= most).all(), f"{float((off / most).max())} times the bound"
    last = int(pos.max())
    base = torch.zeros_like(got) if prior is None else prior
    assert torch.equal(got[:, :, last + 1 :], base[:, :, last + 1 :])


@pytest.mark.parametrize("Hq,Hkv,D,N,n", SHAPES)
def test_every_form_matches_the_plain_form(Hq, Hkv, D, N, n):
    """Query rows at the end of the cache, as a follow-up question has them, n - n // 4 of them; the rest anywhere."""
    q, K = _randn((1, n, Hq, D), N).transpose(1, 2), _randn((1, Hkv, N, D), n, 1.5)
    head = torch.randperm(N - n + n // 4, generator=torch.Generator().manual_seed(n))[: n // 4].sort().values
    pos = torch.cat([head, torch.arange(N - (n - n // 4), N)])
    _check(q, K, pos, torch.rand((1, Hkv, N), device=DEV) if n % 2 else None)


@pytest.mark.parametrize("Hq,Hkv,D,N,n", [(28, 4, 128, 16500, 300), (32, 32, 64, 8302, 129), (64, 8, 128, 513, 513), (14, 2, 128, 41000, 10)])
def test_rows_behind_the_positions(Hq, Hkv, D, N, n):
    """Rows past the last position hold NaN, in tiles and splits that no query reaches too; positions in any order."""
    K, last = _randn((1, Hkv, N, D), 3), N // 3
    K[:, :, last + 1 :] = float("nan")
    pos = torch.randint(0, last + 1, (n,), generator=torch.Generator().manual_seed(N))
    pos[n // 2] = last
    _check(_randn((1, Hq, n, D), 4), K, pos, torch.rand((1, Hkv, N), device=DEV))


@pytest.mark.parametrize("Hq,Hkv,D,N,n", [(28, 4, 128, 16500, 300), (28, 4, 128, 2100, 2100), (64, 8, 64, 513, 513)])
def test_replays_match_eager_over_workspaces_full_of_nan(Hq, Hkv, D, N, n):
    K, q, pos = _randn((1, Hkv, N, D), 1), _randn((1, Hq, n, D), 2), torch.arange(N - n, N, device=DEV)
    ops.attention_weights(q, K, pos)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.attention_weights(q, K, pos)
    for step in range(4):
        q.copy_(_randn((1, Hq, n, D), 20 + step))
        pos.copy_(torch.randint(0, N, (n,), generator=torch.Generator().manual_seed(step)))
        graph.replay()
        for mb in (4, 32, 128):
            torch.full((mb << 18,), float("nan"), device=DEV)
        eager = ops.attention_weights(q, K, pos)
        assert torch.equal(out, eager) and torch.isfinite(eager).all()
