"""ops.attention_quantized in every kernel form that a launch can take, against a 64-bit softmax over the rows that codes and scales
stand for. tests/test_decode_cache_forms.py checks on the host that the shapes below, with those of test_gpu_quantized_cache.py, leave no
form out."""

import pytest
import torch

from chunkkv_amd import ops
from tests import test_gpu_quantized_cache as Q

pytestmark = pytest.mark.gpu
DEV = "cuda"

# Hq, Hkv, D, N, rows, n, block
SHAPES = [
    (28, 4, 128, 8302, 8300, 1000, 64),  # the cache as bf16, then split 128-query workgroups: one workspace for both
    (3, 1, 128, 8302, 8257, 2976, 128),
    (14, 2, 64, 5121, 5121, 513, 32),
    (64, 8, 64, 1000, 990, 900, 64),  # unsplit
    (64, 8, 128, 1000, 1000, 438, 32),  # 3504 rows of a KV head: the cache as bf16; 3496: codes
    (64, 8, 128, 1000, 1000, 437, 32),
    (32, 32, 128, 8302, 8290, 84, 64),  # split 128-query workgroups over codes
    (1, 1, 128, 33, 33, 19, 32),  # 16 or 32 rows a workgroup, four or eight wavefronts; heads of one token side by side or not
    (28, 4, 128, 192, 190, 180, 64),
    (1, 1, 128, 800, 797, 19, 32),
    (28, 4, 128, 64, 63, 5, 32),
    (28, 4, 128, 1000, 999, 5, 128),
    (64, 8, 128, 257, 257, 200, 64),
    (1, 1, 128, 2050, 2049, 25, 64),
    (64, 1, 64, 650, 641, 4, 32),
    (14, 2, 64, 100, 97, 5, 32),
    (1, 1, 64, 2600, 2590, 25, 128),
    (14, 2, 64, 1000, 1000, 5, 64),
    (14, 2, 64, 3300, 3299, 7, 32),
    (64, 8, 64, 257, 250, 200, 64),
]


def _positions(rows, n):
    """Query rows at the end of the cache, as a follow-up question has them, n - n // 4 of them; the rest anywhere before."""
    head = torch.randperm(rows - n + n // 4, generator=torch.Generator().manual_seed(n))[: n // 4].sort().values
    return torch.cat([head, torch.arange(rows - (n - n // 4), rows)])


@pytest.mark.parametrize("Hq,Hkv,D,N,rows,n,block", SHAPES)
def test_every_form_matches_the_plain_form(Hq, Hkv, D, N, rows, n, block):
    c = Q._filled(Hkv, N, D, block, rows, N + n)
    Q._attends(Q._q(Hq, n, D, rows, token_major=n % 2 == 0), c, _positions(rows, n), rows)


@pytest.mark.parametrize("Hq,Hkv,D,N,n,block", [(28, 4, 128, 8302, 251, 64), (14, 2, 64, 16400, 160, 32)])
def test_a_follow_up_question_over_a_long_cache(Hq, Hkv, D, N, n, block):
    """Splits of grouped rows where every query row sits at the end of the cache: every split has work for every block."""
    c = Q._filled(Hkv, N, D, block, N - 3, n)
    Q._attends(Q._q(Hq, n, D, 1), c, torch.arange(N - 3 - n, N - 3), N - 3)


@pytest.mark.parametrize("Hq,Hkv,D,N,n", [(28, 4, 128, 8302, 1000), (64, 8, 64, 1000, 900), (32, 32, 128, 8302, 84), (14, 2, 64, 3300, 7)])
def test_replays_match_eager_over_workspaces_full_of_nan(Hq, Hkv, D, N, n):
    c, q, pos = Q._filled(Hkv, N, D, 32, N, 5), Q._q(Hq, n, D, 1), torch.arange(N - n, N, device=DEV)
    ops.attention_quantized(q, c, pos)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.attention_quantized(q, c, pos)
    for step in range(4):
        q.copy_(Q._q(Hq, n, D, 10 + step))
        pos.copy_(torch.randint(0, N, (n,), generator=torch.Generator().manual_seed(step)).sort().values)
        graph.replay()
        for mb in (4, 32, 128):
            torch.full((mb << 18,), float("nan"), device=DEV)
        eager = ops.attention_quantized(q, c, pos)
        assert torch.equal(out, eager) and torch.isfinite(eager).all()
