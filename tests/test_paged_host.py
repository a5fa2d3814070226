"""The paged cache's and the logits' entry points on a host without a GPU: arguments that the C ABI refuses before any launch, workspace
sizes, launch plans, and calls whose operands cannot be launched, which end in a Python exception."""

import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from chunkkv_amd import _native, ops
from tests.paged_ref import FORMS, Book, adjusted, attention

ROOT = Path(__file__).resolve().parents[1]
INVALID, RANGE, LARGE, OK = (_native.CKV_ERR_INVALID_ARGUMENT, _native.CKV_ERR_OUT_OF_RANGE, _native.CKV_ERR_TOO_LARGE, _native.CKV_OK)

BOOK = [("table", 16), ("lengths", 16), ("refs", 16), ("S", 4), ("M", 8), ("P", 20), ("T", 32)]
POOL = [("k", 16), ("v", 16), ("ls", 2 * 640 * 64), ("hs", 640 * 64), ("L", 3), ("H", 2), ("D", 64), ("dtype", 1)]
EXTEND = [("positions", 16), ("rows", 16), ("starts", 16), ("n", 5), ("counts", 16), *BOOK, ("err", None), ("stream", None)]
FORK = [*POOL, ("sources", 16), ("targets", 16), ("n", 2), *BOOK, ("ws", 16), ("wsb", 1 << 20), ("err", None), ("stream", None)]
FREE = [("sequences", 16), ("keep", None), ("n", 2), *BOOK, ("ws", 16), ("wsb", 8), ("err", None), ("stream", None)]
COMPACT = [*POOL, ("used", 16), *BOOK, ("ws", 16), ("wsb", 1 << 20), ("err", None), ("stream", None)]
ATTN = [("out", 16), ("q", 16), ("q_hs", 64), ("q_ts", 256), ("k", 16), ("v", 16), ("hs", 640 * 64), ("table", 16), ("lengths", 16), ("starts", 16),
        ("n", 5), ("most", 0), ("longest", 0), ("total", 0), ("S", 4), ("M", 8), ("P", 20), ("T", 32), ("Hq", 4), ("Hkv", 2), ("D", 64), ("dtype", 1), ("scale", 0.125), ("ws", None),
        ("wsb", 0), ("err", None), ("stream", None)]
LOGITS = [("logits", 16), ("row", 100), ("n", 2), ("vocab", 100), ("dtype", 1), ("prompt", 16), ("p_row", 7), ("np", 7), ("gen", 16), ("g_row", 3), ("ng", 3),
          ("rep_rows", None), ("rep", 1.0), ("freq_rows", None), ("freq", 0.0), ("pres_rows", None), ("pres", 0.0), ("bias", 16), ("b_row", 0),
          ("allowed", 16), ("a_row", 4)]
ADJUST = [("out", 16), *LOGITS, ("stream", None)]
NEXT = [("tokens", 16), *LOGITS, ("ws", None), ("wsb", 0), ("err", None), ("stream", None)]

BAD_BOOK = [(dict(table=None), INVALID), (dict(lengths=None), INVALID), (dict(refs=None), INVALID), (dict(S=0), INVALID), (dict(M=0), INVALID),
            (dict(P=-1), INVALID), (dict(T=16), INVALID), (dict(T=48), INVALID), (dict(S=4097), LARGE), (dict(M=1 << 27), LARGE), (dict(P=1 << 26), LARGE)]
BAD_POOL = [(dict(k=None), INVALID), (dict(v=8), INVALID), (dict(D=96), INVALID), (dict(dtype=2), INVALID), (dict(L=0), INVALID), (dict(H=0), INVALID),
            (dict(hs=640 * 64 + 4), INVALID), (dict(hs=639 * 64), RANGE), (dict(ls=640 * 64), RANGE)]
BAD_LOGITS = [(dict(logits=None), INVALID), (dict(logits=17), INVALID), (dict(logits=18, dtype=0), INVALID), (dict(dtype=2), INVALID), (dict(vocab=0), INVALID),
              (dict(n=-1), INVALID), (dict(np=-1), INVALID), (dict(prompt=None), INVALID), (dict(gen=12), INVALID), (dict(bias=18), INVALID), (dict(allowed=2), INVALID),
              (dict(row=99), RANGE), (dict(b_row=-1), RANGE), (dict(p_row=-7), RANGE), (dict(n=65536), LARGE), (dict(vocab=2**31 - 1, row=2**31), LARGE),
              (dict(n=0, logits=None), OK)]


def _with(base, **kw):
    names, values = zip(*base)
    assert set(kw) <= set(names)
    return [kw.get(n, v) for n, v in zip(names, values)]


@pytest.mark.parametrize("fn,base,cases", [
    ("ckv_extend_pages", EXTEND, BAD_BOOK + [(dict(n=-1), INVALID), (dict(counts=None), INVALID), (dict(starts=None), INVALID), (dict(rows=None), INVALID),
                                             (dict(positions=None), INVALID)]),
    ("ckv_fork_pages", FORK, BAD_BOOK + BAD_POOL + [(dict(n=-1), INVALID), (dict(sources=None), INVALID), (dict(targets=None), INVALID), (dict(ws=None), INVALID),
                                                    (dict(wsb=8), INVALID), (dict(ws=2), INVALID), (dict(n=4097), LARGE), (dict(n=0, sources=None, ws=None), OK)]),
    ("ckv_free_pages", FREE, BAD_BOOK + [(dict(n=-1), INVALID), (dict(sequences=None), INVALID), (dict(keep=16, ws=None), INVALID), (dict(keep=16, wsb=7), INVALID),
                                         (dict(n=4097), LARGE), (dict(n=0, sequences=None), OK)]),
    ("ckv_compact_pages", COMPACT, BAD_BOOK + BAD_POOL + [(dict(used=None), INVALID), (dict(ws=None), INVALID), (dict(wsb=100), INVALID)]),
    ("ckv_attention_paged", ATTN, [
        (dict(out=None), INVALID), (dict(q=None), INVALID), (dict(k=None), INVALID), (dict(table=None), INVALID), (dict(lengths=None), INVALID),
        (dict(starts=None), INVALID), (dict(q=8), INVALID), (dict(v=8), INVALID), (dict(out=8), INVALID), (dict(D=256), INVALID), (dict(dtype=0), INVALID),
        (dict(T=16), INVALID), (dict(Hq=3), INVALID), (dict(Hkv=0), INVALID), (dict(n=-1), INVALID), (dict(most=-1), INVALID), (dict(longest=-1), INVALID), (dict(total=-1), INVALID), (dict(S=0), INVALID), (dict(M=0), INVALID),
        (dict(P=0), INVALID), (dict(scale=0.0), INVALID), (dict(scale=float("inf")), INVALID), (dict(scale=1e-40), INVALID), (dict(q_hs=68), INVALID),
        (dict(q_ts=56), RANGE), (dict(hs=639 * 64), RANGE), (dict(S=4097), LARGE), (dict(M=1 << 26), LARGE), (dict(P=1 << 26, hs=1 << 40), LARGE), (dict(n=1 << 30), LARGE),
        (dict(n=0, q=None, out=None), OK)]),
    ("ckv_adjust_logits", ADJUST, BAD_LOGITS + [(dict(out=None), INVALID), (dict(out=18), INVALID)]),
    ("ckv_next_tokens", NEXT, BAD_LOGITS + [(dict(tokens=None), INVALID), (dict(tokens=20), INVALID), (dict(vocab=152064, row=152064), INVALID),
                                            (dict(vocab=152064, row=152064, ws=16, wsb=64), INVALID), (dict(vocab=152064, row=152064, ws=20, wsb=1 << 20), INVALID)]),
])
def test_arguments_are_refused_before_any_launch(fn, base, cases):
    call = getattr(_native.lib(), fn)
    for kw, want in cases:
        assert call(*_with(base, **kw)) == want, kw


def test_workspace_sizes_are_host_only():
    lib = _native.lib()
    assert lib.ckv_fork_pages_workspace_bytes(0) == 0 and lib.ckv_fork_pages_workspace_bytes(7) == 7 * lib.ckv_fork_pages_workspace_bytes(1) > 0
    assert lib.ckv_compact_pages_workspace_bytes(0) == 0 and lib.ckv_compact_pages_workspace_bytes(10) == 4 * (1 + 10 + 10)
    assert lib.ckv_next_tokens_workspace_bytes(3, 100) == 0 and lib.ckv_next_tokens_workspace_bytes(0, 152064) == 0
    assert lib.ckv_next_tokens_workspace_bytes(3, 152064) % 24 == 0 and lib.ckv_next_tokens_workspace_bytes(3, 152064) > 0
    w = lib.ckv_attention_paged_workspace_bytes
    assert w(1, 1, 1, 0, 0, 2, 64, 28, 4, 128) == 0  # a table of one split's rows
    assert w(1, 1, 1, 0, 0, 200, 64, 28, 4, 128) > 0 and w(1, 1, 1, 0, 0, 200, 64, 28, 4, 128) % (4 * 16 * 132 * 4) == 0
    assert w(1, 1, 1, 500, 0, 200, 64, 28, 4, 128) == 0  # short rows, if they are known to be
    assert w(8000, 2, 4000, 0, 0, 200, 64, 28, 4, 128) == 0  # tiles enough
    assert w(0, 1, 1, 0, 0, 200, 64, 28, 4, 128) == w(1, 1, 1, 0, 0, 200, 64, 28, 3, 128) == w(1, 0, 1, 0, 0, 200, 64, 28, 4, 128) == 0


def test_every_paged_plan_can_be_launched(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = tmp_path / "attention_paged_plan_walk"
    subprocess.run([gxx, "-O2", "-std=c++17", f"-I{ROOT / 'chunkkv_amd' / 'csrc'}", str(ROOT / "tests" / "native" / "attention_paged_plan_walk.cpp"), "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=300).stdout
    checked, split, bad = map(int, out.splitlines()[-1].split())
    assert checked > 40_000 and split > 10_000 and bad == 0, out


def test_every_kernel_form_is_tested(tmp_path):
    """The launches that tests/test_gpu_attention_paged.py compares reach every form that a plan can name."""
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = tmp_path / "attention_paged_forms"
    subprocess.run([gxx, "-O2", "-std=c++17", f"-I{ROOT / 'chunkkv_amd' / 'csrc'}", str(ROOT / "tests" / "native" / "attention_paged_forms.cpp"), "-o", str(exe)], check=True)
    lines = []
    for (hq, hkv, d), seqs, most, known in FORMS:
        entries = max(-(-r // 64) for r, _ in seqs) + 1  # as the GPU test's batches have them
        total = sum(r for r, _ in seqs) if known else 0
        lines.append(f"{sum(c for _, c in seqs)} {len(seqs)} {most} {entries * 64} {total} {hq} {hkv} {d} 1")
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True, input="\n".join(lines), timeout=60).stdout
    got = {tuple(map(int, line.split())) for line in out.splitlines()}
    want = {(d, r, split, spread, many) for d in (64, 128) for r in (16, 32, 128) for split, spread in ((0, 0), (1, 0), (1, 1)) for many in ((0, 1) if r < 128 else (0,))}
    assert got == want, (want - got, got - want)


def test_host_tensors_and_page_sizes_are_refused():
    c = ops.paged_cache(2, 4, 2, 64, 3, 100, "cpu", 32)
    assert c.k.shape == (2, 1, 2, 128, 64) and c.table.shape == (3, 4) and c.refs.shape == (4,) and int(c.lengths.sum()) == 0
    one, x = torch.zeros(3, dtype=torch.int32), torch.zeros(2, 100)
    for call in (lambda: ops.extend_pages(c, one, 2), lambda: ops.fork_pages(c, one, one), lambda: ops.free_pages(c, one), lambda: ops.compact_pages(c),
                 lambda: ops.attention_paged(torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16), c, 0, torch.zeros(4, dtype=torch.int32)),
                 lambda: ops.adjust_logits(x), lambda: ops.next_tokens(x)):
        with pytest.raises(ValueError, match="HIP device"):
            call()
    with pytest.raises(ValueError, match="page_tokens"):
        ops.paged_cache(2, 4, 2, 64, 3, 100, "cpu", 16)
    with pytest.raises(ValueError, match="at least"):
        ops.paged_cache(2, 0, 2, 64, 3, 100, "cpu")
    with pytest.raises(TypeError):
        ops.paged_cache(2, 4, 2, 64, 3, 100, "cpu", dtype=torch.float16)


def test_token_bits():
    bits = ops.token_bits([0, 31, 32, 99], 100, "cpu")
    assert bits.dtype == torch.int32 and bits.tolist() == [1 - 2**31, 1, 0, 8]
    for bad in (-1, 100):
        with pytest.raises(ValueError):
            ops.token_bits([bad], 100, "cpu")


def test_the_plain_forms_agree_with_simple_cases():
    """What the GPU tests compare with, by hand."""
    b = Book(3, 4, 6, 32)
    assert b.extend([33, 0, 1], 40) == ([*range(33), 0] + [0] * 6, [*range(33), 64] + [-1] * 6, [0, 33, 33, 34])
    b.fork([0], [1])
    assert b.table == [[0, 1], [0, 3], [2]] and b.refs == [2, 1, 1, 1, 0, 0] and b.moves == [(1, 3)]
    b.free([0])
    assert b.refs == [1, 0, 1, 1, 0, 0] and b.compact() == 3 and b.table == [[], [0, 1], [2]]
    assert b.extend([200, 0, 0], 300)[2] == [0, 0, 0, 0] and b.err == 1
    x = adjusted(torch.tensor([[2.0, -2.0, 1.0, 5.0]]), torch.tensor([[1, -1]]), torch.tensor([[0, 0, 9]]), 2.0, 0.25, 0.5, None, torch.tensor([7], dtype=torch.int32))
    assert x.tolist() == [[1.0 - 0.5 - 0.5, -4.0, 1.0, -torch.inf]]
    q, K = torch.ones(2, 1, 64), torch.zeros(1, 4, 64)
    out, bound = attention(q, K, torch.arange(4.0)[None, :, None].expand(1, 4, 64), 1)
    assert torch.allclose(out, torch.full((1, 2, 64), 1.5, dtype=torch.float64)) and (bound > 0).all()


PRELUDE = """
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from chunkkv_amd import ops
BF, I32, I64 = torch.bfloat16, torch.int32, torch.int64
def t(*shape, dtype=I32):
    return torch.empty(shape, dtype=dtype, device="cuda")
def cache():
    return ops.PagedCache(t(2, 1, 2, 128, 64, dtype=BF), t(2, 1, 2, 128, 64, dtype=BF), t(3, 4), t(3), t(4), 32)
def batched(fn, x):
    return torch.func.vmap(fn)(torch.stack([x, x]))
CALLS = {
    "extend_pages": lambda wrap: wrap(lambda c: ops.extend_pages(cache(), c, 5), t(3)),
    "fork_pages": lambda wrap: wrap(lambda c: ops.fork_pages(cache(), c, t(2)), t(2)),
    "free_pages": lambda wrap: wrap(lambda c: ops.free_pages(cache(), c), t(2)),
    "free_pages_keep": lambda wrap: wrap(lambda c: ops.free_pages(cache(), t(2), c), t(2)),
    "compact_pages": lambda wrap: wrap(lambda e: ops.compact_pages(cache(), e), t(1)),
    "attention_paged": lambda wrap: wrap(lambda q: ops.attention_paged(q, cache(), 0, t(4)), t(1, 4, 8, 64, dtype=BF)),
    "adjust_logits": lambda wrap: wrap(lambda x: ops.adjust_logits(x, generated=t(2, 3, dtype=I64)), t(2, 100, dtype=BF)),
    "next_tokens": lambda wrap: wrap(lambda x: ops.next_tokens(x, repetition=t(2, dtype=torch.float32)), t(2, 100, dtype=BF)),
}
"""


@pytest.mark.parametrize("wrap", ["lambda fn, x: fn(x)", "batched"], ids=["plain", "vmap"])
def test_failing_lookups_raise(wrap):
    body = f"""
with FakeTensorMode():
    for name, call in CALLS.items():
        try:
            call({wrap})
        except Exception as e:
            print(name, type(e).__name__, flush=True)
        else:
            raise SystemExit(name + " did not raise")
print("alive")
"""
    env = dict(os.environ, HIP_VISIBLE_DEVICES="-1")  # no device, also where there is one
    r = subprocess.run([sys.executable, "-c", PRELUDE + body], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.returncode, r.stdout[-2000:], r.stderr[-2000:])


MISUSE = PRELUDE + """
F32 = torch.float32
def bad(name, error, call):
    try:
        call()
    except error as e:
        print(name, e, flush=True)
    else:
        raise SystemExit(name + " did not raise")
P = ops.PagedCache
def book(**kw):
    c = cache()
    for k, v in kw.items():
        setattr(c, k, v)
    return c
with FakeTensorMode():
    E = lambda c, n=t(3), m=5, **kw: ops.extend_pages(c, n, m, **kw)
    bad("page size", ValueError, lambda: E(book(page_tokens=16)))
    bad("table type", TypeError, lambda: E(book(table=t(3, 4, dtype=I64))))
    bad("lengths shape", ValueError, lambda: E(book(lengths=t(2))))
    bad("table strides", ValueError, lambda: E(book(table=t(3, 8)[:, :4])))
    bad("no page", ValueError, lambda: E(book(refs=t(0))))
    bad("counts shape", ValueError, lambda: E(cache(), t(4)))
    bad("counts type", ValueError, lambda: E(cache(), t(3, dtype=I64)))
    bad("negative n", ValueError, lambda: E(cache(), t(3), -1))
    bad("large n", ValueError, lambda: E(cache(), t(3), 2**31))
    bad("err type", ValueError, lambda: E(cache(), err=t(1, dtype=I64)))
    bad("pairs", ValueError, lambda: ops.fork_pages(cache(), t(2), t(3)))
    bad("pool shape", ValueError, lambda: ops.fork_pages(book(k=t(2, 1, 2, 96, 64, dtype=BF), v=t(2, 1, 2, 96, 64, dtype=BF)), t(2), t(2)))
    bad("pool type", TypeError, lambda: ops.fork_pages(book(v=t(2, 1, 2, 128, 64, dtype=F32)), t(2), t(2)))
    bad("pool half", TypeError, lambda: ops.compact_pages(book(k=t(2, 1, 2, 128, 64, dtype=torch.half), v=t(2, 1, 2, 128, 64, dtype=torch.half))))
    bad("pool strides", ValueError, lambda: ops.compact_pages(book(k=t(2, 1, 128, 2, 64, dtype=BF).transpose(2, 3))))
    bad("keep", ValueError, lambda: ops.free_pages(cache(), t(2), t(3)))
    q = t(1, 4, 8, 64, dtype=BF)
    A = ops.attention_paged
    bad("q type", TypeError, lambda: A(q.float(), cache(), 0, t(4)))
    bad("q head size", ValueError, lambda: A(t(1, 4, 8, 128, dtype=BF), cache(), 0, t(4)))
    bad("q heads", ValueError, lambda: A(t(1, 3, 8, 64, dtype=BF), cache(), 0, t(4)))
    bad("layer", ValueError, lambda: A(q, cache(), 2, t(4)))
    bad("negative layer", ValueError, lambda: A(q, cache(), -1, t(4)))
    bad("starts", ValueError, lambda: A(q, cache(), 0, t(3)))
    bad("most", ValueError, lambda: A(q, cache(), 0, t(4), most=0))
    bad("longest", ValueError, lambda: A(q, cache(), 0, t(4), longest=0))
    bad("total", ValueError, lambda: A(q, cache(), 0, t(4), total=0))
    bad("out", ValueError, lambda: A(q, cache(), 0, t(4), out=t(1, 8, 4, 32, dtype=BF)))
    bad("f32 cache", TypeError, lambda: A(q, book(k=t(2, 1, 2, 128, 64, dtype=F32), v=t(2, 1, 2, 128, 64, dtype=F32)), 0, t(4)))
    x = t(2, 100, dtype=BF)
    for call in (ops.adjust_logits, ops.next_tokens):
        bad("logits type", TypeError, lambda: call(t(2, 100, dtype=torch.half)))
        bad("logits shape", ValueError, lambda: call(t(100, dtype=BF)))
        bad("logits strides", ValueError, lambda: call(t(100, 2, dtype=BF).t()))
        bad("prompt type", ValueError, lambda: call(x, prompt=t(2, 5)))
        bad("prompt rows", ValueError, lambda: call(x, generated=t(3, 5, dtype=I64)))
        bad("repetition", ValueError, lambda: call(x, repetition=0.0))
        bad("repetition rows", ValueError, lambda: call(x, repetition=t(3, dtype=F32)))
        bad("frequency type", ValueError, lambda: call(x, frequency=t(2, dtype=BF)))
        bad("bias width", ValueError, lambda: call(x, bias=t(99, dtype=F32)))
        bad("bias type", ValueError, lambda: call(x, bias=t(100, dtype=BF)))
        bad("bias rows", ValueError, lambda: call(x, bias=t(3, 100, dtype=F32)))
        bad("allowed width", ValueError, lambda: call(x, allowed=t(2, 3)))
        bad("allowed type", ValueError, lambda: call(x, allowed=t(2, 4, dtype=I64)))
    bad("logits out", ValueError, lambda: ops.adjust_logits(x, out=t(2, 100, dtype=BF)))
    bad("tokens out", ValueError, lambda: ops.next_tokens(x, out=t(2)))
print("alive")
"""


def test_misuse_is_refused_by_name():
    """Shapes, types and strides that the calls refuse, on tensors that only look like a device's."""
    env = dict(os.environ, HIP_VISIBLE_DEVICES="-1")
    r = subprocess.run([sys.executable, "-c", MISUSE], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.rstrip().endswith("alive"), (r.returncode, r.stdout[-2000:], r.stderr[-2000:])
