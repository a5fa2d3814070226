"""The decode cache's entry points (8-bit rows, attention over them, attention weights, eviction) on a host without a GPU:
arguments that the C ABI refuses before any launch, workspace sizes, launch plans, and calls whose operands cannot be
launched, which end in a Python exception."""

import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

from chunkkv_amd import _native, ops

ROOT = Path(__file__).resolve().parents[1]
INVALID, RANGE, LARGE, OK = (_native.CKV_ERR_INVALID_ARGUMENT, _native.CKV_ERR_OUT_OF_RANGE, _native.CKV_ERR_TOO_LARGE, _native.CKV_OK)


def _with(base, **kw):
    names, values = zip(*base)
    assert set(kw) <= set(names)
    return [kw.get(n, v) for n, v in zip(names, values)]


QUANT = [("kc", 16), ("vc", 16), ("ks", 16), ("vs", 16), ("k", 16), ("k_hs", 512), ("k_ts", 64), ("v", 16), ("v_hs", 512), ("v_ts", 64),
         ("start", 0), ("start_dev", None), ("n", 8), ("N", 100), ("H", 2), ("D", 64), ("block", 64), ("dtype", 1), ("err", None),
         ("stream", None)]
ATTN = [("out", 16), ("q", 16), ("q_hs", 64), ("q_ts", 256), ("kc", 16), ("vc", 16), ("ks", 16), ("vs", 16), ("pos", 16), ("n", 2), ("N", 100),
        ("Hq", 4), ("Hkv", 2), ("D", 64), ("block", 32), ("scale", 0.125), ("ws", None), ("wsb", 0), ("err", None), ("stream", None)]
WEIGHTS = [("out", 16), ("prior", None), ("q", 16), ("q_hs", 64), ("q_ts", 256), ("k", 16), ("k_hs", 6400), ("pos", 16), ("n", 2), ("N", 100),
           ("Hq", 4), ("Hkv", 2), ("D", 64), ("dtype", 1), ("scale", 0.125), ("ws", 16), ("wsb", 1 << 20), ("err", None), ("stream", None)]
EVICT = [("ko", 16), ("ko_hs", 640), ("vo", 16), ("vo_hs", 640), ("rows", 16), ("wo", 16), ("k", 16), ("k_hs", 6400), ("v", 16),
         ("v_hs", 6400), ("w", 16), ("w_hs", 100), ("N", 100), ("keep", 10), ("sink", 2), ("recent", 3), ("H", 2), ("D", 64), ("dtype", 1),
         ("stream", None)]


@pytest.mark.parametrize("fn,base,cases", [
    ("ckv_quantize_rows", QUANT, [
        (dict(kc=None), INVALID), (dict(vs=None), INVALID), (dict(v=None), INVALID), (dict(kc=8), INVALID), (dict(k=8), INVALID),
        (dict(k_ts=68), INVALID), (dict(v_hs=510), INVALID), (dict(D=96), INVALID), (dict(D=256), INVALID), (dict(block=16), INVALID),
        (dict(block=96), INVALID), (dict(dtype=7), INVALID), (dict(n=-1), INVALID), (dict(N=0), INVALID), (dict(H=0), INVALID),
        (dict(start=-1), RANGE), (dict(start=93), RANGE), (dict(n=101), RANGE), (dict(n=101, start_dev=16), RANGE), (dict(H=70000), LARGE),
        (dict(n=0, k=None, v=None, kc=None), OK)]),
    ("ckv_attention_quantized", ATTN, [
        (dict(out=None), INVALID), (dict(ks=None), INVALID), (dict(pos=None), INVALID), (dict(q=8), INVALID), (dict(vc=8), INVALID),
        (dict(D=256), INVALID), (dict(block=0), INVALID), (dict(Hq=3), INVALID), (dict(Hkv=0), INVALID), (dict(N=0), INVALID), (dict(n=-1), INVALID),
        (dict(scale=0.0), INVALID), (dict(scale=float("nan")), INVALID), (dict(q_hs=68), INVALID), (dict(q_ts=56), RANGE),
        (dict(Hq=131072, Hkv=2), LARGE), (dict(n=0, q=None, out=None, pos=None), OK)]),
    ("ckv_attention_weights", WEIGHTS, [
        (dict(out=None), INVALID), (dict(q=None), INVALID), (dict(k=None), INVALID), (dict(pos=None), INVALID), (dict(k=8), INVALID),
        (dict(dtype=0), INVALID), (dict(D=256), INVALID), (dict(Hq=3), INVALID), (dict(N=0), INVALID), (dict(n=-1), INVALID),
        (dict(scale=-1.0), INVALID), (dict(q_hs=68), INVALID), (dict(q_ts=56), RANGE), (dict(k_hs=6392), RANGE), (dict(ws=None, n=400), INVALID),
        (dict(wsb=16, n=400), INVALID), (dict(ws=8, n=400), INVALID), (dict(n=1 << 30), LARGE),
        (dict(out=4096, prior=4096 + 796), INVALID), (dict(out=4096, prior=4096 - 4), INVALID), (dict(out=4096, prior=4100, n=0), INVALID), (dict(n=0, q=None, k=None, pos=None, prior=16), OK)]),
    ("ckv_evict_rows", EVICT, [
        (dict(ko=None), INVALID), (dict(rows=None), INVALID), (dict(w=None), INVALID), (dict(vo=8), INVALID), (dict(k=8), INVALID),
        (dict(ko_hs=644), INVALID), (dict(D=96), INVALID), (dict(dtype=2), INVALID), (dict(N=0), INVALID), (dict(sink=-1), INVALID),
        (dict(recent=-1), INVALID), (dict(keep=-1), INVALID), (dict(keep=101), RANGE), (dict(sink=8), RANGE), (dict(sink=2**31 - 1), RANGE),
        (dict(k_hs=6392), RANGE), (dict(w_hs=99), RANGE), (dict(ko_hs=632), RANGE), (dict(H=70000), LARGE), (dict(keep=0, sink=0, recent=0, ko=None), OK)]),
])
def test_arguments_are_refused_before_any_launch(fn, base, cases):
    call = getattr(_native.lib(), fn)
    for kw, want in cases:
        assert call(*_with(base, **kw)) == want, kw


def test_workspace_sizes_are_host_only():
    lib = _native.lib()
    attn = lib.ckv_attention_quantized_workspace_bytes
    assert attn(1, 100, 28, 4, 128) == 0  # one launch
    row = 28 * 132 * 4  # a partial row per query head: 128 values, its maximum and sum
    assert attn(1, 8256, 28, 4, 128) > row and attn(1, 8256, 28, 4, 128) % row == 0
    mid = attn(160, 8256, 28, 4, 128)  # splits of grouped rows, no bf16 copy
    assert 0 < mid <= 64 * 160 * row and mid % (160 * row) == 0
    assert attn(2976, 8256, 28, 4, 128) >= 2 * 2 * 4 * 8256 * 128  # the cache as bf16
    assert attn(0, 100, 28, 4, 128) == attn(1, 0, 28, 4, 128) == attn(1, 100, 28, 3, 128) == attn(1, 100, 28, 0, 128) == 0
    w = lib.ckv_attention_weights_workspace_bytes
    assert w(400, 100, 4, 4, 64) > 0 and w(40, 300, 4, 4, 64) > 0 and w(1, 100, 4, 4, 64) == w(40, 100, 4, 4, 64) == 0 and w(1, 2000, 4, 4, 64) > 0 and w(0, 100, 28, 4, 64) == w(1, 100, 28, 3, 64) == 0
    assert w(2**31 - 1, 100, 64, 1, 64) == 0  # refused by the call


def test_every_wave_plan_can_be_launched(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = tmp_path / "attention_wave_plan_walk"
    subprocess.run([gxx, "-O2", "-std=c++17", f"-I{ROOT / 'chunkkv_amd' / 'csrc'}",
                    str(ROOT / "tests" / "native" / "attention_wave_plan_walk.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=300).stdout
    checked, bad = map(int, out.splitlines()[-1].split())
    assert checked > 40_000 and bad == 0, out


def test_every_grouped_plan_can_be_launched(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = tmp_path / "attention_grouped_plan_walk"
    subprocess.run([gxx, "-O2", "-std=c++17", f"-I{ROOT / 'chunkkv_amd' / 'csrc'}",
                    str(ROOT / "tests" / "native" / "attention_grouped_plan_walk.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=300).stdout
    checked, taken, bad = map(int, out.splitlines()[-1].split())
    assert checked > 40_000 and taken > 2_000 and bad == 0, out


def test_host_tensors_and_block_sizes_are_refused():
    import torch

    bf = torch.bfloat16
    c = ops.quantized_cache(2, 64, 64, "cpu", 32)
    assert c.k.shape == (1, 2, 64, 64) and c.k_scale.shape == (1, 2, 2)
    k, pos = torch.zeros(1, 2, 4, 64, dtype=bf), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: ops.quantize_rows(c, k, k), lambda: ops.attention_quantized(k, c, pos), lambda: ops.attention_weights(k, k, pos),
                 lambda: ops.evict_rows(k, k, torch.zeros(1, 2, 4), 2)):
        with pytest.raises(ValueError, match="HIP device"):
            call()
    with pytest.raises(ValueError, match="block_tokens"):
        ops.quantized_cache(2, 64, 64, "cpu", 48)


PRELUDE = """
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from chunkkv_amd import ops
BF, I64 = torch.bfloat16, torch.int64
def t(*shape, dtype=BF):
    return torch.empty(shape, dtype=dtype, device="cuda")
def cache():
    return ops.QuantizedCache(t(1, 2, 64, 64, dtype=torch.float8_e4m3fn), t(1, 2, 64, 64, dtype=torch.float8_e4m3fn),
                              t(1, 2, 2, dtype=torch.float8_e8m0fnu), t(1, 2, 2, dtype=torch.float8_e8m0fnu), 32)
def batched(fn, x):
    return torch.func.vmap(fn)(torch.stack([x, x]))
CALLS = {
    "quantize_rows": lambda wrap: wrap(lambda k: ops.quantize_rows(cache(), k, t(1, 2, 8, 64)), t(1, 2, 8, 64)),
    "quantize_rows_dev": lambda wrap: wrap(lambda k: ops.quantize_rows(cache(), k, t(1, 2, 8, 64), t(1, dtype=I64)), t(1, 2, 8, 64)),
    "attention_quantized": lambda wrap: wrap(lambda q: ops.attention_quantized(q, cache(), t(8, dtype=I64)), t(1, 4, 8, 64)),
    "attention_weights": lambda wrap: wrap(lambda q: ops.attention_weights(q, t(1, 2, 64, 64), t(8, dtype=I64)), t(1, 4, 8, 64)),
    "evict_rows": lambda wrap: wrap(lambda k: ops.evict_rows(k, t(1, 2, 64, 64), t(1, 2, 64, dtype=torch.float32), 8), t(1, 2, 64, 64)),
    "evict_rows_out": lambda wrap: wrap(lambda k: ops.evict_rows(k, t(1, 2, 64, 64), t(1, 2, 64, dtype=torch.float32), 8,
                                                                 k_out=t(1, 2, 8, 64)), t(1, 2, 64, 64)),
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
    assert r.stdout.splitlines()[-1] == "alive"


@pytest.mark.parametrize("scale", [1e-39, 1e-60, 5e-324, 3e38, 1e300, float("inf"), -float("inf")])
def test_scales_that_fp32_cannot_hold_are_refused(scale):
    """Their product with log2(e) is 0, subnormal or infinite there, and a masked score times it a NaN."""
    assert _native.lib().ckv_attention_quantized(*_with(ATTN, scale=scale)) == INVALID
    assert _native.lib().ckv_attention_weights(*_with(WEIGHTS, scale=scale)) == INVALID
    assert _native.lib().ckv_attention_quantized(*_with(ATTN, scale=1e-37, n=0)) == OK
    assert _native.lib().ckv_attention_weights(*_with(WEIGHTS, scale=2e38, n=0, prior=16)) == OK
