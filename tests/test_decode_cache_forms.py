"""The kernel forms that the decode cache's launches can take, walked on the host, and whether the GPU tests' shapes leave one out."""

import shutil
import subprocess
from pathlib import Path

import pytest

from tests import test_gpu_attention_weights as weights_tests
from tests import test_gpu_attention_weights_forms as weights_forms
from tests import test_gpu_quantized_attention_forms as quantized_forms
from tests import test_gpu_quantized_cache as quantized_tests

ROOT = Path(__file__).resolve().parents[1]


def _shapes(test, names):
    """The parametrised shapes of a test."""
    return next(m.args[1] for m in test.pytestmark if m.name == "parametrize" and m.args[0] == names)


def _walker(tmp_path, name):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = tmp_path / name
    subprocess.run([gxx, "-O2", "-std=c++17", f"-I{ROOT / 'chunkkv_amd' / 'csrc'}", str(ROOT / "tests" / "native" / f"{name}.cpp"), "-o", str(exe)],
                   check=True)

    def run(shapes=()):
        text = "".join(" ".join(map(str, s)) + "\n" for s in shapes)
        return subprocess.run([str(exe)], input=text, check=True, capture_output=True, text=True, timeout=300).stdout.splitlines()

    return run


def _forms(run, shapes):
    lines = run(shapes)
    assert len(lines) == len(shapes)
    return {f for line in lines for f in line.split("; ")}


def test_every_form_of_the_attention_weights_is_tested(tmp_path):
    run = _walker(tmp_path, "attention_weights_forms")
    *every, counts = run()
    walked, bad = map(int, counts.split())
    assert walked > 100_000 and bad == 0, every
    shapes = _shapes(weights_tests.test_weights_match_the_plain_form, "Hq,Hkv,D,N,n") + weights_forms.SHAPES
    assert set(every) - _forms(run, shapes) == set()


def test_every_form_of_attention_over_an_8_bit_cache_is_tested(tmp_path):
    run = _walker(tmp_path, "attention_quantized_forms")
    *every, counts = run()
    walked, bad = map(int, counts.split())
    assert walked > 100_000 and bad == 0, every
    both = _shapes(quantized_tests.test_attention_matches_the_plain_form, "Hq,Hkv,D,N,rows,n,block")  # with and without a workspace
    shapes = [(hq, hkv, d, N, n, ws) for hq, hkv, d, N, _, n, _ in both for ws in (0, 1)]
    shapes += [(hq, hkv, d, N, n, 1) for hq, hkv, d, N, _, n, _ in quantized_forms.SHAPES]
    assert set(every) - _forms(run, shapes) == set()
