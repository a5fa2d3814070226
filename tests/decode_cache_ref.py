"""Plain 64-bit forms of the decode cache's operators, on the CPU, for their tests."""

from __future__ import annotations

import numpy as np
import torch

BF16_STEP = 2.0 ** -8  # half a step of bf16, relative
F32_STEP = 2.0 ** -24


def e4m3(x: np.ndarray) -> np.ndarray:
    """The nearest e4m3 value to each x (|x| <= 448), of two the even one."""
    x = np.asarray(x, dtype=np.float64)
    _, e = np.frexp(x)  # x = m 2^e, 0.5 <= |m| < 1
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.round(x / step) * step


def scale_exponent(amax: float) -> int:
    """The least e >= -126 with amax <= 448 * 2^e."""
    e = -126
    while amax > np.ldexp(448.0, e):
        e += 1
    return e


def write_rows(values: np.ndarray, exps: np.ndarray, x: np.ndarray, start: int, block: int) -> None:
    """Rows x (n, D) into one head's code values (N, D) and exponents (blocks,), in place."""
    hi = start + len(x)
    for b in range(start // block, -(-hi // block)):
        lo, to = max(b * block, start), min((b + 1) * block, hi)
        e = scale_exponent(float(np.abs(x[lo - start:to - start]).max()))
        if lo > b * block:
            e = max(e, int(exps[b]))
            kept = values[b * block:lo]
            values[b * block:lo] = e4m3(np.ldexp(kept, int(exps[b]) - e))
        values[lo:to] = e4m3(np.ldexp(x[lo - start:to - start], -e))
        exps[b] = e


def rows_of(codes: torch.Tensor, scales: torch.Tensor, block: int) -> torch.Tensor:
    """(1, H, N, D) float64: what codes and scales stand for."""
    n = codes.shape[2]
    at = torch.arange(n) // block
    return codes.cpu().to(torch.float64) * scales.cpu().to(torch.float64)[:, :, at, None]


def softmax_rows(q: torch.Tensor, K: torch.Tensor, pos: torch.Tensor, scale: float):
    """Per query head h the softmax (n, N) of its rows, and a bound of what fp32 scores are off by: the sum of D exact
    products rounded at each addition, the scale's product and the exponential's argument, each by half a step."""
    q, K, pos = q[0].double().cpu(), K[0].double().cpu(), pos.cpu()
    group, D = q.shape[0] // K.shape[0], q.shape[2]
    seen = torch.arange(K.shape[1])[None, :] <= pos[:, None]
    K = torch.where((torch.arange(K.shape[1]) <= pos.max())[None, :, None], K, torch.zeros((), dtype=torch.float64))
    out, worst = [], 0.0
    for h in range(q.shape[0]):
        k = K[h // group]
        out.append(torch.softmax((q[h] @ k.T * scale).masked_fill(~seen, -torch.inf), 1))
        worst = max(worst, float((q[h].abs() @ k.abs().T * scale).max()) * (D + 3) * F32_STEP)
    return out, worst


def attention(q, K, V, pos, scale):
    """(n, Hq, D) output and the most each element may be off: every weight rounded to bf16 (and off by the scores' error,
    the exponential's last bit) in the sum and in the normaliser, one rounding at the end."""
    p, e_s = softmax_rows(q, K, pos, scale)
    V = V[0].double().cpu()
    V = torch.where((torch.arange(V.shape[1]) <= pos.max().cpu())[None, :, None], V, torch.zeros((), dtype=torch.float64))
    group = len(p) // V.shape[0]
    out = torch.stack([p[h] @ V[h // group] for h in range(len(p))], 1)
    mass = torch.stack([p[h] @ V[h // group].abs() for h in range(len(p))], 1)
    w = BF16_STEP + 2 * e_s + 4 * F32_STEP  # of a weight, relative
    chain = V.shape[1] * F32_STEP  # fp32 additions, at worst one after the other
    return out, ((w + chain) * (mass + out.abs()) * 1.02 + BF16_STEP * out.abs() + 2.0 ** -126)


def weights(q, K, pos, scale, prior=None):
    """(1, Hkv, N) weights and the most each may be off: a weight by its scores' and normaliser's error, the sum over R rows
    by a chain of R / 16 + 68 additions (16 lanes a row of the cache, 64 parts, the lanes' tree). An exponential below 2^-126
    is 0 on the device, whichever way its weight is normalised: each of the R weights may be off by that (R of 100 rows, sum
    3.9e-38: 1.61 * 2^-126)."""
    p, e_s = softmax_rows(q, K, pos, scale)
    H, group = K.shape[1], len(p) // K.shape[1]
    got = torch.stack([sum(p[h].sum(0) for h in range(k * group, (k + 1) * group)) for k in range(H)])[None]
    rows = group * pos.numel()
    per = 4 * e_s + (K.shape[2] / 64 + 80) * F32_STEP + (rows / 16 + 68) * F32_STEP
    base = torch.zeros_like(got) if prior is None else prior.double().cpu()
    return base + got, per * got + 2 * F32_STEP * (base.abs() + got) + rows * 2.0 ** -126


def kept_rows(w: np.ndarray, keep: int, sink: int, recent: int) -> list[int]:
    """One head's kept rows, ascending."""
    n = len(w)
    fixed = set(range(sink)) | set(range(n - recent, n))
    key = lambda r: (bool(np.isnan(w[r])), -float(w[r]) if not np.isnan(w[r]) else 0.0, r)  # noqa: E731
    return sorted(list(fixed) + sorted((r for r in range(n) if r not in fixed), key=key)[: keep - len(fixed)])
