"""Inputs of the packed-prompt and budgeted-cache tests, and how far a correct kernel may be from 64 bits.

Tolerances. Scores are sums of D exact products in fp32: each within ``D 2^-24 scale sum |q_i k_i|`` of its value, which
Cauchy-Schwarz bounds by ``D 2^-24 scale |q| |k|``; scaling, the soft cap, the exponential (relative 2^-22 for the
argument's rounding per unit of its size) and a sum of n terms add ``(|x| + n / 64 + 32) 2^-22``. Weights are rounded to the
type once (relative u = eps / 2), and outputs once more, so an output is within ``(u + e) sum p |v| + u |o|``, with e twice
the scores' error (a weight and its denominator).
"""

from __future__ import annotations

import numpy as np
import torch


def f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().double().cpu().numpy()


def score_error(q: torch.Tensor, k: torch.Tensor, scale: float, keys: int) -> float:
    d = q.shape[-1]
    qn = f64(q)[np.isfinite(f64(q)).all(-1)]
    kn = f64(k)[np.isfinite(f64(k)).all(-1)]
    size = scale * np.linalg.norm(qn, axis=-1).max(initial=0) * np.linalg.norm(kn, axis=-1).max(initial=0)
    return float(d * 2.0 ** -24 * size + (size + keys / 64 + 32) * 2.0 ** -22)


def assert_output(got: torch.Tensor, want: np.ndarray, size: np.ndarray, error: float) -> None:
    u = torch.finfo(got.dtype).eps / 2
    g = f64(got)
    finite = np.isfinite(want)
    assert np.array_equal(finite, np.isfinite(g)), "infinities and NaN elsewhere"
    assert np.array_equal(np.isnan(want), np.isnan(g))
    tiny = torch.finfo(got.dtype).smallest_normal
    bound = (u + 2 * error) * 1.01 * size + u * np.abs(want) + tiny
    with np.errstate(invalid="ignore"):
        off = np.abs(g - want)
    worst = np.max((off / bound)[finite], initial=0)
    assert worst <= 1, f"{worst:.3g} times the bound"


def prompt_inputs(seed: int, lens_q, lens_k, heads, dim, dtype, tail=0, device="cuda"):
    """Queries [T, Hq, D], keys and values [Tk, Hkv, D] with some heavy keys, and cu_seqlens of both."""
    gen = torch.Generator().manual_seed(seed)
    hq, hkv = heads
    t, tk = sum(lens_q) + tail, sum(lens_k) + tail
    u = torch.randn(hkv, dim, generator=gen)
    q = torch.randn(t, hkv, hq // hkv, dim, generator=gen) + 0.6 * u[:, None]
    k = torch.randn(tk, hkv, dim, generator=gen)
    k = k + (torch.rand(tk, hkv, 1, generator=gen) < 1 / 16) * 0.5 * u
    v = torch.randn(tk, hkv, dim, generator=gen)

    def cu(lens):
        return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=device)

    return (q.reshape(t, hq, dim).to(dtype).to(device), k.to(dtype).to(device), v.to(dtype).to(device), cu(lens_q),
            cu(lens_k))
