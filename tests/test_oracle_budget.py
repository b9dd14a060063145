"""The oracle of packed prompts and budgeted caches (``oracle/budget.py``) against loops over single pairs, closed forms
and a brute-force selection."""

from __future__ import annotations

import math

import numpy as np

from oracle import budget as ob
from oracle.attention import reference_attention


def _inputs(seed, tq, tk, hq, hkv, d):
    rng = np.random.default_rng(seed)
    return (rng.standard_normal((tq, hq, d)), rng.standard_normal((tk, hkv, d)), rng.standard_normal((tk, hkv, d)))


def test_prompt_is_the_masked_attention_of_each_sequence() -> None:
    q, k, v = _inputs(0, 11, 15, 4, 2, 8)
    cu_q, cu_k = [0, 4, 4, 11], [0, 6, 6, 15]
    out, lse, _ = ob.prompt_attention(q, k, v, cu_q, cu_k, 0.3, 5.0, [0.1, -2.0, 0.0, 1.0])
    for (a, b), (c, e) in (((0, 4), (0, 6)), ((4, 11), (6, 15))):
        mask = np.arange(e - c)[None] <= np.arange(b - a)[:, None] + (e - c) - (b - a)
        want = reference_attention(q[None, a:b].transpose(0, 2, 1, 3), k[None, c:e].transpose(0, 2, 1, 3),
                                   v[None, c:e].transpose(0, 2, 1, 3), mask[None, None], 0.3, 5.0,
                                   np.array([0.1, -2.0, 0.0, 1.0]))[0]
        np.testing.assert_allclose(out[a:b], want, atol=1e-5)
    # one pair by hand: the second sequence's query 4 sees keys 6 .. 8
    x = [5 * math.tanh(0.3 * float(q[4, 1] @ k[j, 0]) / 5) for j in range(6, 9)]
    assert math.isclose(lse[1, 4], math.log(sum(map(math.exp, x)) + math.exp(-2.0)), rel_tol=1e-12)


def test_rows_without_keys_and_unseen_infinities() -> None:
    q, k, v = _inputs(1, 5, 2, 2, 1, 8)
    v[1] = np.inf
    out, lse, _ = ob.prompt_attention(q, k, v, [0, 5], [0, 2], 1.0)
    assert not out[:3].any() and np.isneginf(lse[:, :3]).all()
    assert np.isfinite(out[3]).all() and np.isinf(out[4]).all()


def test_masses_sum_to_one_per_query_and_head() -> None:
    q, k, v = _inputs(2, 9, 12, 4, 2, 8)
    _, lse, _ = ob.prompt_attention(q, k, v, [0, 9], [0, 12], 0.5)
    mass = ob.attention_mass(q, k, lse, [0, 9], [0, 12], 0.5)
    np.testing.assert_allclose(mass.sum(1), 9 * 2)
    window = ob.attention_mass(q, k, lse, [0, 9], [0, 12], 0.5, window=3)
    np.testing.assert_allclose(window.sum(1), 3 * 2)
    by_hand = sum(math.exp(0.5 * float(q[i, h] @ k[10, 1]) - lse[h, i]) for h in (2, 3) for i in range(7, 9))
    assert math.isclose(mass[1, 10], by_hand, rel_tol=1e-12)


def test_eviction_keeps_the_heaviest_and_the_lower_of_equals() -> None:
    mass = np.array([0.0, 9.0, 2.0, 2.0, np.nan, 2.0, -np.inf, 5.0, 0.0, 0.0])
    assert ob.evict(mass, 6, 2, 1).tolist() == [0, 1, 2, 7, 8, 9]
    assert ob.evict(mass, 9, 2, 1).tolist() == [0, 1, 2, 3, 5, 6, 7, 8, 9]
    assert ob.evict(mass, 10, 2, 1).tolist() == list(range(10))
    assert ob.evict(mass, 3, 2, 1).tolist() == [0, 8, 9]


def test_steps_keep_the_budget_and_the_weights() -> None:
    rng = np.random.default_rng(3)
    c, d = 5, 4
    state = dict(keys=np.zeros((1, c, d)), values=np.zeros((1, c, d)), score=np.zeros((1, c)),
                 position=np.zeros((1, c), int), count=np.zeros(1, int), length=0)
    gained = 0.0
    for t in range(12):
        lost = state["score"][0].min() if state["count"][0] == c else 0.0
        q, k, v = (rng.standard_normal((n, d)) for n in (2, 1, 1))
        before = state["score"][0].copy()
        pos = state["position"][0].copy()
        ob.heavy_step(state, q, k, v, c, 2, 1, 0.5)
        if t >= c:
            to = int(np.nonzero(state["position"][0] == t)[0][0])
            free = [s for s in range(c) if 1 <= pos[s] <= t - 2]
            assert to in free and before[to] == min(before[s] for s in free)
            lost = before[to]
        else:
            lost = 0.0
        gained += 2 - lost
        np.testing.assert_allclose(state["score"][0].sum(), gained)
    assert 0 in state["position"][0] and {10, 11} <= set(state["position"][0].tolist())
